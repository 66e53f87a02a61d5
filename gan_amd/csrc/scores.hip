// Candidate logits by class: out[r, i] = table[kind of row r][class of candidate i], and the gradient of the table.
#include "common.h"

namespace aig {
namespace {

constexpr float NOTHING = -__builtin_inff();

struct Windows {
    long long rows;
    int width, classes;
    long long nodes;
    int kinds;
    const int *cand, *counts, *cls, *row_kind, *by_kind, *kind_start;
    __device__ __forceinline__ int count(long long r) const { return counts ? min(max(counts[r], 0), width) : width; }
    // kind of the p-th row in the order of kinds, -1 where there is none
    __device__ __forceinline__ int kind_at(long long p) const {
        const int r = by_kind[p], k = r >= 0 && r < rows ? row_kind[r] : -1;
        return k < kinds ? k : -1;
    }
    // class of a candidate, -1 where it is none
    __device__ __forceinline__ int cls_of(int c) const {
        const int k = c >= 0 && c < nodes ? cls[c] : -1;
        return k >= 0 && k < classes ? k : -1;
    }
};

__global__ __launch_bounds__(256) void k_class_scores(Windows w, const float* __restrict__ table, float* __restrict__ out) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= w.rows * w.width) return;
    const long long r = i / w.width;
    const int at = (int)(i - r * w.width), kind = w.row_kind[r];
    float v = NOTHING;
    if (at < w.count(r) && kind >= 0 && kind < w.kinds) {
        const int c = w.cls_of(w.cand[i]);
        if (c >= 0) v = table[(long long)kind * w.classes + c];
    }
    out[i] = v;
}

// Rows in the order of their kinds are dealt to blocks in runs of RUN; a run may hold rows of several kinds.  A block adds
// the gradients of one kind's rows into private columns acc[class][thread] in LDS, sums the columns in a fixed order when
// the kind ends, and writes the sum as partial number (block + kind): no two (block, kind) pairs that occur share it.
constexpr int RUN = 64;

__global__ __launch_bounds__(256) void k_class_scores_bwd(Windows w, int threads, const float* __restrict__ grad, double* __restrict__ partial) {
    extern __shared__ float acc[];          // [classes][threads]
    const int t = threadIdx.x;
    const long long p0 = (long long)blockIdx.x * RUN, p1 = min(p0 + RUN, w.rows);
    for (int i = t; i < w.classes * threads; i += threads) acc[i] = 0.0f;
    __syncthreads();
    long long p = p0;
    while (p < p1) {
        const int kind = w.kind_at(p);
        if (kind < 0) {
            ++p;
            continue;
        }
        for (; p < p1 && w.kind_at(p) == kind; ++p) {
            const long long r = w.by_kind[p];
            const int n = w.count(r);
            for (int i = t; i < n; i += threads) {
                const int c = w.cls_of(w.cand[r * w.width + i]);
                if (c >= 0) acc[c * threads + t] += grad[r * w.width + i];
            }
        }
        __syncthreads();
        for (int c = t; c < w.classes; c += threads) {
            double s = 0.0;
            for (int j = 0; j < threads; ++j) {
                s += (double)acc[c * threads + j];
                acc[c * threads + j] = 0.0f;
            }
            partial[((long long)blockIdx.x + kind) * w.classes + c] = s;
        }
        __syncthreads();
    }
}

__global__ __launch_bounds__(64) void k_class_scores_finish(Windows w, const double* __restrict__ partial, float* __restrict__ d_table) {
    const int kind = blockIdx.x;
    const long long s = max(w.kind_start[kind], 0), e = min((long long)w.kind_start[kind + 1], w.rows);
    for (int c = threadIdx.x; c < w.classes; c += 64) {
        double sum = 0.0;
        if (e > s)
            for (long long b = s / RUN; b <= (e - 1) / RUN; ++b) sum += partial[(b + kind) * w.classes + c];
        d_table[(long long)kind * w.classes + c] = (float)sum;
    }
}
}  // namespace
}  // namespace aig

using namespace aig;

static int check_windows(const char* what, const aig_score_windows* w) {
    AIG_REQUIRE(w, "%s: null argument block", what);
    AIG_REQUIRE(w->rows >= 0 && w->width >= 1 && w->nodes >= 0 && w->kinds >= 1 && w->classes >= 1,
                "%s: bad sizes rows=%lld width=%lld nodes=%lld kinds=%lld classes=%lld", what, (long long)w->rows, (long long)w->width,
                (long long)w->nodes, (long long)w->kinds, (long long)w->classes);
    if (w->classes > AIG_MAX_CLASSES || w->kinds > AIG_MAX_KINDS || w->width > AIG_ROWS_MAX_WIDTH ||
        w->rows >= (1ll << 31) || w->rows * w->width > (1ll << 32) - 256)
        return fail(AIG_ELIMIT, "%s: rows=%lld width=%lld kinds=%lld classes=%lld: at most %d classes, %d kinds, rows of %d and fewer than 2^32 places", what,
                    (long long)w->rows, (long long)w->width, (long long)w->kinds, (long long)w->classes, AIG_MAX_CLASSES,
                    AIG_MAX_KINDS, AIG_ROWS_MAX_WIDTH);
    AIG_REQUIRE(w->rows == 0 || (w->cand && w->cls && w->row_kind), "%s: null pointer", what);
    return AIG_OK;
}
static Windows windows_of(const aig_score_windows* w) {
    return Windows{w->rows, (int)w->width, (int)w->classes, w->nodes, (int)w->kinds, w->cand, w->counts, w->cls, w->row_kind,
                   w->by_kind, w->kind_start};
}

extern "C" int aig_class_scores(const aig_score_windows* w, const float* table, float* out, void* stream) {
    if (const int rc = check_windows("aig_class_scores", w)) return rc;
    if (w->rows == 0) return AIG_OK;
    AIG_REQUIRE(table && out, "aig_class_scores: null pointer");
    hipLaunchKernelGGL(k_class_scores, dim3((unsigned)((w->rows * w->width + 255) / 256)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), windows_of(w), table, out);
    AIG_LAUNCH_CHECK();
    return AIG_OK;
}

extern "C" size_t aig_class_scores_bwd_ws_bytes(int64_t rows, int64_t kinds, int64_t classes) {
    if (rows < 0 || kinds < 1 || classes < 1) return 0;
    return align_up((size_t)((rows + RUN - 1) / RUN + kinds) * (size_t)classes * sizeof(double));
}

extern "C" int aig_class_scores_bwd(const aig_score_windows* w, const float* grad, float* d_table, void* ws, size_t ws_bytes, void* stream) {
    if (const int rc = check_windows("aig_class_scores_bwd", w)) return rc;
    AIG_REQUIRE(d_table && (w->rows == 0 || (grad && w->by_kind)) && w->kind_start, "aig_class_scores_bwd: null pointer");
    if (!ws || ws_bytes < aig_class_scores_bwd_ws_bytes(w->rows, w->kinds, w->classes))
        return fail(AIG_EWORKSPACE, "aig_class_scores_bwd: workspace of %zu bytes is too small", ws_bytes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    double* partial = static_cast<double*>(ws);
    const int threads = w->classes <= 128 ? 256 : w->classes <= 512 ? 64 : 32;      // columns of at most 128 KB
    const size_t lds = (size_t)w->classes * threads * sizeof(float);
    AIG_HIP_CHECK(ensure_dynamic_lds(reinterpret_cast<const void*>(k_class_scores_bwd), 128 * 1024));
    if (w->rows)
        hipLaunchKernelGGL(k_class_scores_bwd, dim3((unsigned)((w->rows + RUN - 1) / RUN)), dim3(threads), lds, s, windows_of(w), threads,
                           grad, partial);
    hipLaunchKernelGGL(k_class_scores_finish, dim3((unsigned)w->kinds), dim3(64), 0, s, windows_of(w), partial, d_table);
    AIG_LAUNCH_CHECK();
    return AIG_OK;
}
