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

// V places a lane (4 where rows start on 16 bytes and hold whole vectors), LPR lanes a row: a row's kind and count are read
// once for its places, and there is no division by the width.
template <int V, typename W> __device__ __forceinline__ void load_vec(const W* p, W (&v)[V]) {
    if constexpr (V == 4) {
        const int4 q = *reinterpret_cast<const int4*>(p);
        __builtin_memcpy(v, &q, 16);
    } else {
        v[0] = p[0];
    }
}

// 4 bytes read and 4 written a place; classes and table stay in the caches.  100,000 x 64: 51 MB in 18 us (2.9 TB/s), 26,279 x
// 512: 108 MB in 32 us (3.4 TB/s): the chain row -> candidate -> class -> score is four memory trips, and lanes with two or four
// rows in flight were no faster (18 and 19 us; eight waves a SIMD hide as much).
template <int V>
__global__ __launch_bounds__(256) void k_class_scores(Windows w, int lpr_bits, const float* __restrict__ table, float* __restrict__ out) {
    const int lpr = 1 << lpr_bits, slots = 256 >> lpr_bits;
    const long long r = (long long)blockIdx.x * slots + (threadIdx.x >> lpr_bits);
    if (r >= w.rows) return;
    const int kind = w.row_kind[r], n = kind >= 0 && kind < w.kinds ? w.count(r) : 0;
    const float* row = table + (long long)(n > 0 ? kind : 0) * w.classes;
    for (int at = (threadIdx.x & (lpr - 1)) * V; at < w.width; at += lpr * V) {
        int c[V];
        float v[V];
        load_vec<V>(w.cand + r * w.width + at, c);
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = at + j < n ? w.cls_of(c[j]) : -1;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = c[j] >= 0 ? row[c[j]] : NOTHING;
        if constexpr (V == 4)
            *reinterpret_cast<float4*>(out + r * w.width + at) = make_float4(v[0], v[1], v[2], v[3]);
        else
            out[r * w.width + at] = v[0];
    }
}

// Rows in the order of their kinds are dealt to blocks in runs of RUN; a run may hold rows of several kinds.  A block adds
// the gradients of one kind's rows into private columns acc[class][thread] in LDS - a thread's own additions, in order, no
// atomics - sums the columns in a fixed order in f64 when the kind ends, and writes the sum as partial number (block +
// kind): no two (block, kind) pairs that occur share it.  A column is f32: a thread adds some 16 values of a run for rows
// to 512 places and width / 32 for wider ones (4,096 at 131,072; with more than 128 classes, on fewer threads, as many times more),
// each addition off by half a step at most; 256 columns of 128 classes in f64 would not fit LDS.
// A run holds about 4096 places: enough that the columns' sums at its end weigh little, few enough that there are several
// blocks for every CU.  100,000 x 64, 9 kinds of 9 classes: 51 MB in 22 us (2.3 TB/s); 26,279 x 512, 99 kinds: 108 MB in 34 us
// (3.2 TB/s): the dependent trip from candidate to class, and a read-add-write of LDS a place.
static int run_rows(int64_t width) { return width >= 512 ? 8 : width <= 64 ? 64 : (int)(4096 / width); }

template <int V>
__global__ __launch_bounds__(256) void k_class_scores_bwd(Windows w, int run, int lpr_bits, const float* __restrict__ grad, double* __restrict__ partial) {
    extern __shared__ float acc[];          // [classes][threads]
    const int t = threadIdx.x, threads = blockDim.x, lpr = 1 << lpr_bits, slots = threads >> lpr_bits;
    const long long p0 = (long long)blockIdx.x * run, p1 = min(p0 + run, w.rows);
    for (int i = t; i < w.classes * threads; i += threads) acc[i] = 0.0f;
    __syncthreads();
    long long p = p0;
    while (p < p1) {
        const int kind = w.kind_at(p);
        if (kind < 0) {
            ++p;
            continue;
        }
        const long long end = min(max((long long)w.kind_start[kind + 1], p + 1), p1);      // (ends whatever the array holds)
        for (long long at_row = p + (t >> lpr_bits); at_row < end; at_row += slots) {
            const int r = w.by_kind[at_row];
            if (r < 0 || r >= w.rows) continue;
            const int n = w.count(r);
            const long long first = (long long)r * w.width;
            for (int at = (t & (lpr - 1)) * V; at < n; at += lpr * V) {
                int c[V];
                float g[V];
                load_vec<V>(w.cand + first + at, c);
                load_vec<V>(grad + first + at, g);
#pragma unroll
                for (int j = 0; j < V; ++j) c[j] = at + j < n ? w.cls_of(c[j]) : -1;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (c[j] >= 0) acc[c[j] * threads + t] += g[j];
            }
        }
        p = end;
        __syncthreads();
        const int lane = t & 63, waves = (threads + 63) >> 6;
        for (int c = t >> 6; c < w.classes; c += waves) {
            double s = 0.0;
            for (int j = lane; j < threads; j += 64) {
                s += (double)acc[c * threads + j];
                acc[c * threads + j] = 0.0f;
            }
            for (int o = 32; o; o >>= 1) {
                const double other = __shfl_down(s, o);
                s += lane + o < threads ? other : 0.0;
            }
            if (lane == 0) partial[((long long)blockIdx.x + kind) * w.classes + c] = s;
        }
        __syncthreads();
    }
}

// A block a kind: class c of every groups-th partial by a thread, the groups' sums in order.  4 to 5 us, a launch and a chain.
__global__ __launch_bounds__(256) void k_class_scores_finish(Windows w, int run, int cp_bits, const double* __restrict__ partial, float* __restrict__ d_table) {
    __shared__ double red[256];
    const int kind = blockIdx.x, cp = 1 << cp_bits, groups = 256 >> cp_bits, g = threadIdx.x >> cp_bits;
    const long long s = max(w.kind_start[kind], 0), e = min((long long)w.kind_start[kind + 1], w.rows);
    for (int c0 = 0; c0 < w.classes; c0 += cp) {
        const int c = c0 + (threadIdx.x & (cp - 1));
        double sum = 0.0;
        if (e > s && c < w.classes)
            for (long long b = s / run + g; b <= (e - 1) / run; b += groups) sum += partial[(b + kind) * w.classes + c];
        red[threadIdx.x] = sum;
        __syncthreads();
        if (g == 0 && c < w.classes) {
            for (int j = 1; j < groups; ++j) sum += red[(j << cp_bits) + threadIdx.x];
            d_table[(long long)kind * w.classes + c] = (float)sum;
        }
        __syncthreads();
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

static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
// lanes a row (a power of two, as its logarithm): enough for the row's vectors, at most 2^most
static int lanes_a_row(int64_t width, int per_lane, int most) {
    int bits = 0;
    while (bits < most && ((int64_t)per_lane << bits) < width) ++bits;
    return bits;
}

// a launch has fewer than 2^32 threads
static int check_launch(const char* what, const aig_score_windows* w, int64_t blocks, int64_t threads) {
    if (blocks * threads >= (1ll << 32))
        return fail(AIG_ELIMIT, "%s: %lld rows of %lld take %lld threads: fewer than 2^32 fit a launch", what, (long long)w->rows,
                    (long long)w->width, (long long)(blocks * threads));
    return AIG_OK;
}

extern "C" int aig_class_scores(const aig_score_windows* w, const float* table, float* out, void* stream) {
    if (const int rc = check_windows("aig_class_scores", w)) return rc;
    if (w->rows == 0) return AIG_OK;
    AIG_REQUIRE(table && out, "aig_class_scores: null pointer");
    const bool vec = w->width % 4 == 0 && aligned16(w->cand) && aligned16(out);
    const int bits = lanes_a_row(w->width, vec ? 4 : 1, 8);
    const int64_t per_block = 256 >> bits;
    const int64_t blocks = (w->rows + per_block - 1) / per_block;
    if (const int rc = check_launch("aig_class_scores", w, blocks, 256)) return rc;
    const dim3 grid((unsigned)blocks);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (vec) hipLaunchKernelGGL(k_class_scores<4>, grid, dim3(256), 0, s, windows_of(w), bits, table, out);
    else hipLaunchKernelGGL(k_class_scores<1>, grid, dim3(256), 0, s, windows_of(w), bits, table, out);
    AIG_LAUNCH_CHECK();
    return AIG_OK;
}

extern "C" size_t aig_class_scores_bwd_ws_bytes(int64_t rows, int64_t width, int64_t kinds, int64_t classes) {
    if (rows < 0 || width < 1 || kinds < 1 || classes < 1) return 0;
    return align_up((size_t)((rows + run_rows(width) - 1) / run_rows(width) + kinds) * (size_t)classes * sizeof(double));
}

extern "C" int aig_class_scores_bwd(const aig_score_windows* w, const float* grad, float* d_table, void* ws, size_t ws_bytes, void* stream) {
    if (const int rc = check_windows("aig_class_scores_bwd", w)) return rc;
    const int run = run_rows(w->width), threads = w->classes <= 128 ? 256 : w->classes <= 512 ? 64 : 32;      // columns of at most 128 KB
    const int64_t blocks = (w->rows + run - 1) / run;
    if (const int rc = check_launch("aig_class_scores_bwd", w, blocks, threads)) return rc;
    AIG_REQUIRE(d_table && (w->rows == 0 || (grad && w->by_kind)) && w->kind_start, "aig_class_scores_bwd: null pointer");
    if (!ws || ws_bytes < aig_class_scores_bwd_ws_bytes(w->rows, w->width, w->kinds, w->classes))
        return fail(AIG_EWORKSPACE, "aig_class_scores_bwd: workspace of %zu bytes is too small", ws_bytes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    double* partial = static_cast<double*>(ws);
    const size_t lds = (size_t)w->classes * threads * sizeof(float);
    if (w->rows) {
        const bool vec = w->width % 4 == 0 && aligned16(w->cand) && aligned16(grad);
        const int bits = lanes_a_row(w->width, vec ? 4 : 1, threads == 256 ? 8 : threads == 64 ? 6 : 5);
        const dim3 grid((unsigned)blocks);
        AIG_HIP_CHECK(ensure_dynamic_lds(vec ? reinterpret_cast<const void*>(k_class_scores_bwd<4>) : reinterpret_cast<const void*>(k_class_scores_bwd<1>), lds));
        if (vec) hipLaunchKernelGGL(k_class_scores_bwd<4>, grid, dim3(threads), lds, s, windows_of(w), run, bits, grad, partial);
        else hipLaunchKernelGGL(k_class_scores_bwd<1>, grid, dim3(threads), lds, s, windows_of(w), run, bits, grad, partial);
    }
    int cp_bits = 0;
    while (cp_bits < 8 && (1 << cp_bits) < w->classes) ++cp_bits;
    hipLaunchKernelGGL(k_class_scores_finish, dim3((unsigned)w->kinds), dim3(256), 0, s, windows_of(w), run, cp_bits, partial, d_table);
    AIG_LAUNCH_CHECK();
    return AIG_OK;
}
