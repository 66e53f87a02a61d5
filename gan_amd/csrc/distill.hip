// Distillation from a teacher's top logits: the loss of each row of a student's logits, its gradient, and both in one pass.
#include "rows.h"

namespace aig {
namespace {
using namespace rows;

// Row r: y = l / T over the row's valid places, p = softmax(y); the teacher's listed places i_j with logits t_j,
//   q_j = exp(t_j / T - lse), lse = the teacher's own log-sum-exp (tail) or that of the listed entries
//   loss = w T^2 [ sum_j q_j (log q_j - log p[i_j]) + q_R (log q_R - log p_R) ]
//   dloss/dl_i = w T [ p_i (sum_j q_j + q_R - [i in R] q_R / p_R) - sum over j with i_j = i of q_j ]
// R: the valid places that are not listed, q_R = 1 - sum_j q_j (tail; 0 otherwise, and where R is empty).
struct DistillArgs {
    long long rows, ld, grad_ld;
    int width, m, vec, grad_vec;
    float temperature;
    const int* counts;
    const float *values, *lse, *weight;
    const int* index;
    const float* upstream;       // factor of the gradient: one (stride 0) or one a row, or none
    long long upstream_stride;
    float* loss;                 // may be null
    __device__ __forceinline__ int count(long long r) const { return counts ? min(max(counts[r], 0), width) : width; }
    // whether entry j of the teacher's row names a place of the student's (absent entries: -1, or a logit of -inf)
    __device__ __forceinline__ bool names(long long r, int j, int n) const {
        const int i = index[r * m + j];
        return i >= 0 && i < n && !(values[r * m + j] == -__builtin_inff());
    }
};

// Exponentials in base 2.  An argument of -d carries an error of d 2^-23, its exponential one of d 2^-d 2^-23 relative to the
// row's largest: nowhere more than 2^-23.
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }
constexpr float LN2F = 0.69314718056f;
__device__ __forceinline__ float probability(float log_q) { return log_q > 0.0f ? 1.0f : expf(log_q); }      // (NaN stays NaN)

// A listed entry's probability is added to its place in LDS as a whole number of 2^-30: entries that name one place twice
// add up to the same bits in any order.
constexpr float Q_UNIT = 1073741824.0f;

template <typename T, int G, int E, bool LOSS, bool GRAD>
__global__ __launch_bounds__(256) void k_distill(const T* __restrict__ x, T* __restrict__ grad, DistillArgs a) {
    constexpr int ROWS = 256 / G, WORDS = (G * E + 31) / 32;
    __shared__ unsigned listed_bits[ROWS][WORDS];
    __shared__ unsigned listed_q[GRAD ? ROWS : 1][GRAD ? G * E : 1];
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / G;
    if (r >= a.rows) return;
    const int lane = threadIdx.x & (G - 1), slot = threadIdx.x / G;
    unsigned* bits = listed_bits[slot];
    unsigned* qsum = listed_q[GRAD ? slot : 0];
    for (int w = lane; w < WORDS; w += G) bits[w] = 0;
    if (GRAD)
        for (int i = lane; i < G * E; i += G) qsum[i] = 0;

    const int n = a.count(r);
    x += r * a.ld;
    float v[E];
    load_values<T, E>(x, n, a.width, a.vec, lane, v);
    float top = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, v[e]);
    top = all<G>(top, Max());
    const float inv_t = 1.0f / a.temperature, per = (float)LOG2E * inv_t;
    const float base = top > -__builtin_inff() ? top : 0.0f;
    float ex[E];
    double z = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        ex[e] = exp2_fast((v[e] - base) * per);
        z += (double)ex[e];
    }
    z = all<G>(z, Add());
    const float logz = logf((float)z);

    // the teacher's entries: the log-sum-exp of those that name a place of this row, where none is given
    float lse = 0.0f;
    int named = 0;
    if (a.lse) {
        lse = a.lse[r];
        for (int j = lane; j < a.m; j += G) {
            named += a.names(r, j, n);
        }
    } else {
        float tm = -__builtin_inff();
        for (int j = lane; j < a.m; j += G) {
            const bool in = a.names(r, j, n);
            named += in;
            tm = in ? fmaxf(tm, a.values[r * a.m + j]) : tm;
        }
        tm = all<G>(tm, Max());
        float s = 0.0f;
        for (int j = lane; j < a.m; j += G) {
            if (a.names(r, j, n)) s += exp2_fast((a.values[r * a.m + j] - tm) * per);
        }
        lse = tm * inv_t + logf(all<G>(s, Add()));
    }
    named = all<G>(named, Add());
    const bool live = z != 0.0 && named > 0;        // (a NaN among the logits is not nothing: it shows in the loss)

    float sum_q = 0.0f, l = 0.0f;
    for (int j = lane; j < a.m; j += G) {
        if (!a.names(r, j, n)) continue;
        const int i = a.index[r * a.m + j];
        const float lq = a.values[r * a.m + j] * inv_t - lse, q = probability(lq);
        sum_q += q;
        atomicOr(&bits[i >> 5], 1u << (i & 31));
        if (GRAD) atomicAdd(&qsum[i], (unsigned)__float2int_rn(q * Q_UNIT));
        if (LOSS && q > 0.0f) l += q * (lq - ((as_float(x[i]) - base) * inv_t - logz));
    }
    sum_q = all<G>(sum_q, Add());
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();

    // the places that are not listed
    double rest = 0.0;
    float rest_top = -__builtin_inff();
    unsigned mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int i = lane * E + e;
        const bool in = (bits[i >> 5] >> (i & 31)) & 1u;
        mine |= (unsigned)in << e;
        rest += in ? 0.0 : (double)ex[e];
        rest_top = in ? rest_top : fmaxf(rest_top, v[e]);
    }
    rest = all<G>(rest, Add());
    rest_top = all<G>(rest_top, Max());
    const float rest_q = a.lse && rest_top > -__builtin_inff() ? fmaxf(1.0f - sum_q, 0.0f) : 0.0f;
    // (their sum may be too small for f32 beside the largest place: then beside their own largest)
    float shift = 0.0f;
    if (rest_q > 0.0f && rest < 1e-30) {
        shift = (base - rest_top) * per;
        rest = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) rest += (mine >> e) & 1u ? 0.0 : (double)exp2_fast((v[e] - rest_top) * per);
        rest = all<G>(rest, Add());
    }
    const float scale = a.temperature * a.temperature * (a.weight ? a.weight[r] : 1.0f);
    if (LOSS) {
        l = all<G>(l, Add());
        if (rest_q > 0.0f) l += rest_q * (logf(rest_q) - (logf((float)rest) - shift * LN2F - logz));
        if (lane == 0) a.loss[r] = live ? scale * l : 0.0f;
    }
    if (GRAD) {
        const float up = a.upstream ? a.upstream[r * a.upstream_stride] : 1.0f;
        const float c = live ? scale * inv_t * up : 0.0f, inv_z = 1.0f / (float)z, inv_rest = rest_q > 0.0f ? rest_q / (float)rest : 0.0f;
        grad += r * a.grad_ld;
        T g[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = lane * E + e;
            const float p = ex[e] * inv_z;
            float d = p * (sum_q + rest_q);
            if ((mine >> e) & 1u)
                d -= (float)qsum[i] * (1.0f / Q_UNIT);
            else
                d -= (shift > 0.0f ? exp2_fast((v[e] - rest_top) * per) : ex[e]) * inv_rest;
            g[e] = from_float<T>(i < n && live ? c * d : 0.0f);
        }
        typedef Places<T, E> P;
        if (a.grad_vec && lane * E + E <= a.width) {
            union { typename P::word w[E / P::PER]; T t[E]; } u;
#pragma unroll
            for (int e = 0; e < E; ++e) u.t[e] = g[e];
#pragma unroll
            for (int j = 0; j < E / P::PER; ++j) reinterpret_cast<typename P::word*>(grad + lane * E)[j] = u.w[j];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (lane * E + e < a.width) grad[lane * E + e] = g[e];
        }
    }
}

// ---------------------------------------------------------------- wide rows: a workgroup per row
constexpr int WIDE_T = 1024;

template <typename V, typename OP> __device__ __forceinline__ V block_all(V v, OP op, double* red) {
    V* s = reinterpret_cast<V*>(red);
    v = all<64>(v, op);
    __syncthreads();
    if (lane_id() == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    V t = s[0];
#pragma unroll
    for (int w = 1; w < WIDE_T / 64; ++w) t = op(t, s[w]);
    return t;
}

template <typename T, bool LOSS, bool GRAD>
__global__ __launch_bounds__(WIDE_T) void k_distill_wide(const T* __restrict__ x, T* __restrict__ grad, DistillArgs a) {
    __shared__ double red[WIDE_T / 64];
    __shared__ unsigned bits[MAX_WIDTH / 32];
    __shared__ int place[AIG_ROWS_MAX_TOP];
    __shared__ float prob[AIG_ROWS_MAX_TOP];
    const long long r = blockIdx.x;
    const int n = a.count(r), t = threadIdx.x;
    x += r * a.ld;
    for (int w = t; w < (n + 31) / 32; w += WIDE_T) bits[w] = 0;
    float top = -__builtin_inff();
    for (int i = t; i < n; i += WIDE_T) top = fmaxf(top, as_float(x[i]));
    top = block_all(top, Max(), red);
    const float inv_t = 1.0f / a.temperature, per = (float)LOG2E * inv_t;
    const float base = top > -__builtin_inff() ? top : 0.0f;

    // (at most AIG_ROWS_MAX_TOP entries: one a thread)
    int i_mine = -1;
    float v_mine = -__builtin_inff();
    if (t < a.m && a.names(r, t, n)) {
        i_mine = a.index[r * a.m + t];
        v_mine = a.values[r * a.m + t];
    }
    const int named = block_all((int)(i_mine >= 0), Add(), red);
    float lse;
    if (a.lse)
        lse = a.lse[r];
    else {
        const float tm = block_all(v_mine, Max(), red);
        lse = tm * inv_t + logf(block_all(i_mine >= 0 ? exp2_fast((v_mine - tm) * per) : 0.0f, Add(), red));
    }
    const float lq = v_mine * inv_t - lse, q = i_mine >= 0 ? probability(lq) : 0.0f;
    const float sum_q = block_all(q, Add(), red);
    if (t < AIG_ROWS_MAX_TOP) {
        place[t] = i_mine;
        prob[t] = q;
    }
    if (i_mine >= 0) atomicOr(&bits[i_mine >> 5], 1u << (i_mine & 31));
    __syncthreads();

    double z = 0.0, rest = 0.0;
    float rest_top = -__builtin_inff();
    for (int i = t; i < n; i += WIDE_T) {
        const float v = as_float(x[i]), ex = exp2_fast((v - base) * per);
        const bool in = (bits[i >> 5] >> (i & 31)) & 1u;
        z += (double)ex;
        rest += in ? 0.0 : (double)ex;
        rest_top = in ? rest_top : fmaxf(rest_top, v);
    }
    z = block_all(z, Add(), red);
    rest = block_all(rest, Add(), red);
    rest_top = block_all(rest_top, Max(), red);
    const bool live = z != 0.0 && named > 0;
    const float logz = logf((float)z);
    const float rest_q = a.lse && rest_top > -__builtin_inff() ? fmaxf(1.0f - sum_q, 0.0f) : 0.0f;
    float shift = 0.0f;
    if (rest_q > 0.0f && rest < 1e-30) {
        shift = (base - rest_top) * per;
        rest = 0.0;
        for (int i = t; i < n; i += WIDE_T)
            rest += (bits[i >> 5] >> (i & 31)) & 1u ? 0.0 : (double)exp2_fast((as_float(x[i]) - rest_top) * per);
        rest = block_all(rest, Add(), red);
    }
    const float scale = a.temperature * a.temperature * (a.weight ? a.weight[r] : 1.0f);
    if (LOSS) {
        float l = i_mine >= 0 && q > 0.0f ? q * (lq - ((as_float(x[i_mine]) - base) * inv_t - logz)) : 0.0f;
        l = block_all(l, Add(), red);
        if (rest_q > 0.0f) l += rest_q * (logf(rest_q) - (logf((float)rest) - shift * LN2F - logz));
        if (t == 0) a.loss[r] = live ? scale * l : 0.0f;
    }
    if (GRAD) {
        const float up = a.upstream ? a.upstream[r * a.upstream_stride] : 1.0f;
        const float c = live ? scale * inv_t * up : 0.0f, inv_z = 1.0f / (float)z, inv_rest = rest_q > 0.0f ? rest_q / (float)rest : 0.0f;
        grad += r * a.grad_ld;
        for (int i = t; i < a.width; i += WIDE_T) {
            float d = 0.0f;
            if (i < n && live) {
                if ((bits[i >> 5] >> (i & 31)) & 1u) continue;       // below
                const float v = as_float(x[i]), ex = exp2_fast((v - base) * per);
                d = c * (ex * inv_z * (sum_q + rest_q) - (shift > 0.0f ? exp2_fast((v - rest_top) * per) : ex) * inv_rest);
            }
            grad[i] = from_float<T>(d);
        }
        if (live && i_mine >= 0) {        // a listed place is written by the first entry that names it, for all of them
            float s = 0.0f;
            bool is_first = true;
            for (int j = 0; j < a.m; ++j)
                if (place[j] == i_mine) {
                    is_first = is_first && j >= t;
                    s += prob[j];
                }
            if (is_first) {
                const float p = exp2_fast((as_float(x[i_mine]) - base) * per) * inv_z;
                grad[i_mine] = from_float<T>(c * (p * (sum_q + rest_q) - s));
            }
        }
    }
}

// The sum of the rows' losses, in an order that the number of rows alone gives.
constexpr int SUM_T = 1024, SUM_BLOCKS = 256;
__global__ __launch_bounds__(SUM_T) void k_sum_rows(long long n, const float* __restrict__ v, double* __restrict__ partial,
                                                    const double* __restrict__ partial_in, float factor, float* __restrict__ out) {
    __shared__ double red[SUM_T / 64];
    double s = 0.0;
    if (partial_in)
        for (long long i = threadIdx.x; i < n; i += SUM_T) s += partial_in[i];
    else
        for (long long i = (long long)blockIdx.x * SUM_T + threadIdx.x; i < n; i += (long long)gridDim.x * SUM_T) s += (double)v[i];
    s = block_all(s, Add(), red);
    if (threadIdx.x == 0) {
        if (out)
            out[0] = (float)(s * (double)factor);
        else
            partial[blockIdx.x] = s;
    }
}

template <typename T, int G, int E> void launch_narrow(hipStream_t s, const T* x, T* grad, DistillArgs a) {
    const size_t align = E * sizeof(T) < 16 ? E * sizeof(T) : 16;
    a.vec = reinterpret_cast<uintptr_t>(x) % align == 0 && (a.ld * sizeof(T)) % align == 0;
    a.grad_vec = reinterpret_cast<uintptr_t>(grad) % align == 0 && (a.grad_ld * sizeof(T)) % align == 0;
    const dim3 grid((unsigned)((a.rows * G + 255) / 256));
    if (grad && a.loss) hipLaunchKernelGGL((k_distill<T, G, E, true, true>), grid, dim3(256), 0, s, x, grad, a);
    else if (grad) hipLaunchKernelGGL((k_distill<T, G, E, false, true>), grid, dim3(256), 0, s, x, grad, a);
    else hipLaunchKernelGGL((k_distill<T, G, E, true, false>), grid, dim3(256), 0, s, x, grad, a);
}

template <typename T> int distill(hipStream_t s, const T* x, T* grad, const DistillArgs& a) {
    if (a.width <= 64) launch_narrow<T, 16, 4>(s, x, grad, a);
    else if (a.width <= 256) launch_narrow<T, 16, 16>(s, x, grad, a);
    else if (a.width <= 512) launch_narrow<T, 64, 8>(s, x, grad, a);
    else if (a.width <= NARROW) launch_narrow<T, 64, 16>(s, x, grad, a);
    else {
        const dim3 grid((unsigned)a.rows);
        if (grad && a.loss) hipLaunchKernelGGL((k_distill_wide<T, true, true>), grid, dim3(WIDE_T), 0, s, x, grad, a);
        else if (grad) hipLaunchKernelGGL((k_distill_wide<T, false, true>), grid, dim3(WIDE_T), 0, s, x, grad, a);
        else hipLaunchKernelGGL((k_distill_wide<T, true, false>), grid, dim3(WIDE_T), 0, s, x, grad, a);
    }
    AIG_LAUNCH_CHECK();
    return AIG_OK;
}
}  // namespace
}  // namespace aig

using namespace aig;

extern "C" int aig_distill_rows(const aig_distill* d, float* loss, void* grad, int64_t grad_ld, const float* upstream,
                                int64_t upstream_stride, void* stream) {
    AIG_REQUIRE(d, "aig_distill_rows: null argument block");
    AIG_REQUIRE(d->rows >= 0 && d->width >= 1 && d->ld >= 0, "aig_distill_rows: bad sizes rows=%lld width=%lld ld=%lld",
                (long long)d->rows, (long long)d->width, (long long)d->ld);
    AIG_REQUIRE(d->dtype == AIG_F32 || d->dtype == AIG_F16 || d->dtype == AIG_BF16, "aig_distill_rows: unknown dtype %d", d->dtype);
    if (const int rc = check_row_limits("aig_distill_rows", d->rows, d->width)) return rc;
    AIG_REQUIRE(d->m >= 1 && d->m <= AIG_ROWS_MAX_TOP, "aig_distill_rows: m=%lld is not in 1..%d", (long long)d->m, AIG_ROWS_MAX_TOP);
    AIG_REQUIRE(d->temperature > 0.0f && d->temperature < __builtin_inff(), "aig_distill_rows: the temperature must be positive and finite");
    AIG_REQUIRE(!grad || grad_ld >= d->width, "aig_distill_rows: rows of the gradient overlap (grad_ld=%lld)", (long long)grad_ld);
    AIG_REQUIRE(upstream_stride == 0 || upstream_stride == 1, "aig_distill_rows: upstream_stride is 0 or 1");
    if (d->rows == 0) return AIG_OK;
    AIG_REQUIRE(loss || grad, "aig_distill_rows: nothing to compute");
    AIG_REQUIRE(d->logits && d->values && d->index, "aig_distill_rows: null pointer");
    DistillArgs a{};
    a.rows = d->rows; a.ld = d->ld; a.grad_ld = grad_ld; a.width = (int)d->width; a.m = (int)d->m; a.temperature = d->temperature;
    a.counts = d->counts; a.values = d->values; a.lse = d->lse; a.weight = d->weight; a.index = d->index;
    a.upstream = upstream; a.upstream_stride = upstream_stride; a.loss = loss;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (d->dtype == AIG_F32) return distill(s, static_cast<const float*>(d->logits), static_cast<float*>(grad), a);
    if (d->dtype == AIG_F16) return distill(s, static_cast<const __half*>(d->logits), static_cast<__half*>(grad), a);
    return distill(s, static_cast<const __hip_bfloat16*>(d->logits), static_cast<__hip_bfloat16*>(grad), a);
}

extern "C" size_t aig_sum_rows_ws_bytes(int64_t rows) { return rows > SUM_T * 8 ? SUM_BLOCKS * sizeof(double) : 0; }

extern "C" int aig_sum_rows(int64_t rows, const float* v, float factor, float* out, void* ws, size_t ws_bytes, void* stream) {
    AIG_REQUIRE(rows >= 0 && out && (v || rows == 0), "aig_sum_rows: bad argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (rows <= SUM_T * 8) {
        hipLaunchKernelGGL(k_sum_rows, dim3(1), dim3(SUM_T), 0, s, (long long)rows, v, nullptr, nullptr, factor, out);
    } else {
        if (ws_bytes < aig_sum_rows_ws_bytes(rows) || !ws) return fail(AIG_EWORKSPACE, "aig_sum_rows: workspace too small");
        double* partial = static_cast<double*>(ws);
        hipLaunchKernelGGL(k_sum_rows, dim3(SUM_BLOCKS), dim3(SUM_T), 0, s, (long long)rows, v, partial, nullptr, 1.0f, nullptr);
        hipLaunchKernelGGL(k_sum_rows, dim3(1), dim3(SUM_T), 0, s, (long long)SUM_BLOCKS, nullptr, nullptr, partial, factor, out);
    }
    AIG_LAUNCH_CHECK();
    return AIG_OK;
}
