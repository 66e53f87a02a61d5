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
    double per;                  // log2(e) / T
    float temperature, factor;
    const int* counts;
    const float *values, *lse, *weight;
    const int* index;
    const float* upstream;       // factor of the gradient: one (stride 0) or one a row, or none
    long long upstream_stride;
    float* loss;                 // may be null
    float* stats;                // [rows][STATS], wide rows: written with the loss, read for a gradient alone; may be null
    __device__ __forceinline__ int count(long long r) const { return counts ? min(max(counts[r], 0), width) : width; }
    __device__ __forceinline__ float scale(long long r) const { return temperature * temperature * factor * (weight ? weight[r] : 1.0f); }
    __device__ __forceinline__ float scale_of_gradient(long long r) const {
        return temperature * factor * (weight ? weight[r] : 1.0f) * (upstream ? upstream[r * upstream_stride] : 1.0f);
    }
};
// An entry of the teacher's row names a place of the student's (absent entries: place -1, or a logit of -inf).
__device__ __forceinline__ bool names(int i, float v, int n) { return i >= 0 && i < n && !(v == -__builtin_inff()); }

// Exponentials in base 2.  An argument of -d carries an error of d 2^-23, its exponential one of d 2^-d 2^-23 relative to the
// row's largest: nowhere more than 2^-23.  What is summed or subtracted (probabilities, logarithms) is held in f64: the loss is a
// small difference of numbers of the size of the logits, and the rest of a row a small difference from 1.
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }
constexpr double LN2 = 0.69314718055994531;
__device__ __forceinline__ float probability(double log2_q) { return log2_q > 0.0 ? 1.0f : exp2_fast((float)log2_q); }      // (NaN stays NaN)
// a sum over the rest of a row that is below this beside the row's largest place is taken again beside its own largest
constexpr double FAINT = 1e-30;

// A listed entry's probability is added to its place in LDS as a whole number of 2^-30, shifted up by one, or as 1 where that
// number is 0: entries that name one place twice add up to the same bits in any order, a place is listed where the sum is not
// 0, and an entry without probability (a masked place of the teacher's) adds none.  Only entries that repeat a place can add up
// to the 2 that 31 bits do not hold: where a row's entries come near it, they are added again in steps that their sum fits.
// (An entry is off by half a step, 256 of them by 4 half steps of f32 of the sum at most.)
constexpr float Q_UNIT = 1073741824.0f;
__device__ __forceinline__ unsigned units_of(float q, float unit) { return max((unsigned)__float2int_rn(q * unit) << 1, 1u); }

// A group of lanes per row, the row in registers, its listed places in LDS: the logits are read once, the gradient written once.
// Loss and gradient of 1,000,000 x 64 f32 with 8 entries each: 588 MB in 119 to 127 us, where a large copy takes 128: bound by
// memory.  26,279 x 512 bf16 with 32 entries: loss 21 us (34 MB, 1.6 TB/s), gradient 23.5 us (60 MB, 2.6 TB/s): bound by the
// latency of a row's chain - load, largest, sum, entries, rest - at eight waves a SIMD.  243 x 16: 2.8 us, a launch.
template <typename T, int G, int E, bool LOSS, bool GRAD>
__global__ __launch_bounds__(256) void k_distill(const T* __restrict__ x, T* __restrict__ grad, DistillArgs a) {
    constexpr int ROWS = 256 / G;
    __shared__ __attribute__((aligned(16))) float row_values[ROWS][G * E];
    __shared__ __attribute__((aligned(16))) unsigned row_listed[ROWS][G * E];
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / G;
    if (r >= a.rows) return;
    const int lane = threadIdx.x & (G - 1), slot = threadIdx.x / G;
    float* lv = row_values[slot];
    unsigned* listed = row_listed[slot];
    const int n = a.count(r);
    float v[E];
    load_values<T, E>(x + r * a.ld, n, a.width, a.vec, lane, v);
    const int* index = a.index + r * a.m;
    const float* values = a.values + r * a.m;
    const int i0 = lane < a.m ? index[lane] : -1;
    const float v0 = lane < a.m ? values[lane] : 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        lv[lane * E + e] = v[e];
        listed[lane * E + e] = 0;
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, v[e]);
    top = all<G>(top, Max());
    const float base = top > -__builtin_inff() ? top : 0.0f, per = (float)a.per;
    float ex[E];
    double z = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        ex[e] = exp2_fast((v[e] - base) * per);
        z += (double)ex[e];
    }
    z = all<G>(z, Add());

    // the teacher's log-sum-exp in base 2, or that of the entries
    double lse;
    if (a.lse) {
        lse = (double)a.lse[r] * LOG2E;
    } else {
        float tm = names(i0, v0, n) ? v0 : -__builtin_inff();
        for (int j = lane + G; j < a.m; j += G) tm = names(index[j], values[j], n) ? fmaxf(tm, values[j]) : tm;
        tm = all<G>(tm, Max());
        double s = names(i0, v0, n) ? (double)exp2_fast((v0 - tm) * per) : 0.0;
        for (int j = lane + G; j < a.m; j += G) s += names(index[j], values[j], n) ? (double)exp2_fast((values[j] - tm) * per) : 0.0;
        lse = (double)tm * a.per + log2_of(all<G>(s, Add()));
    }
    // (sum_q counts the entries along, NAMED each: at most 256 of at most 1 stay below it, and 2^-34 is left of its steps)
    constexpr double NAMED = 1024.0;
    double sum_q = 0.0, l = 0.0;
    auto entry = [&](int i, float t) {
        if (!names(i, t, n)) return;
        const double lq = (double)t * a.per - lse;
        const float q = probability(lq);
        sum_q += NAMED + (double)q;
        if (GRAD) atomicAdd(&listed[i], units_of(q, Q_UNIT));
        else listed[i] = 1u;
        if (LOSS) l += q > 0.0f ? (double)q * (lq - ((double)lv[i] - (double)base) * a.per) : q == 0.0f ? 0.0 : (double)q;
    };
    entry(i0, v0);
    for (int j = lane + G; j < a.m; j += G) entry(index[j], values[j]);
    sum_q = all<G>(sum_q, Add());
    const bool live = z != 0.0 && sum_q != 0.0;        // (a NaN among the logits is not nothing: it shows in the loss)
    sum_q -= NAMED * __builtin_floor(sum_q * (1.0 / NAMED));
    float q_step = 1.0f / Q_UNIT;
    if (GRAD && sum_q >= 1.75) {
        const int e2 = __builtin_amdgcn_frexp_exp((float)sum_q);      // (the sum is below 2^e2, which is at most 512)
        q_step = ldexpf(1.0f, e2 - 30);
#pragma unroll
        for (int e = 0; e < E; ++e) listed[lane * E + e] = 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
        for (int j = lane; j < a.m; j += G)
            if (names(index[j], values[j], n))
                atomicAdd(&listed[index[j]], units_of(probability((double)values[j] * a.per - lse), ldexpf(1.0f, 30 - e2)));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();

    // the places that are not listed
    unsigned q_here[E];
    double rest = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q_here[e] = listed[lane * E + e];
        rest += q_here[e] ? 0.0 : (double)ex[e];
    }
    rest = all<G>(rest, Add());
    float rest_q = a.lse ? (float)fmax(1.0 - sum_q, 0.0) : 0.0f;
    float rest_top = base;
    if (a.lse && rest < FAINT) {
        rest_top = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < E; ++e) rest_top = q_here[e] ? rest_top : fmaxf(rest_top, v[e]);
        rest_top = all<G>(rest_top, Max());
        if (!(rest_top > -__builtin_inff())) rest_q = 0.0f;
        rest = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) rest += q_here[e] || rest_q == 0.0f ? 0.0 : (double)exp2_fast((v[e] - rest_top) * per);
        rest = all<G>(rest, Add());
    }
    const bool faint = rest_q > 0.0f && rest_top != base;
    if (LOSS) {
        l = all<G>(l, Add());
        // three logarithms at once, one in each of three lanes of every four
        const bool some = rest_q > 0.0f;
        const double of = (lane & 3) == 0 ? z : !some ? 1.0 : (lane & 3) == 1 ? rest : (double)rest_q;
        const double lg = log2_of(of), logz = dpp<0x00>(lg), log_rest = dpp<0x55>(lg), log_rest_q = dpp<0xAA>(lg);
        l += sum_q * logz;
        if (some) l += (double)rest_q * (log_rest_q - log_rest + logz - ((double)rest_top - (double)base) * a.per);
        if (lane == 0) a.loss[r] = live ? (float)((double)a.scale(r) * LN2 * l) : 0.0f;
    }
    if (GRAD) {
        const float c = live ? a.scale_of_gradient(r) : 0.0f, full = ((float)sum_q + rest_q) * __builtin_amdgcn_rcpf((float)z),
                    outside = rest_q > 0.0f ? rest_q * __builtin_amdgcn_rcpf((float)rest) : 0.0f;
        T g[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float d = faint && !q_here[e] ? exp2_fast((v[e] - rest_top) * per) : ex[e];
            d = q_here[e] ? (float)(q_here[e] >> 1) * q_step : d * outside;
            g[e] = from_float<T>(lane * E + e < n && live ? c * (ex[e] * full - d) : 0.0f);
        }
        grad += r * a.grad_ld;
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
constexpr int WIDE_T = 1024, STATS = 8;

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

// two sums over the workgroup at once
__device__ __forceinline__ void block_sums(double& a, double& b, double* red) {
    a = all<64>(a, Add());
    b = all<64>(b, Add());
    __syncthreads();
    if (lane_id() == 0) {
        red[threadIdx.x >> 6] = a;
        red[WIDE_T / 64 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = red[0];
    b = red[WIDE_T / 64];
#pragma unroll
    for (int w = 1; w < WIDE_T / 64; ++w) {
        a += red[w];
        b += red[WIDE_T / 64 + w];
    }
}

// One pass over the row for the largest place, the sum of exponentials and that of the places that are not listed (each
// thread beside its own largest so far), a second one for the gradient.  Listed places are a bitmap in LDS, shifted so that a
// vector's bits are one byte of it (f32: half a byte).  512 x 32,001 bf16, two rows a CU: loss 17.3 us (33 MB, 1.9 TB/s), its
// gradient from the sums that the loss left 27 us (66 MB, 2.4 TB/s): a row's reductions over sixteen waves, nine barriers, stand
// between its passes, and two workgroups a CU hide them in part.
template <typename T, bool LOSS, bool GRAD>
__global__ __launch_bounds__(WIDE_T) void k_distill_wide(const T* __restrict__ x, T* __restrict__ grad, DistillArgs a) {
    constexpr int PER = Span<T>::PER;
    __shared__ double red[2 * (WIDE_T / 64)];
    __shared__ unsigned bits[MAX_WIDTH / 32 + 1];
    __shared__ int place[AIG_ROWS_MAX_TOP];
    __shared__ float prob[AIG_ROWS_MAX_TOP];
    const long long r = blockIdx.x;
    const int n = a.count(r), t = threadIdx.x;
    x += r * a.ld;
    const Span<T> row(x, n);
    const int pad = (PER - row.head) & (PER - 1);
    auto listed = [&](int i) { return bits[(i + pad) >> 5] >> ((i + pad) & 31); };      // bit 0: place i, bits 1 .. PER-1: the next ones of its vector
    for (int w = t; w < (n + pad + 31) / 32; w += WIDE_T) bits[w] = 0;
    const float per = (float)a.per;

    // (at most AIG_ROWS_MAX_TOP entries: one a thread)
    int i_mine = -1;
    float v_mine = -__builtin_inff();
    if (t < a.m) {
        const int i = a.index[r * a.m + t];
        const float v = a.values[r * a.m + t];
        if (names(i, v, n)) {
            i_mine = i;
            v_mine = v;
        }
    }
    typename Span<T>::Batch ahead{};
    if (LOSS) ahead = row.fetch(t, WIDE_T);       // (on its way under the entries' sums; a gradient alone reads the row behind them)
    __syncthreads();
    if (i_mine >= 0) atomicOr(&bits[(i_mine + pad) >> 5], 1u << ((i_mine + pad) & 31));
    double lse;
    if (a.lse) {
        lse = (double)a.lse[r] * LOG2E;
    } else {
        const float tm = block_all(v_mine, Max(), red);
        lse = (double)tm * a.per + log2_of(block_all(i_mine >= 0 ? (double)exp2_fast((v_mine - tm) * per) : 0.0, Add(), red));
    }
    const double lq = (double)v_mine * a.per - lse;
    const float q = i_mine >= 0 ? probability(lq) : 0.0f;
    if (GRAD && t < AIG_ROWS_MAX_TOP) {
        place[t] = i_mine;
        prob[t] = q;
    }
    double sum_q = (double)q, named = i_mine >= 0 ? 1.0 : 0.0;
    block_sums(sum_q, named, red);        // (its barriers are also those between the bitmap's writers and its readers)

    float top, rest_top;
    double z, rest;
    const bool known = GRAD && !LOSS && a.stats;
    if (known) {
        const float* s = a.stats + r * STATS;
        top = s[0];
        rest_top = s[1];
        z = *reinterpret_cast<const double*>(s + 2);
        rest = *reinterpret_cast<const double*>(s + 4);
    } else {
        float mine = -__builtin_inff();
        z = rest = 0.0;
        row.each(t, WIDE_T, LOSS ? ahead : row.fetch(t, WIDE_T), [&](int i, const float (&v)[PER], int count) {
            float here = v[0];
            for (int j = 1; j < PER; ++j) here = j < count ? fmaxf(here, v[j]) : here;
            if (here > mine) {
                const double shrink = mine > -__builtin_inff() ? (double)exp2_fast((mine - here) * per) : 0.0;
                z *= shrink;
                rest *= shrink;
                mine = here;
            }
            const float base = mine > -__builtin_inff() ? mine : 0.0f;
            const unsigned in = listed(i);
            float s = 0.0f, u = 0.0f;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const float e = j < count ? exp2_fast((v[j] - base) * per) : 0.0f;
                s += e;
                u += (in >> j) & 1u ? 0.0f : e;
            }
            z += (double)s;
            rest += (double)u;
        });
        top = block_all(mine, Max(), red);
        const float shrink = mine > -__builtin_inff() ? exp2_fast((mine - top) * per) : 1.0f;      // (1: keeps a NaN)
        z *= (double)shrink;
        rest *= (double)shrink;
        block_sums(z, rest, red);
        rest_top = top;
        if (a.lse && rest < FAINT) {
            float u = -__builtin_inff();
            for (int i = t; i < n; i += WIDE_T) u = listed(i) & 1u ? u : fmaxf(u, as_float(x[i]));
            rest_top = block_all(u, Max(), red);
            double s = 0.0;
            if (rest_top > -__builtin_inff())
                for (int i = t; i < n; i += WIDE_T) s += listed(i) & 1u ? 0.0 : (double)exp2_fast((as_float(x[i]) - rest_top) * per);
            rest = block_all(s, Add(), red);
        }
        if (LOSS && a.stats && t == 0) {
            float* s = a.stats + r * STATS;
            s[0] = top;
            s[1] = rest_top;
            *reinterpret_cast<double*>(s + 2) = z;
            *reinterpret_cast<double*>(s + 4) = rest;
        }
    }
    const float base = top > -__builtin_inff() ? top : 0.0f;
    const bool live = z != 0.0 && named > 0.0;
    const float rest_q = a.lse && rest_top > -__builtin_inff() ? (float)fmax(1.0 - sum_q, 0.0) : 0.0f;
    const bool faint = rest_q > 0.0f && rest_top != top;
    if (LOSS) {
        double l = 0.0;
        if (i_mine >= 0) l = q > 0.0f ? (double)q * (lq - ((double)as_float(x[i_mine]) - (double)base) * a.per) : q == 0.0f ? 0.0 : (double)q;
        l = block_all(l, Add(), red);
        if (t == 0) {
            const double logz = log2_of(z);
            l += sum_q * logz;
            if (rest_q > 0.0f) l += (double)rest_q * (log2_of((double)rest_q / rest) + logz - ((double)rest_top - (double)base) * a.per);
            a.loss[r] = live ? (float)((double)a.scale(r) * LN2 * l) : 0.0f;
        }
    }
    if (GRAD) {
        const float c = live ? a.scale_of_gradient(r) : 0.0f, full = (float)((sum_q + (double)rest_q) / z),
                    outside = rest_q > 0.0f ? (float)((double)rest_q / rest) : 0.0f;
        grad += r * a.grad_ld;
        const bool vec = ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(x)) & 15) == 0;
        auto slope = [&](float v) {
            const float e = exp2_fast((v - base) * per);
            return c * (e * full - (faint ? exp2_fast((v - rest_top) * per) : e) * outside);
        };
        if (live)
            row.each(t, WIDE_T, [&](int i, const float (&v)[PER], int count) {
                const unsigned in = listed(i) & ((1u << count) - 1u);
                if (vec && count == PER && in == 0u) {
                    union { uint4 w; T t[PER]; } u;
#pragma unroll
                    for (int j = 0; j < PER; ++j) u.t[j] = from_float<T>(slope(v[j]));
                    *reinterpret_cast<uint4*>(grad + i) = u.w;
                } else {
                    for (int j = 0; j < PER; ++j)
                        if (j < count && !((in >> j) & 1u)) grad[i + j] = from_float<T>(slope(v[j]));       // (listed places: below)
                }
            });
        for (int i = (live ? n : 0) + t; i < a.width; i += WIDE_T) grad[i] = from_float<T>(0.0f);
        if (live && i_mine >= 0) {        // a listed place is written by the first entry that names it, for all of them
            double s = 0.0;
            bool is_first = true;
            for (int j = 0; j < a.m; ++j)
                if (place[j] == i_mine) {
                    is_first = is_first && j >= t;
                    s += (double)prob[j];
                }
            if (is_first) grad[i_mine] = from_float<T>(c * (exp2_fast((as_float(x[i_mine]) - base) * per) * full - (float)s));
        }
    }
}

// The sum of the rows' losses, in an order that the number of rows alone gives.  26,279 rows: 3 us in one launch (105 KB by one
// CU); more than 32,768 take a second one.
constexpr int SUM_T = 1024, SUM_BLOCKS = 256, SUM_ONE = 32 * SUM_T;      // (up to SUM_ONE rows: one block, one launch)
__global__ __launch_bounds__(SUM_T) void k_sum_rows(long long n, const float* __restrict__ v, double* __restrict__ partial,
                                                    const double* __restrict__ partial_in, float factor, float* __restrict__ out) {
    __shared__ double red[SUM_T / 64];
    double s = 0.0;
    if (partial_in) {
        for (long long i = threadIdx.x; i < n; i += SUM_T) s += partial_in[i];
    } else {
#pragma unroll 8
        for (long long i = (long long)blockIdx.x * SUM_T + threadIdx.x; i < n; i += (long long)gridDim.x * SUM_T) s += (double)v[i];
    }
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
    if (a.width <= 16) launch_narrow<T, 4, 4>(s, x, grad, a);
    else if (a.width <= 64) launch_narrow<T, 8, 8>(s, x, grad, a);
    else if (a.width <= 256) launch_narrow<T, 16, 16>(s, x, grad, a);
    else if (a.width <= 512) launch_narrow<T, 64, 8>(s, x, grad, a);
    else if (a.width <= NARROW) launch_narrow<T, 64, 16>(s, x, grad, a);
    else if (in_registers(a.rows, a.width)) launch_narrow<T, 64, 32>(s, x, grad, a);
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
    AIG_REQUIRE(d->temperature >= 1e-6f && d->temperature <= 1e6f, "aig_distill_rows: the temperature %g is not in 1e-6..1e6", (double)d->temperature);
    AIG_REQUIRE(!grad || grad_ld >= d->width, "aig_distill_rows: rows of the gradient overlap (grad_ld=%lld)", (long long)grad_ld);
    AIG_REQUIRE(upstream_stride == 0 || upstream_stride == 1, "aig_distill_rows: upstream_stride is 0 or 1");
    if (d->rows == 0) return AIG_OK;
    AIG_REQUIRE(loss || grad, "aig_distill_rows: nothing to compute");
    AIG_REQUIRE(d->logits && d->values && d->index, "aig_distill_rows: null pointer");
    DistillArgs a{};
    a.rows = d->rows; a.ld = d->ld; a.grad_ld = grad_ld; a.width = (int)d->width; a.m = (int)d->m;
    a.temperature = d->temperature; a.factor = d->scale;
    a.per = rows::LOG2E / (double)d->temperature;
    a.stats = d->stats;
    a.counts = d->counts; a.values = d->values; a.lse = d->lse; a.weight = d->weight; a.index = d->index;
    a.upstream = upstream; a.upstream_stride = upstream_stride; a.loss = loss;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (d->dtype == AIG_F32) return distill(s, static_cast<const float*>(d->logits), static_cast<float*>(grad), a);
    if (d->dtype == AIG_F16) return distill(s, static_cast<const __half*>(d->logits), static_cast<__half*>(grad), a);
    return distill(s, static_cast<const __hip_bfloat16*>(d->logits), static_cast<__hip_bfloat16*>(grad), a);
}

extern "C" size_t aig_sum_rows_ws_bytes(int64_t rows) { return rows > SUM_ONE ? SUM_BLOCKS * sizeof(double) : 0; }

extern "C" int aig_sum_rows(int64_t rows, const float* v, float factor, float* out, void* ws, size_t ws_bytes, void* stream) {
    AIG_REQUIRE(rows >= 0 && out && (v || rows == 0), "aig_sum_rows: bad argument");
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (rows <= SUM_ONE) {
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
