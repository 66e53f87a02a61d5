// Rows of logits: what the kernels on them share (rows.hip, distill.hip).  A row is held by a GROUP of 4 to 64 lanes, lane L
// of which owns the E consecutive places L*E .. L*E + E - 1 in registers, so that an order by place is an order by lane: one
// scan over the group's lanes orders everything.  What is done once a row - sums and scans over its lanes, draws - is done for
// the 64 / G rows of a wave at once, which speaks for few lanes of many places; registers, and the time that the last wave
// takes alone, speak for many lanes of few.  Measured, 64 places on 4 lanes of 16, 8 of 8 and 16 of 4: sampling 100,000 rows
// 24.4 us and 22.8 (a sort over 16 lanes is not built), loss and gradient of 1,000,000 rows 140, 135 and 158.  256 places on 16
// lanes of 16 and 64 of 4: loss and gradient of 150,000 rows 80 and 104.  512 places on 64 lanes of 8 and 16 of 32: loss and
// gradient of 50,000 rows 47 and 65, sampling 96 and 99, and of a single row 5.1 and 10.2.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace aig {
namespace rows {

constexpr int MAX_WIDTH = AIG_ROWS_MAX_WIDTH;
constexpr int NARROW = 1024;            // rows up to this width are held by a group's registers
// Wider ones have a workgroup each, but for rows to 2048 places that are more than the workgroups the chip holds at a time: 32
// places a lane then, a wave a row.  4,000 x 2,000 in registers and by workgroups: top-p 37 and 202 us, top-k 50 36 and 145, top 16
// 15 and 60, loss and gradient 31 and 106; 512 rows 16 and 28, 23 and 20, 9 and 9, 10 and 16; 64 rows 16 and 14, 9 and 11, 9 and 5,
// 9 and 8.
constexpr int NARROW_MANY = 2048, MANY_ROWS = 512;
__host__ __device__ constexpr bool in_registers(long long rows, long long width) {
    return width <= NARROW || (width <= NARROW_MANY && rows >= MANY_ROWS);
}

// ---------------------------------------------------------------- values
// logits as f32, exactly, whatever they are stored in
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half(v); }
template <> __device__ __forceinline__ __hip_bfloat16 from_float<__hip_bfloat16>(float v) { return __float2bfloat16(v); }

// Order of the logits as whole numbers: larger logit, larger key.  A place that holds nothing (masked, NaN, past the row's
// count) is -inf, whose key is NO_KEY: whatever is above it holds something.  The two zeros are one value (x + 0 turns the
// negative one over).
constexpr unsigned NO_KEY = 0x007FFFFFu;
__device__ __forceinline__ float or_nothing(float v) { return fmaxf(v, -__builtin_inff()); }       // (NaN: the other operand)
__device__ __forceinline__ unsigned key_of(float v) {
    const int b = __float_as_int(v + 0.0f);
    return (unsigned)b ^ ((unsigned)(b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key ^ (~(unsigned)((int)key >> 31) | 0x80000000u));
}

// ---------------------------------------------------------------- lane exchange
// (DPP controls: row_shr:n = 0x110 + n moves a value n lanes up inside a row of 16, row_ror:n = 0x120 + n rotates it;
//  lanes that nothing reaches get 0)
template <int CTRL> __device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true); }
template <int CTRL> __device__ __forceinline__ unsigned dpp(unsigned v) { return (unsigned)dpp<CTRL>((int)v); }
template <int CTRL> __device__ __forceinline__ float dpp(float v) { return __int_as_float(dpp<CTRL>(__float_as_int(v))); }
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
    const long long b = __double_as_longlong(v);
    const int lo = dpp<CTRL>((int)(b & 0xFFFFFFFFll)), hi = dpp<CTRL>((int)(b >> 32));
    return __longlong_as_double(((long long)hi << 32) | (unsigned)lo);
}

struct Add { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; } };
struct Max {
    template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; }
};
// The larger of v and the value N lanes round in the row of 16 (N < 0: -N apart in each four; -8: mirrored in each eight), as
// one vector instruction: from fmaxf the compiler makes a move and two maxima, the first to make the moved value canonical.
// (Two wait states between a vector write and a lane permutation that reads it: the s_nop.)
template <int N> __device__ __forceinline__ float max_rotated(float v) {
    float r;
    if constexpr (N == 8) asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 row_ror:8 row_mask:0xf bank_mask:0xf" : "=v"(r) : "v"(v));
    if constexpr (N == 4) asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 row_ror:4 row_mask:0xf bank_mask:0xf" : "=v"(r) : "v"(v));
    if constexpr (N == 2) asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 row_ror:2 row_mask:0xf bank_mask:0xf" : "=v"(r) : "v"(v));
    if constexpr (N == -2) asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf" : "=v"(r) : "v"(v));
    if constexpr (N == -1) asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf" : "=v"(r) : "v"(v));
    if constexpr (N == -8) asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 row_half_mirror row_mask:0xf bank_mask:0xf" : "=v"(r) : "v"(v));
    if constexpr (N == 1) asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 row_ror:1 row_mask:0xf bank_mask:0xf" : "=v"(r) : "v"(v));
    return r;
}
struct Min { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a < b ? a : b; } };

// op over v and the value of the lane 16 (32) apart: the half-swaps of gfx950 put the two side by side, in either order
template <int X, typename OP> __device__ __forceinline__ unsigned across(unsigned v, OP op) {
    const auto r = X == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return op((unsigned)r[0], (unsigned)r[1]);
}
template <int X, typename OP> __device__ __forceinline__ int across(int v, OP op) {
    const auto r = X == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return op((int)r[0], (int)r[1]);
}
template <int X, typename OP> __device__ __forceinline__ float across(float v, OP op) {
    const unsigned b = __float_as_uint(v);
    const auto r = X == 16 ? __builtin_amdgcn_permlane16_swap(b, b, false, false) : __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int X, typename OP> __device__ __forceinline__ double across(double v, OP op) {
    const long long b = __double_as_longlong(v);
    const unsigned lo = (unsigned)b, hi = (unsigned)(b >> 32);
    const auto l = X == 16 ? __builtin_amdgcn_permlane16_swap(lo, lo, false, false) : __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto h = X == 16 ? __builtin_amdgcn_permlane16_swap(hi, hi, false, false) : __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    return op(__longlong_as_double((long long)h[0] << 32 | (unsigned)l[0]), __longlong_as_double((long long)h[1] << 32 | (unsigned)l[1]));
}

// v over the lanes of a group, in every lane of it
template <int G, typename V, typename OP> __device__ __forceinline__ V all(V v, OP op) {
    static_assert(G == 4 || G == 8 || G == 16 || G == 64, "groups of 4, 8, 16 or 64 lanes");
    if constexpr (G <= 8) {
        v = op(v, dpp<0x4E>(v));
        v = op(v, dpp<0xB1>(v));
        return G == 8 ? op(v, dpp<0x141>(v)) : v;        // (the other four's, by the mirror of eight)
    }
    v = op(v, dpp<0x128>(v));
    v = op(v, dpp<0x124>(v));
    v = op(v, dpp<0x122>(v));
    v = op(v, dpp<0x121>(v));
    if (G == 64) {
        v = across<16>(v, op);
        v = across<32>(v, op);
    }
    return v;
}
template <int G> __device__ __forceinline__ float all(float v, Max op) {
    if constexpr (G <= 8) {
        v = max_rotated<-1>(max_rotated<-2>(v));
        return G == 8 ? max_rotated<-8>(v) : v;
    }
    v = max_rotated<1>(max_rotated<2>(max_rotated<4>(max_rotated<8>(v))));
    if (G == 64) {
        v = across<16>(v, op);
        v = across<32>(v, op);
    }
    return v;
}
// sum over the lanes of the group in front of this one
template <int G, typename V> __device__ __forceinline__ V before(V v) {
    V s = v;
    if constexpr (G == 4) {
        const int lane = lane_id() & 3;
        const V one = dpp<0x90>(s);          // lanes 0 0 1 2 of each four
        s += lane > 0 ? one : V(0);
        const V two = dpp<0x40>(s);          // lanes 0 0 0 1
        s += lane > 1 ? two : V(0);
        return s - v;
    }
    if constexpr (G == 8) {
        const int lane = lane_id() & 7;
        const V one = dpp<0x111>(s);
        s += lane > 0 ? one : V(0);
        const V two = dpp<0x112>(s);
        s += lane > 1 ? two : V(0);
        const V four = dpp<0x114>(s);
        s += lane > 3 ? four : V(0);
        return s - v;
    }
    s += dpp<0x111>(s);
    s += dpp<0x112>(s);
    s += dpp<0x114>(s);
    s += dpp<0x118>(s);
    if (G == 64) {
        const V t0 = __shfl(s, 15), t1 = __shfl(s, 31), t2 = __shfl(s, 47);
        const int row = lane_id() >> 4;
        s += (row > 0 ? t0 : V(0)) + (row > 1 ? t1 : V(0)) + (row > 2 ? t2 : V(0));
    }
    return s - v;        // (exact in whole numbers; in f32 a rounding of the sum, one of those that MARGIN counts)
}

// ---------------------------------------------------------------- weights
// A row's weights exp((l - max)/T) as whole multiples of 2^-36 of the largest: sums of up to 2^17 of them stay below 2^53
// and are exact in f64 in whatever order they are taken - by lanes, by blocks, by atomics - so a draw is a function of its
// row alone.  What is lost is a weight's 2^-37, far below the 2^-24 steps of the random numbers.
constexpr double UNIT = 68719476736.0;          // 2^36
// 2^(d + SHIFT), d in [-900, 900], to 4e-14 of itself (2^-44; what it is used for has steps of 2^-36 and 2^-24): on |f| <= 1/2,
// 2^f = 1 + f P(f) with the P of degree 8 whose largest error is least (Remez exchange).  Exact at d = 0.  The coefficients are
// held in scalar registers: as literals each costs two vector moves beside its product.
__device__ __forceinline__ double scalar(double c) {
    asm("" : "+s"(c));
    return c;
}
template <int SHIFT> __device__ __forceinline__ double pow2(double d) {
    const double n = __builtin_rint(d), f = d - n;
    double p = scalar(1.0208624985451055e-07);
    p = fma(p, f, scalar(1.3255224921011604e-06));
    p = fma(p, f, scalar(1.5252659326736988e-05));
    p = fma(p, f, scalar(1.5403455852016875e-04));
    p = fma(p, f, scalar(1.3333558222014398e-03));
    p = fma(p, f, scalar(9.6181291594041980e-03));
    p = fma(p, f, scalar(5.5504108664546310e-02));
    p = fma(p, f, scalar(2.4022650695812967e-01));
    p = fma(p, f, scalar(6.9314718055994710e-01));
    p = fma(p, f, 1.0);
    return p * __longlong_as_double((long long)(1023 + SHIFT + (int)n) << 52);
}
// d = (l - max) log2(e) / T <= 0: the weight rint(2^d UNIT)
__device__ __forceinline__ double weight_of(double d) { return __builtin_rint(pow2<36>(fmax(d, -64.0))); }
// log2(z) to about 2^-45, z in the range of f32: the hardware's logarithm and one Newton step
__device__ __forceinline__ double log2_of(double z) {
    const double l = (double)__builtin_amdgcn_logf((float)z);
    return fma(fma(z, pow2<0>(-l), -1.0), 1.4426950408889634, l);
}
constexpr double LOG2E = 1.4426950408889634;

// ---------------------------------------------------------------- loading and selecting in registers
// The E places of lane `lane` as keys; places from n on hold nothing and are not read (a vector may reach past n, never
// past width).  vec: rows start on the alignment of a lane's E values (or of 16 bytes).
template <int BYTES> struct Words;
template <> struct Words<2> { typedef unsigned short type; };
template <> struct Words<4> { typedef unsigned type; };
template <> struct Words<8> { typedef uint2 type; };
template <> struct Words<16> { typedef uint4 type; };
template <typename T, int E> struct Places {
    static constexpr int BYTES = E * (int)sizeof(T) < 16 ? E * (int)sizeof(T) : 16;
    static constexpr int PER = BYTES / (int)sizeof(T);
    typedef typename Words<BYTES>::type word;
};
template <typename T, int E>
__device__ __forceinline__ void load_values(const T* __restrict__ row, int n, int width, bool vec, int lane, float (&v)[E]) {
    typedef Places<T, E> P;
    const int at = lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = -__builtin_inff();
    if (at >= n) return;
    if (vec && at + E <= width) {
        union { typename P::word w[E / P::PER]; T t[E]; } u;
#pragma unroll
        for (int j = 0; j < E / P::PER; ++j) u.w[j] = reinterpret_cast<const typename P::word*>(row + at)[j];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = as_float(u.t[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = at + e < n ? as_float(row[at + e]) : -__builtin_inff();
    }
    if (at + E > n) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = at + e < n ? v[e] : -__builtin_inff();
    }
}

// The keys of a group in descending order by place (lane 0's first is the largest): a bitonic network.  Blocks that sort the
// other way hold their keys complemented, so that every exchange puts the larger key first; an exchange between lanes is a
// lane permutation and a median with 0 or the largest key (that is: the larger, or the smaller).
// Keys of 64 bits (a key and its place) are compared and selected instead.
template <int X> __device__ __forceinline__ unsigned exchanged(unsigned v, bool keep_larger) {
    unsigned a = v, b;
    if constexpr (X == 1) b = dpp<0xB1>(v);
    if constexpr (X == 2) b = dpp<0x4E>(v);
    if constexpr (X == 4) b = dpp<0x1B>(dpp<0x141>(v));       // 7 - i, then 3 - i inside each four: i ^ 4
    if constexpr (X == 8) b = dpp<0x128>(v);
    if constexpr (X == 16) {                                  // (v and the partner's, in either order)
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        a = r[0];
        b = r[1];
    }
    if constexpr (X == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        a = r[0];
        b = r[1];
    }
    return max(min(a, b), min(max(a, b), keep_larger ? 0xFFFFFFFFu : 0u));
}
typedef unsigned long long wide_key;
template <int X> __device__ __forceinline__ wide_key exchanged(wide_key v, bool keep_larger) {
    const unsigned lo = (unsigned)v, hi = (unsigned)(v >> 32);
    wide_key a = v, b;
    if constexpr (X == 1) b = (wide_key)dpp<0xB1>(hi) << 32 | dpp<0xB1>(lo);
    if constexpr (X == 2) b = (wide_key)dpp<0x4E>(hi) << 32 | dpp<0x4E>(lo);
    if constexpr (X == 4) b = (wide_key)dpp<0x1B>(dpp<0x141>(hi)) << 32 | dpp<0x1B>(dpp<0x141>(lo));
    if constexpr (X == 8) b = (wide_key)dpp<0x128>(hi) << 32 | dpp<0x128>(lo);
    if constexpr (X == 16 || X == 32) {
        const auto l = X == 16 ? __builtin_amdgcn_permlane16_swap(lo, lo, false, false) : __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
        const auto h = X == 16 ? __builtin_amdgcn_permlane16_swap(hi, hi, false, false) : __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
        a = (wide_key)(unsigned)h[0] << 32 | (unsigned)l[0];
        b = (wide_key)(unsigned)h[1] << 32 | (unsigned)l[1];
    }
    return (a > b) == keep_larger ? a : b;
}
template <int X, int E, typename K> __device__ __forceinline__ void exchange_lanes(K (&k)[E], int lane) {
    const bool keep_larger = (lane & X) == 0;
#pragma unroll
    for (int e = 0; e < E; ++e) k[e] = exchanged<X>(k[e], keep_larger);
    if constexpr (X > 1) exchange_lanes<X / 2, E>(k, lane);
}
template <typename K> __device__ __forceinline__ void exchange_places(K& a, K& b) {
    const K larger = a > b ? a : b;
    b = a > b ? b : a;
    a = larger;
}
// places D, D/2, .. 1 apart inside a lane; blocks of SIZE alternate in direction (SIZE = E: one block)
template <int D, int SIZE, int E, typename K> __device__ __forceinline__ void exchange_inside(K (&k)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e)
        if ((e & D) == 0) {
            if (SIZE < E && (e & SIZE)) exchange_places(k[e | D], k[e]);
            else exchange_places(k[e], k[e | D]);
        }
    if constexpr (D > 1) exchange_inside<D / 2, SIZE, E>(k);
}
template <int SIZE, int E, typename K> __device__ __forceinline__ void sort_inside(K (&k)[E]) {
    if constexpr (SIZE < E) {
        exchange_inside<SIZE / 2, SIZE, E>(k);
        sort_inside<SIZE * 2, E>(k);
    }
}
template <int L, int G, int E, typename K> __device__ __forceinline__ void sort_lanes(K (&k)[E], int lane) {
    const K m = ((lane & (L / 2)) != 0) != (L < G && (lane & L) != 0) ? ~K(0) : K(0);
#pragma unroll
    for (int e = 0; e < E; ++e) k[e] ^= m;
    exchange_lanes<L / 2, E>(k, lane);
    exchange_inside<E / 2, E, E>(k);
    if constexpr (L < G) sort_lanes<L * 2, G, E>(k, lane);
}
template <int G, int E, typename K> __device__ __forceinline__ void sort_keys(K (&k)[E], int lane) {
    sort_inside<2, E>(k);
    const K m = lane & 1 ? ~K(0) : K(0);
#pragma unroll
    for (int e = 0; e < E; ++e) k[e] ^= m;
    exchange_inside<E / 2, E, E>(k);
    sort_lanes<2, G, E>(k, lane);
}
// the key at a rank of a sorted group: every lane offers its key of that register, the lane that owns the rank is read
template <int G, int E> __device__ __forceinline__ unsigned at_rank(const unsigned (&k)[E], int rank) {
    unsigned v = k[0];
#pragma unroll
    for (int e = 1; e < E; ++e) v = (rank & (E - 1)) == e ? k[e] : v;
    return __shfl(v, rank / E, G);
}

// ---------------------------------------------------------------- wide rows
// A row of n values read by a workgroup: single places up to the first 16-byte boundary, vectors, single places behind the
// last one - whatever the row's alignment.  f(i, v, count): the places i .. i + count - 1, count 1 or PER; `first` and `step`
// are the caller's thread and the number of threads.
template <typename T> struct Span {
    static constexpr int PER = 16 / (int)sizeof(T);
    const T* x;
    int n, head, vecs;
    __device__ __forceinline__ Span(const T* row, int count) : x(row), n(count) {
        head = min((int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T), n);
        vecs = (n - head) / PER;
    }
    // four vectors on their way at a time: one CU's share of memory is latency
    struct Batch { uint4 w[4]; };
    __device__ __forceinline__ Batch fetch(int k0, int step) const {
        Batch u{};
        if (k0 < vecs) {
#pragma unroll
            for (int b = 0; b < 4; ++b) u.w[b] = reinterpret_cast<const uint4*>(x + head)[min(k0 + b * step, vecs - 1)];
        }
        return u;
    }
    template <typename F> __device__ __forceinline__ void each(int first, int step, F f) const { each(first, step, fetch(first, step), f); }
    // (with the first vectors on their way already)
    template <typename F> __device__ __forceinline__ void each(int first, int step, Batch ahead, F f) const {
        if (first < head) {
            const float v[PER] = {as_float(x[first])};
            f(first, v, 1);
        }
        for (int k0 = first; k0 < vecs; k0 += 4 * step) {
            if (k0 != first) ahead = fetch(k0, step);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int k = k0 + b * step;
                if (k >= vecs) break;
                union { uint4 w; T t[PER]; } u;
                u.w = ahead.w[b];
                float v[PER];
#pragma unroll
                for (int j = 0; j < PER; ++j) v[j] = as_float(u.t[j]);
                f(head + k * PER, v, PER);
            }
        }
        const int tail = head + vecs * PER + first;
        if (tail < n) {
            const float v[PER] = {as_float(x[tail])};
            f(tail, v, 1);
        }
    }
};

}  // namespace rows
}  // namespace aig
