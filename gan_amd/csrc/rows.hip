// Operators on rows of logits: sampling from given random numbers, and the largest logits of a row.
#include <type_traits>

#include "rows.h"

namespace aig {
namespace {
using namespace rows;

struct Settings {       // of every row, or of each where a pointer is given
    float temperature, top_p, min_p, per;       // per: log2(e) / temperature
    int top_k;
    const float *temperature_rows, *top_p_rows, *min_p_rows;
    const int* top_k_rows;
};
struct RowSettings {
    float temperature, top_p, min_p, per;
    int top_k;
    __device__ __forceinline__ RowSettings(const Settings& s, long long r)
        : temperature(s.temperature_rows ? s.temperature_rows[r] : s.temperature), top_p(s.top_p_rows ? s.top_p_rows[r] : s.top_p),
          min_p(s.min_p_rows ? s.min_p_rows[r] : s.min_p), per(s.temperature_rows ? (float)(LOG2E / (double)temperature) : s.per),
          top_k(s.top_k_rows ? s.top_k_rows[r] : s.top_k) {}
    // the smallest weight that min-p and the unit leave
    __device__ __forceinline__ double floor() const { return min_p > 0.0f ? fmax((double)fminf(min_p, 1.0f) * UNIT, 1.0) : 1.0; }
    // the mass that top-p keeps of `total`: a place stays while the mass in front of it is below this; the first always does
    __device__ __forceinline__ double mass(double total) const { return fmax((double)top_p * total, 1.0); }
};

struct SampleRows {
    long long rows, ld;
    int width, draws, vec, fill;
    long long period;           // counts and want are shared by rows a period apart (0: every row has its own)
    const int *counts, *want;
    const float* u;
    int* out;
    Settings how;
    __device__ __forceinline__ long long plan_row(long long r) const { return period ? r % period : r; }
    __device__ __forceinline__ int count(long long r) const { return counts ? min(max(counts[plan_row(r)], 0), width) : width; }
    __device__ __forceinline__ int wanted(long long r) const { return want ? min(want[plan_row(r)], draws) : draws; }
    __device__ __forceinline__ float uniform(long long r, int d) const {
        return fminf(fmaxf(u[r * draws + d], 0.0f), 1.0f - 1.0f / 16777216.0f);
    }
    // the d-th pick of row r (-1: none).  For wiring every fan-in needs an answer: the first pick stands in for a missing
    // second one, the row's last place for a missing first.
    __device__ __forceinline__ void store(long long r, int d, int pick, int& first, int n) const {
        if (fill) {
            if (d == 0) first = pick < 0 ? n - 1 : pick;
            if (pick < 0) pick = first;
        }
        out[r * draws + d] = pick;
    }
};

// Places that a row keeps, of those whose key is the threshold the first `quota` by place: w = 0 for the others.
template <int G, int E, typename W> __device__ __forceinline__ void keep_first(const unsigned (&key)[E], W (&w)[E], unsigned thr, int quota) {
    int ties = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) ties += key[e] == thr;
    int tie = before<G>(ties);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const bool stays = key[e] > thr || (key[e] == thr && tie < quota);
        tie += key[e] == thr;
        w[e] = stays ? w[e] : W(0);
    }
}

// The draws of a row as they are defined, in whole weights (f64).  guess: the key at top-p's border or one near it (0: none).
template <int G, int E>
__device__ __forceinline__ void exact_draws(const SampleRows& a, const RowSettings& how, long long r, int lane, int n, int want,
                                            const unsigned (&key)[E], unsigned top, unsigned guess) {
    const float m = value_of(top);
    const double m64 = (double)m, per = LOG2E / (double)how.temperature;
    double q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        // (no branch: the places' chains of products run side by side.  The largest place, infinite or not, has weight 1, and
        //  a place that holds nothing, at -inf, has none)
        const float v = value_of(key[e]);
        q[e] = weight_of(v == m ? 0.0 : ((double)v - m64) * per);
    }
    if (how.top_k > 0 && how.top_k < a.width) {
        unsigned s[E];
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] = key[e];
        sort_keys<G, E>(s, lane);
        const unsigned thr = at_rank<G, E>(s, how.top_k - 1);
        int over = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) over += key[e] > thr;
        keep_first<G, E>(key, q, thr, how.top_k - all<G>(over, Add()));
    }
    if (how.top_p < 1.0f) {
        double total = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) total += q[e];
        const double p = how.mass(all<G>(total, Add()));
        // the border: the largest key that, with everything above it, holds mass p
        auto from = [&](unsigned c) {
            double w = 0.0;
#pragma unroll
            for (int e = 0; e < E; ++e) w += key[e] >= c ? q[e] : 0.0;
            return all<G>(w, Add());
        };
        unsigned t = guess;
        if (t != 0u) {
            while (from(t) < p) {              // too high: the next key below
                unsigned next = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) next = max(next, key[e] < t ? key[e] : 0u);
                t = all<G>(next, Max());
            }
            while (from(t + 1) >= p) {         // too low: the next key above
                unsigned next = 0xFFFFFFFFu;
#pragma unroll
                for (int e = 0; e < E; ++e) next = min(next, key[e] > t ? key[e] : 0xFFFFFFFFu);
                t = all<G>(next, Min());
            }
        } else {
            for (int bit = 31; bit >= 0; --bit)
                if (from(t | (1u << bit)) >= p) t |= 1u << bit;
        }
        double above = 0.0;
        int ties = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            above += key[e] > t ? q[e] : 0.0;
            ties += key[e] == t;
        }
        above = all<G>(above, Add());
        int tie = before<G>(ties);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool stays = key[e] > t || (key[e] == t && above + (double)tie * q[e] < p);
            tie += key[e] == t;
            q[e] = stays ? q[e] : 0.0;
        }
    }
    const double least = how.floor();
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] = q[e] >= least ? q[e] : 0.0;

    int first = -1;
    for (int d = 0; d < a.draws; ++d) {
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) sum += q[e];
        const double total = all<G>(sum, Add());
        double upto = before<G>(sum);
        const double t = (double)a.uniform(r, d) * total;
        int at = -1;                       // one lane's range holds t (none: nothing is left)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const double next = upto + q[e];
            const bool here = upto <= t && t < next;
            at = here ? lane * E + e : at;
            q[e] = here ? 0.0 : q[e];
            upto = next;
        }
        at = all<G>(at, Max());
        if (lane == 0) a.store(r, d, d < want ? at : -1, first, n);
    }
}

// The same in f32, as long as that is certain.  A sum of weights in f32 is off by less than 2^-19 of the row's total (2^-18 for
// rows of 2048 places): an exponential of -d carries three roundings of d (2^-24 each, times ln 2) and its own last bit, the
// average of d over the weights of 1024 places is at most 6.5 (2048: 7.2); a sum of 16 (32) in a lane rounds by half of as many
// such steps of the lane's, the six steps over the lanes by six of the total: 0.8e-6 + 0.1e-6 + 0.8e-6 (0.9 + 0.1 + 1.3).  A
// decision between two numbers that lie further apart than margin_of of the total is therefore the exact one; a row with a
// closer one is drawn again in f64 (returns false).  So is a min-p within half a unit of 2^-36 of a weight, and a draw that finds no
// weight left in the sums while a place still has some.  How many rows that is, of normal logits of deviation 2 at T 0.8, two
// draws: under top-p 0.9 0.1 % of 64 places, 0.3 % of 256, 1 % of 1,024, 4 % of 2,000; under top-p 0.99 0.7, 3, 12 and 46 % (the
// border lies among places of small weight); of 64 places without filters 0.1 %, at T 0.1 26 % (the second draw does).
// What that buys: an f64 exponential alone is 26 instructions a place, and sums in f32 take their lane permutations along.
template <int PLACES> __device__ __host__ constexpr float margin_of() { return PLACES <= 1024 ? 1.0f / 262144.0f : 1.0f / 131072.0f; }

constexpr float HALF_UNIT = (float)(0.5 / UNIT);       // of the largest weight's 1: less is no whole multiple of 2^-36 but 0

// Weights that cannot be told apart by their order: exponentials of different logits are in order but for two last bits (2^-22).
__device__ __forceinline__ float band_high(float thr) { return thr * (1.0f + 1.0f / 1048576.0f); }
__device__ __forceinline__ float band_low(float thr) { return thr * (1.0f - 1.0f / 1048576.0f); }

// The border of top-p, or of a top-k of few places and then top-p, without sorting the row: the bits between a lower bound of
// it and the largest weight are halved (the bits of a float are nearly its logarithm) until few places lie between, and those
// are sorted.  Top-p: what goes is (1 - p) of the total on fewer than n places, none larger than the last place that stays, so
// that one's weight is at least (1 - p) total / n; a halving is a comparison, a selection and an addition a place, and two do
// for most rows of 256.  Top-k: by the number of places, from their mean weight; the list is all places from lo on.
// 152,896 rows of 256, top-p 0.9: 89 us sorted whole, 64 like this.
// lds: [G M].  Returns false where places do not get few (hundreds of equal ones); keep, over and from count inside the list.
constexpr int HALVINGS = 12;
template <int G> __device__ __host__ constexpr int listed_a_lane() { return G == 16 ? 4 : 2; }
template <int G, int E>
__device__ __forceinline__ bool border_in_list(const float (&w)[E], int top_k, float top_p, int n, int lane, float* lds, bool& sure,
                                               float& thr, int& keep, int& over, int& from) {
    constexpr int M = listed_a_lane<G>();
    const bool by_k = top_k > 0, by_p = top_p < 1.0f;
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += w[e];
    float total = all<G>(sum, Add()), p = top_p * total;
    constexpr float LEAST = 1e-30f;
    constexpr unsigned TOP = 0x3F800001u;        // over the bits of 1, the largest weight
    unsigned lo = __float_as_uint(by_k ? LEAST : fmaxf((total - p) / (float)n * 0.999f, LEAST)), hi = TOP;
    float front = 0.0f;          // top-p: the mass of the places from hi on: below p; that from lo on is not
    int count = n, here = 0;
    if (by_k) {                  // fewer than top_k places from hi on; from lo on there are as many, or lo is LEAST
        unsigned mid = __float_as_uint(fmaxf(total / (float)n, 2.0f * LEAST));
        for (int round = 0; count > G * M && round < HALVINGS; ++round) {
            int c = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) c += __float_as_uint(w[e]) >= mid;
            c = all<G>(c, Add());
            const bool enough = c >= top_k;
            lo = enough ? mid : lo;
            hi = enough ? hi : mid;
            count = enough ? c : count;
            mid = lo + (hi - lo) / 2;
        }
        hi = TOP;
        if (count > G * M) return false;
#pragma unroll
        for (int e = 0; e < E; ++e) here += __float_as_uint(w[e]) >= lo;
    } else {
        auto halve = [&]() {
            const unsigned mid = lo + (hi - lo) / 2;
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) s += __float_as_uint(w[e]) >= mid ? w[e] : 0.0f;
            s = all<G>(s, Add());
            const bool enough = s >= p;
            lo = enough ? mid : lo;
            hi = enough ? hi : mid;
            front = enough ? front : s;
        };
        halve();
        int round = 0;
        do {
            halve();
            here = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) here += __float_as_uint(w[e]) - lo < hi - lo;
            count = all<G>(here, Add());
        } while (count > G * M && ++round < HALVINGS);
        if (count > G * M) return false;
    }
    int at = before<G>(here);
#pragma unroll
    for (int e = 0; e < M; ++e) lds[lane * M + e] = 0.0f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (__float_as_uint(w[e]) - lo < hi - lo) lds[at++] = w[e];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    unsigned s[M];
#pragma unroll
    for (int e = 0; e < M; ++e) s[e] = __float_as_uint(lds[lane * M + e]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    sort_keys<G, M>(s, lane);
    keep = by_k ? top_k : G * M;
    if (by_p) {
        float ws[M], mine = 0.0f;
#pragma unroll
        for (int e = 0; e < M; ++e) {
            ws[e] = lane * M + e < keep ? __uint_as_float(s[e]) : 0.0f;
            mine += ws[e];
        }
        const float listed = all<G>(mine, Add());
        if (by_k) p = top_p * (total = listed);
        float upto = front + before<G>(mine), nearest = front + listed - p;       // (negative: the list ends too early)
        int stay = 0;
#pragma unroll
        for (int e = 0; e < M; ++e) {
            // (the first place of the row always stays; behind the last one the whole of the list is in front)
            nearest = e > 0 || lane > 0 || front > 0.0f ? fminf(nearest, fabsf(upto - p)) : nearest;
            stay += upto < p;
            upto += ws[e];
        }
        sure = sure && nearest > margin_of<G * E>() * total;
        keep = max(min(keep, all<G>(stay, Add())), 1);
    }
    thr = __uint_as_float(at_rank<G, M>(s, keep - 1));
    const float high = band_high(thr), low = band_low(thr);
    // (a band that is not all in the list)
    sure = sure && (thr == 0.0f || (__float_as_uint(low) >= lo && (__float_as_uint(high) < hi || hi == TOP)));
#pragma unroll
    for (int e = 0; e < M; ++e) {
        over += __uint_as_float(s[e]) > high;
        from += __uint_as_float(s[e]) >= low;
    }
    const int both = all<G>(over | from << 16, Add());
    over = both & 0xFFFF;
    from = both >> 16;
    return true;
}

template <int G, int E>
__device__ __forceinline__ bool quick_draws(const SampleRows& a, const RowSettings& how, long long r, int lane, int n, int want,
                                            const float (&v)[E], float m, float* lds, float& guess) {
    const float per = how.per;
    bool sure = per > 0.0f && per < 1e30f && m < __builtin_inff();
    float w[E];
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = __builtin_amdgcn_exp2f((v[e] - m) * per);
    const bool by_p = how.top_p < 1.0f, by_k = how.top_k > 0 && how.top_k < a.width;
    if (by_p || by_k) {
        // In the order of the weights the places that stay are the first ones.  That is the order of the logits but for the
        // last bit of an exponential, and for logits whose weights round to one number: see below.
        float thr = 0.0f;                       // the weight of the last place that stays
        int keep = 0, over = 0, from = 0;       // of some run of the order around it: places that stay, over the band below, and not under it
        bool found = false;
        if constexpr (G >= 16) {
            if (!by_k || how.top_k <= G * listed_a_lane<G>() / 2)
                found = border_in_list<G, E>(w, by_k ? how.top_k : 0, how.top_p, n, lane, lds, sure, thr, keep, over, from);
        }
        if (!found) {
            unsigned s[E];
#pragma unroll
            for (int e = 0; e < E; ++e) s[e] = __float_as_uint(w[e]);
            sort_keys<G, E>(s, lane);
            keep = by_k ? how.top_k : G * E;
            if (by_p) {
                float ws[E], sum = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    ws[e] = __uint_as_float(s[e]);
                    if (by_k) ws[e] = lane * E + e < keep ? ws[e] : 0.0f;
                    sum += ws[e];
                }
                const float total = all<G>(sum, Add()), p = how.top_p * total;
                float upto = before<G>(sum), nearest = 1e30f;
                int stay = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    // (the first place always stays; behind the last one the whole of the total is in front)
                    nearest = e > 0 || lane > 0 ? fminf(nearest, fabsf(upto - p)) : nearest;
                    stay += upto < p;
                    upto += ws[e];
                }
                sure = sure && nearest > margin_of<G * E>() * total;
                keep = max(min(keep, all<G>(stay, Add())), 1);
            }
            thr = __uint_as_float(at_rank<G, E>(s, keep - 1));
            const float high = band_high(thr), low = band_low(thr);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                over += w[e] > high;
                from += w[e] >= low;
            }
            const int both = all<G>(over | from << 16, Add());
            over = both & 0xFFFF;
            from = both >> 16;
        }
        if (thr > 0.0f) {       // (else every weight stays)
            guess = thr;
            // Places whose weight is within a few last bits of the border's: all of them stay, or their logits are equal and the
            // first of them do - or the exact form has to tell them apart.
            const float high = band_high(thr), low = band_low(thr);
            if (from > keep) {
                const int quota = keep - over;
                float border = -__builtin_inff();           // the largest logit that is not over it
#pragma unroll
                for (int e = 0; e < E; ++e) border = w[e] > high ? border : fmaxf(border, v[e]);
                border = all<G>(border, Max());
                int here = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) here += v[e] == border;
                int tie = before<G>(here);
                sure = sure && all<G>(here, Add()) == from - over;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const bool at = v[e] == border;
                    w[e] = (v[e] > border) | (at & (tie < quota)) ? w[e] : 0.0f;
                    tie += at;
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) w[e] = w[e] >= low ? w[e] : 0.0f;
            }
        }
    }
    if (how.min_p > 2.0f * HALF_UNIT) {       // (a smaller one takes nothing out that is not 0 anyway)
        // (a weight is compared as a multiple of 2^-36: up to half a unit beside itself)
        const float least = fminf(how.min_p, 1.0f), near = 4.0f * margin_of<G * E>() * least + HALF_UNIT;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            sure = sure && !(v[e] < m && fabsf(w[e] - least) <= near);
            w[e] = w[e] >= least ? w[e] : 0.0f;
        }
    }
    if (!all<G>((int)sure, Min())) return false;

    // Draws.  The lane whose places hold t is found from the lanes' sums; its places are then looked through by the group, from
    // LDS.  A lane with few places looks through them by itself.
    constexpr bool BY_GROUP = E > 4;
    constexpr int EACH = E > G ? E / G : 1;       // places of it a lane
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += w[e];
    if (BY_GROUP) {
#pragma unroll
        for (int e = 0; e < E; ++e) lds[lane * E + e] = w[e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    }
    int first = -1;
    float margin = 0.0f;
    for (int d = 0; d < a.draws; ++d) {
        const float total = all<G>(sum, Add());
        margin = fmaxf(margin, margin_of<G * E>() * total);
        float upto = before<G>(sum);
        const float t = a.uniform(r, d) * total;
        int at = -1;
        if (BY_GROUP) {
            const int owner = all<G>(t >= upto && t < upto + sum ? lane : -1, Max());
            const int place = max(owner, 0) * E + (lane * EACH & (E - 1));
            const bool has = lane * EACH < E;
            float here[EACH], end = __shfl(upto, max(owner, 0), G), mine = 0.0f;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                here[e] = lds[place + e];
                here[e] = has ? here[e] : 0.0f;
                mine += here[e];
            }
            end += before<G>(mine);
            float gone = 0.0f;
#pragma unroll
            for (int e = 0; e < EACH; ++e) {
                const bool clear = (owner >= 0) & has & (t - end > margin) & (end + here[e] - t > margin);
                at = clear ? place + e : at;
                gone = clear ? here[e] : gone;
                end += here[e];
            }
            if (at >= 0) lds[at] = 0.0f;
            at = all<G>(at, Max());
            gone = all<G>(gone, Add());
            sum = lane == owner ? fmaxf(sum - gone, 0.0f) : sum;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
        } else {
            // the lane's places that end at or before t, and the nearest end to it
            float end = upto, nearest = fabsf(t - upto);
            int passed = 0;
            const bool mine = t >= upto && t < upto + sum;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                end += w[e];
                nearest = fminf(nearest, fabsf(t - end));
                passed += t >= end;
            }
            const bool clear = mine && nearest > margin;
            at = all<G>(clear ? lane * E + passed : -1, Max());
            sum = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                w[e] = clear && e == passed ? 0.0f : w[e];
                sum += w[e];
            }
        }
        if (at < 0) {
            if (total > 0.0f) return false;
            // No weight is left, or what is left was below the last bit of the sum that it was part of: the exact form draws a
            // place that is there.  (The weights themselves: LDS holds 0 for the places that were drawn, and what is clearly
            // below half a unit is none.)
            if (BY_GROUP) {
                int left = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) left |= lds[lane * E + e] > 0.99f * HALF_UNIT;
                if (all<G>(left, Max())) return false;
            }
        }
        if (lane == 0) a.store(r, d, d < want ? at : -1, first, n);
    }
    return true;
}

// A group of G lanes per row, the row in registers: read once, 8 bytes a draw written.  Bound by the issue of vector
// instructions, not by memory: 100,000 x 64 under top-k 32, top-p 0.9 and min-p (sorted whole: 300 of 877 instructions a wave)
// 22.9 us, of which 18 are issue; 27 MB would be copied in 6.  Without filters, all places valid, 9.7 us.  152,896 x 256 under
// top-p 0.9 64 us, 60 of them issue of 983 instructions a wave (157 MB: 35).  One row 4.4 us: a chain of lane exchanges.
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void k_sample(const T* __restrict__ x, SampleRows a) {
    __shared__ __attribute__((aligned(16))) float lds[E > 4 ? 256 / G : 1][E > 4 ? G * E : 1];
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / G;
    if (r >= a.rows) return;
    const int lane = threadIdx.x & (G - 1);
    const RowSettings how(a.how, r);
    const int n = a.count(r), want = a.wanted(r);
    float v[E];
    load_values<T, E>(x + r * a.ld, n, a.width, a.vec, lane, v);
    float m = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = or_nothing(v[e]);
        m = fmaxf(m, v[e]);
    }
    m = all<G>(m, Max());
    if (!(how.temperature > 0.0f)) {      // the largest, then the next
        int first = -1;
        for (int d = 0; d < a.draws; ++d) {
            int at = 0x7FFFFFFF;
#pragma unroll
            for (int e = E - 1; e >= 0; --e) at = v[e] == m ? lane * E + e : at;
            at = all<G>(at, Min());
            if (lane == 0) a.store(r, d, m > -__builtin_inff() && d < want ? at : -1, first, n);
            m = -__builtin_inff();
#pragma unroll
            for (int e = 0; e < E; ++e) {
                v[e] = lane * E + e == at ? -__builtin_inff() : v[e];
                m = fmaxf(m, v[e]);
            }
            m = all<G>(m, Max());
        }
        return;
    }
    int first = -1;
    if (!(m > -__builtin_inff())) {       // nothing in the row
        for (int d = 0; d < a.draws; ++d)
            if (lane == 0) a.store(r, d, -1, first, n);
        return;
    }
    float guess = 0.0f;
    if (!quick_draws<G, E>(a, how, r, lane, n, want, v, m, lds[E > 4 ? threadIdx.x / G : 0], guess)) {
        unsigned key[E];
#pragma unroll
        for (int e = 0; e < E; ++e) key[e] = key_of(v[e]);
        // (the logit that has the border's weight, or one near it)
        const unsigned near = guess > 0.0f ? key_of(m + __builtin_amdgcn_logf(guess) / how.per) : 0u;
        exact_draws<G, E>(a, how, r, lane, n, want, key, key_of(m), near);
    }
}

// ---------------------------------------------------------------- wide rows: a workgroup per row
constexpr int WIDE_T = 1024, WIDE_E = 8, TILE = WIDE_T * WIDE_E, TILES = MAX_WIDTH / TILE;

struct Block {          // sums and scans over the sixteen waves of a workgroup
    double* d;          // [17]
    template <typename V, typename OP> __device__ __forceinline__ V all(V v, OP op) const {
        V* s = reinterpret_cast<V*>(d);
        v = rows::all<64>(v, op);
        __syncthreads();
        if (lane_id() == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        V t = s[0];
#pragma unroll
        for (int w = 1; w < WIDE_T / 64; ++w) t = op(t, s[w]);
        return t;
    }
    // sum over the threads in front of this one; total over all
    template <typename V> __device__ __forceinline__ V before(V v, V& total) const {
        V* s = reinterpret_cast<V*>(d);
        const V mine = rows::before<64>(v);
        __syncthreads();
        if (lane_id() == 63) s[threadIdx.x >> 6] = mine + v;
        __syncthreads();
        V front = V(0);
        total = V(0);
#pragma unroll
        for (int w = 0; w < WIDE_T / 64; ++w) {
            front += w < (int)(threadIdx.x >> 6) ? s[w] : V(0);
            total += s[w];
        }
        return front + mine;
    }
};

// The largest key such that it and everything above it amount to `target` (AMOUNT of a place: 1, or its weight): eight bits
// at a time, a histogram over the places that share the bits found so far.  above: what the keys over it amount to.
// The sums are of whole numbers below 2^53: exact, in any order of the atomics.
template <typename KEY, typename AMOUNT>
__device__ __forceinline__ unsigned border_key(int n, double target, double* hist, double* found, KEY key, AMOUNT amount, double& above) {
    unsigned prefix = 0, mask = 0;
    above = 0.0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) hist[threadIdx.x] = 0.0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += WIDE_T) {
            const unsigned k = key(i);
            if (k > NO_KEY && (k & mask) == prefix) unsafeAtomicAdd(&hist[(k >> shift) & 255u], amount(k, i));
        }
        __syncthreads();
        if (threadIdx.x < 64) {
            const int hi = 255 - 4 * threadIdx.x;
            const double h[4] = {hist[hi], hist[hi - 1], hist[hi - 2], hist[hi - 3]};
            double upto = above + rows::before<64>(h[0] + h[1] + h[2] + h[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double next = upto + h[j];
                if (upto < target && target <= next) {
                    found[0] = (double)(hi - j);
                    found[1] = upto;
                }
                upto = next;
            }
        }
        __syncthreads();
        prefix |= (unsigned)found[0] << shift;
        mask |= 255u << shift;
        above = found[1];
    }
    return prefix;
}

// Any row of weights that are drawn in parts (no temperature 0): borders bit by bit over the whole row, a handful of
// passes of f64 weights.  Taken where a list below overflows (thousands of equal logits at a border, top-k of thousands).
template <typename T>
__device__ __forceinline__ void general_draws(const T* __restrict__ x, const SampleRows& a) {
    __shared__ double hist[256], found[2], red[WIDE_T / 64 + 1], tile_mass[TILES];
    __shared__ int tile_ties[TILES], picked[8];
    const Block block{red};
    const long long r = blockIdx.x;
    const RowSettings how(a.how, r);
    const int n = a.count(r), want = a.wanted(r);
    x += r * a.ld;
    auto key = [&](int i) { return key_of(or_nothing(as_float(x[i]))); };
    int first = -1;

    unsigned top = 0;
    int held = 0;
    for (int i = threadIdx.x; i < n; i += WIDE_T) {
        const unsigned k = key(i);
        top = max(top, k);
        held += k > NO_KEY;
    }
    top = block.all(top, Max());
    held = block.all(held, Add());
    const double m = (double)value_of(top), per = LOG2E / (double)how.temperature;
    auto weight = [&](unsigned k) { return k <= NO_KEY ? 0.0 : k == top ? UNIT : weight_of(((double)value_of(k) - m) * per); };

    // what top-k keeps: keys over kthr, and the first kquota at it
    unsigned kthr = 0;
    int kquota = 0;
    if (how.top_k > 0 && how.top_k < held) {
        double above;
        kthr = border_key(n, (double)how.top_k, hist, found, key, [](unsigned, int) { return 1.0; }, above);
        kquota = how.top_k - (int)above;
    }
    unsigned pthr = 0;
    double pabove = 0.0, p = 0.0;
    if (how.top_p < 1.0f) {
        double over = 0.0;         // the mass of the keys over top-k's border; the border itself keeps its quota
        for (int i = threadIdx.x; i < n; i += WIDE_T) {
            const unsigned k = key(i);
            over += k > kthr ? weight(k) : 0.0;
        }
        over = block.all(over, Add());
        p = how.mass(over + (double)kquota * weight(kthr));
        if (over >= p) {           // (else the border is top-k's)
            const unsigned lowest = kthr;
            pthr = border_key(n, p, hist, found, [&](int i) { const unsigned k = key(i); return k > lowest ? k : 0u; },
                              [&](unsigned k, int) { return weight(k); }, pabove);
        } else {
            pthr = kthr;
            pabove = over;
        }
    }
    const double least = how.floor();
    // the weight of a place that is the tie-th of its key's (place order) where its key is a border
    auto kept = [&](unsigned k, int ktie, int ptie) {
        double q = weight(k);
        if (k < kthr || (k == kthr && ktie >= kquota)) q = 0.0;
        if (p > 0.0 && (k < pthr || (k == pthr && !(pabove + (double)ptie * q < p)))) q = 0.0;
        return q >= least ? q : 0.0;
    };
    // ties in front of a place are counted for the higher of the two borders only: at the lower one everything is gone
    const unsigned border = max(kthr, pthr);

    // the mass of each tile of places, and the ties in front of it
    double total = 0.0;
    int tiles = (n + TILE - 1) / TILE, ties_so_far = 0;
    auto tile_places = [&](int t, int front, double (&q)[WIDE_E], int& ties_here) {
        const int base = t * TILE + (int)threadIdx.x * WIDE_E;
        unsigned k[WIDE_E];
        int ties = 0;
#pragma unroll
        for (int e = 0; e < WIDE_E; ++e) {
            k[e] = base + e < n ? key(base + e) : 0u;
            ties += k[e] == border && border != 0u;
        }
        int tie = front + block.before(ties, ties_here);
#pragma unroll
        for (int e = 0; e < WIDE_E; ++e) {
            q[e] = kept(k[e], tie, tie);
            tie += k[e] == border && border != 0u;
        }
    };
    for (int t = 0; t < tiles; ++t) {
        double q[WIDE_E], sum = 0.0;
        int ties_here;
        tile_places(t, ties_so_far, q, ties_here);
#pragma unroll
        for (int e = 0; e < WIDE_E; ++e) sum += q[e];
        sum = block.all(sum, Add());
        if (threadIdx.x == 0) {
            tile_mass[t] = sum;
            tile_ties[t] = ties_so_far;
        }
        total += sum;
        ties_so_far += ties_here;
    }
    __syncthreads();

    for (int d = 0; d < a.draws; ++d) {
        if (!(total > 0.0)) {
            if (threadIdx.x == 0) a.store(r, d, -1, first, n);
            continue;
        }
        const double t = (double)a.uniform(r, d) * total;
        int tile = 0;
        double front = 0.0;
        while (tile + 1 < tiles && front + tile_mass[tile] <= t) front += tile_mass[tile++];
        double q[WIDE_E], sum = 0.0, all_mass;
        int ties_here;
        tile_places(tile, tile_ties[tile], q, ties_here);
        const int base = tile * TILE + (int)threadIdx.x * WIDE_E;
#pragma unroll
        for (int e = 0; e < WIDE_E; ++e) {
            for (int j = 0; j < d; ++j) q[e] = picked[j] == base + e ? 0.0 : q[e];
            sum += q[e];
        }
        double upto = front + block.before(sum, all_mass);
#pragma unroll
        for (int e = 0; e < WIDE_E; ++e) {
            const double next = upto + q[e];
            if (upto <= t && t < next) {
                picked[d] = base + e;
                tile_mass[tile] -= q[e];
                found[0] = q[e];
            }
            upto = next;
        }
        __syncthreads();
        total -= found[0];
        if (threadIdx.x == 0) a.store(r, d, d < want ? picked[d] : -1, first, n);
        __syncthreads();
    }
}

// A key with its place in the order that is wanted: larger key first, then the lower place.
__device__ __forceinline__ wide_key with_place(unsigned key, int place) { return (wide_key)key << 32 | (unsigned)~place; }

// Places picked out of a row, in LDS.
constexpr int LIST = 1024, LIST_K = 512;       // (a place a thread)
struct List {
    wide_key key[LIST], sorted[LIST];
    double q[LIST];
    int count;
    __device__ __forceinline__ void add(unsigned k, int i) {
        const int at = atomicAdd(&count, 1);
        if (at < LIST) key[at] = with_place(k, i);
    }
    // key[0 .. n) into sorted[0 .. n), largest first.  All keys differ.  Each wave sorts 64 of them; a key's rank is then its own in
    // there and, by a binary search each, that among the 64 of every other wave.
    __device__ __forceinline__ void sort(int n) {
        const int t = threadIdx.x, wave = t >> 6;
        __syncthreads();
        wide_key mine[1] = {0ull};
        if (wave * 64 < n) {
            if (t < n) mine[0] = key[t];
            sort_keys<64, 1>(mine, t & 63);
            if (n > 64) key[t] = mine[0];
        }
        int rank = t & 63;
        if (n > 64) {
            __syncthreads();
            if (wave * 64 < n) {
                for (int c = 0; c * 64 < n; ++c) {
                    if (c == wave) continue;
                    const wide_key* other = key + c * 64;
                    int front = 0;
#pragma unroll
                    for (int step = 32; step; step >>= 1) front += other[front + step - 1] > mine[0] ? step : 0;
                    rank += front + (other[front] > mine[0]);
                }
            }
        }
        if (t < n) sorted[rank] = mine[0];
        __syncthreads();
    }
};

// the k-th largest of 64 E keys, each the largest of 16 / E threads
template <int E> __device__ __forceinline__ unsigned kth_of_groups(const unsigned* keys, int k) {
    unsigned v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = 0;
#pragma unroll
        for (int j = 0; j < 16 / E; ++j) v[e] = max(v[e], keys[(e * (16 / E) + j) * 64 + threadIdx.x]);
    }
    sort_keys<64, E>(v, threadIdx.x);
    return at_rank<64, E>(v, k - 1);
}

// A key that at least k of the row's places reach, few more do: the k-th largest of the threads' own largest (mine: this
// thread's).  NO_KEY + 1 where fewer than k threads hold a place.
__device__ __forceinline__ unsigned bound_of_top(unsigned mine, int k, unsigned* keys, unsigned* result) {
    keys[threadIdx.x] = mine;
    __syncthreads();
    if (threadIdx.x < 64) {
        // (the largest of several threads: fewer keys sort quicker, and few more places reach their k-th)
        unsigned thr;
        if (k <= 32) {
            thr = kth_of_groups<1>(keys, k);
        } else if (k <= 64) {
            thr = kth_of_groups<2>(keys, k);
        } else if (k <= 128) {
            thr = kth_of_groups<4>(keys, k);
        } else {
            // halvings between the smallest and the largest until few more than k of the threads' are over
            float v[16], least = __builtin_inff(), most = -__builtin_inff();
            int count = 0;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                v[e] = value_of(keys[e * 64 + threadIdx.x]);
                const bool held = v[e] > -__builtin_inff();
                count += held;
                least = held ? fminf(least, v[e]) : least;
                most = fmaxf(most, v[e]);
            }
            count = all<64>(count, Add());
            float lo = all<64>(least, Min()), hi = all<64>(most, Max());
            for (int round = 0; count > k + k / 8 && round < HALVINGS; ++round) {
                const float mid = 0.5f * lo + 0.5f * hi;
                int c = 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) c += v[e] >= mid;
                c = all<64>(c, Add());
                lo = c >= k ? mid : lo;
                hi = c >= k ? hi : mid;
                count = c >= k ? c : count;
            }
            least = __builtin_inff();
#pragma unroll
            for (int e = 0; e < 16; ++e) least = v[e] >= lo ? fminf(least, v[e]) : least;
            thr = count < k ? 0u : key_of(all<64>(least, Min()));
        }
        if (threadIdx.x == 0) *result = max(thr, NO_KEY + 1);
    }
    __syncthreads();
    return *result;
}

// Rows up to this width are read place by place (every thread holds some), wider ones by vectors.
constexpr int BY_PLACE = 8192;
template <typename T, typename F> __device__ __forceinline__ void each_place(const Span<T>& row, F f) {
    if (row.n <= BY_PLACE) {
        for (int i = threadIdx.x; i < row.n; i += WIDE_T) f(i, as_float(row.x[i]));
    } else {
        row.each(threadIdx.x, WIDE_T, [&](int i, const float (&v)[Span<T>::PER], int count) {
#pragma unroll
            for (int j = 0; j < Span<T>::PER; ++j)
                if (j < count) f(i + j, v[j]);
        });
    }
}

// A row in parts that follow each other by place: the places in front of its vectors, the 64 vectors of each wave of each
// sweep of the workgroup over them, the places behind.
constexpr int PARTS = 2 + 16 * (MAX_WIDTH / (4 * WIDE_T) + 1);
template <typename T> struct Parts {
    static constexpr int PER = Span<T>::PER;
    const Span<T>& row;
    int sweeps;
    __device__ __forceinline__ explicit Parts(const Span<T>& r) : row(r), sweeps((r.vecs + WIDE_T - 1) / WIDE_T) {}
    __device__ __forceinline__ int count() const { return 2 + 16 * sweeps; }
    __device__ __forceinline__ int of(int place) const {
        if (place < row.head) return 0;
        const int k = (place - row.head) / PER;
        return k < row.vecs ? 1 + 16 * (k / WIDE_T) + (k % WIDE_T) / 64 : 1 + 16 * sweeps;
    }
    // the places of a lane in a part: first place, and how many
    __device__ __forceinline__ int places(int part, int lane, int& first) const {
        if (part == 0) {
            first = lane;
            return lane < row.head ? 1 : 0;
        }
        if (part == 1 + 16 * sweeps) {
            first = row.head + row.vecs * PER + lane;
            return first < row.n ? 1 : 0;
        }
        const int k = ((part - 1) / 16) * WIDE_T + ((part - 1) % 16) * 64 + lane;
        first = row.head + k * PER;
        return k < row.vecs ? PER : 0;
    }
    // f(part) for every part, by the wave that has it
    template <typename F> __device__ __forceinline__ void each(F f) const {
        const int wave = threadIdx.x >> 6;
        for (int s = 0; s < sweeps; ++s) f(1 + 16 * s + wave);
        if (wave == 0) f(0);
        if (wave == 1) f(1 + 16 * sweeps);
    }
    // The places that hold `value`, in order: their number in front of each part goes to front[part], and f(place, number in
    // order, part) is called for those numbered below `quota` (a lane's own, by that lane).  ties: [count()] in LDS.
    template <typename F> __device__ __forceinline__ void ties_of(float value, int quota, int* ties, int* front, const Block& block, F f) const {
        const int lane = lane_id();
        __syncthreads();
        each([&](int part) {
            int at;
            const int here = places(part, lane, at);
            float v[PER];
            load(at, here, v);
            int c = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) c += (j < here) & (v[j] == value);
            c = all<64>(c, Add());
            if (lane == 0) ties[part] = c;
        });
        __syncthreads();
        int total;
        const int before_part = block.before((int)threadIdx.x < count() ? ties[threadIdx.x] : 0, total);
        if ((int)threadIdx.x < count()) front[threadIdx.x] = before_part;
        __syncthreads();
        each([&](int part) {
            if (front[part] >= quota || ties[part] == 0) return;
            int at;
            const int here = places(part, lane, at);
            float v[PER];
            load(at, here, v);
            int c = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) c += (j < here) & (v[j] == value);
            int number = front[part] + before<64>(c);
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if ((j < here) & (v[j] == value)) {
                    if (number < quota) f(at + j, number, part);
                    ++number;
                }
        });
        __syncthreads();
    }
    __device__ __forceinline__ void load(int first, int n, float (&v)[PER]) const {
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = -__builtin_inff();
        if (n == PER) {
            union { uint4 w; T t[PER]; } u;
            u.w = *reinterpret_cast<const uint4*>(row.x + first);
#pragma unroll
            for (int j = 0; j < PER; ++j) v[j] = or_nothing(as_float(u.t[j]));
        } else if (n == 1) {
            v[0] = or_nothing(as_float(row.x[first]));
        }
    }
};

// The list after it has overflowed: fewer than k places lie over `low`, so those are listed, and the first of the many at it.
// (Where thousands lie over it - rows of a few threads' places - the list stays too long.)
template <typename T>
__device__ __forceinline__ void list_with_ties(const Span<T>& row, const Parts<T>& parts, List& list, unsigned low, int k, const Block& block) {
    __syncthreads();
    if (threadIdx.x == 0) list.count = 0;
    __syncthreads();
    const float value = value_of(low);
    each_place(row, [&](int i, float v) {
        if (v > value) list.add(key_of(v), i);
    });
    __syncthreads();
    const int over = list.count;
    if (over >= k) return;
    int* ties = reinterpret_cast<int*>(list.q);
    parts.ties_of(value, k - over, ties, ties + PARTS, block, [&](int place, int, int) { list.add(low, place); });
}

// A workgroup per row.  Weights are whole numbers in f64 throughout, so their sums do not depend on how the row is split.
//   top-k (to LIST_K): the places that can be among the k largest are picked out into a list, everything else happens there.
//   otherwise: top-p's border from a histogram of the weights over BINS steps of the logit (from the row's smallest, or the
//   smallest that has a weight), the places of its bin in a list, or counted where they are thousands of one value;
//   then the sum of what stays in each part of the row, and for each draw a look through the one part that holds it.
// Rows are as many as a batch has requests, so most CUs idle; what a row costs is its CU's time: 48 x 50,001 bf16 under top-k
// 50 and top-p 15 us (two reads of 100 KB, two lists sorted), top-k 500 27 us; under top-p alone 45 us, two f64
// exponentials a place, and 70 us for 512 rows of 32,001 (two a CU); 150 rows of 131,072 under a top-k
// beyond LIST_K 700 us (general_draws).
constexpr int BINS = 4096;
constexpr float OCTAVES = 37.0f;          // a weight under 2^-37 is 0

template <typename T>
__global__ __launch_bounds__(WIDE_T) void k_sample_wide(const T* __restrict__ x, SampleRows a) {
    constexpr int PER = Span<T>::PER;
    __shared__ double hist[BINS], part_mass[PARTS], red[WIDE_T / 64 + 1], found[2];
    __shared__ List list;
    __shared__ unsigned shared_key;
    __shared__ int picked[AIG_ROWS_MAX_DRAWS], found_at;
    const Block block{red};
    const long long r = blockIdx.x;
    const RowSettings how(a.how, r);
    const int n = a.count(r), want = a.wanted(r), t = threadIdx.x;
    const Span<T> row(x + r * a.ld, n);
    int first = -1;

    if (!(how.temperature > 0.0f)) {      // the largest, then the next
        for (int d = 0; d < a.draws; ++d) {
            unsigned best = 0;
            int at = 0x7FFFFFFF;
            each_place(row, [&](int i, float v) {
                unsigned k = key_of(or_nothing(v));
                for (int j = 0; j < d; ++j) k = picked[j] == i ? 0u : k;
                if (k > best) {
                    best = k;
                    at = i;
                }
            });
            const unsigned top = block.all(best, Max());
            at = block.all(best == top ? at : 0x7FFFFFFF, Min());
            __syncthreads();
            if (t == 0) {
                picked[d] = top > NO_KEY ? at : -1;
                a.store(r, d, top > NO_KEY && d < want ? at : -1, first, n);
            }
            __syncthreads();
        }
        return;
    }
    auto none = [&](int from) {
        if (t == 0)
            for (int d = from; d < a.draws; ++d) a.store(r, d, -1, first, n);
    };

    const bool by_k = how.top_k > 0 && how.top_k < n, by_p = how.top_p < 1.0f;
    float m = -__builtin_inff(), low_end = __builtin_inff();
    if (by_p && !by_k)
        each_place(row, [&](int, float v) {
            m = fmaxf(m, or_nothing(v));
            low_end = v > -__builtin_inff() ? fminf(low_end, v) : low_end;
        });
    else
        each_place(row, [&](int, float v) { m = fmaxf(m, or_nothing(v)); });
    const unsigned my_top = key_of(m);
    m = block.all(m, Max());
    if (!(m > -__builtin_inff())) return none(0);
    low_end = block.all(low_end, Min());
    const double m64 = (double)m, per = LOG2E / (double)how.temperature;
    auto weight = [&](float v) { return weight_of(((double)v - m64) * per); };      // (-inf, which holds nothing: 0)
    const double least = how.floor();
    const float octaves = fminf((m - low_end) * (float)per, OCTAVES);
    const float bins_per = by_p && !by_k && octaves > 0.0f ? (float)per * ((float)BINS / octaves) : 1.0f;
    if ((by_k && how.top_k > LIST_K) || !((float)per > 0.0f && bins_per < 1e30f && m < __builtin_inff())) return general_draws<T>(x, a);
    if (t == 0) list.count = 0;

    if (by_k) {
        const unsigned low = bound_of_top(my_top, how.top_k, reinterpret_cast<unsigned*>(list.key), &shared_key);
        const float low_value = value_of(low);
        each_place(row, [&](int i, float v) {
            if (v >= low_value) list.add(key_of(v), i);
        });
        __syncthreads();
        if (list.count > LIST) list_with_ties(row, Parts<T>(row), list, low, how.top_k, block);
        const int have = list.count;
        if (have > LIST) return general_draws<T>(x, a);
        list.sort(have);
        const int keep = min(how.top_k, have);
        const wide_key mine = t < have ? list.sorted[t] : 0ull;
        double q = t < keep ? weight(value_of((unsigned)(mine >> 32))) : 0.0, total;
        if (by_p) {
            const double front = block.before(q, total);
            if (t > 0 && !(front < how.mass(total))) q = 0.0;
        }
        if (q < least) q = 0.0;
        // and in the order of the places
        if (t < have) {
            list.q[t] = q;
            list.key[t] = mine << 32 | (unsigned)t;
        }
        list.sort(have);
        const wide_key here = t < have ? list.sorted[t] : 0ull;
        const int place = t < have ? (int)~(unsigned)(here >> 32) : -1;
        q = t < have ? list.q[(unsigned)here] : 0.0;
        double upto = block.before(q, total);
        for (int d = 0; d < a.draws; ++d) {
            if (!(total > 0.0)) return none(d);
            const double u = (double)a.uniform(r, d) * total;
            if (q > 0.0 && upto <= u && u < upto + q) {
                found[0] = q;
                found_at = place;
            }
            __syncthreads();
            const double gone = found[0];
            const int at = found_at;
            total -= gone;
            if (place > at) upto -= gone;
            if (place == at) q = 0.0;
            if (t == 0) a.store(r, d, d < want ? at : -1, first, n);
            __syncthreads();
        }
        return;
    }

    const Parts<T> parts(row);
    const int wave = t >> 6, lane = t & 63;
    auto bin_of = [&](float v) { return (int)fminf((m - v) * bins_per, (float)(BINS - 1)); };
    int border_bin = BINS;          // places in bins below it stay; of its own places those up to (thr, last) in the order of the keys
    double above = 0.0, p = 0.0;
    if (by_p) {
        for (int i = t; i < BINS; i += WIDE_T) hist[i] = 0.0;
        __syncthreads();
        each_place(row, [&](int, float raw) {
            const float v = or_nothing(raw);
            const double q = weight(v);
            if (q > 0.0) unsafeAtomicAdd(&hist[bin_of(v)], q);
        });
        __syncthreads();
        double h[BINS / WIDE_T], sum = 0.0, total;
#pragma unroll
        for (int j = 0; j < BINS / WIDE_T; ++j) sum += h[j] = hist[t * (BINS / WIDE_T) + j];
        double upto = block.before(sum, total);
        p = how.mass(total);
#pragma unroll
        for (int j = 0; j < BINS / WIDE_T; ++j) {
            if (upto < p && p <= upto + h[j]) {
                found[0] = upto;
                found_at = t * (BINS / WIDE_T) + j;
            }
            upto += h[j];
        }
        __syncthreads();
        above = found[0];
        border_bin = found_at;
    }
    auto part_sum = [&](int part) {
        int at;
        const int here = parts.places(part, lane, at);
        float v[PER];
        parts.load(at, here, v);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (j >= here) break;
            const int b = bin_of(v[j]);
            const double q = weight(v[j]);
            if (b < border_bin) sum += q >= least ? q : 0.0;
            else if (b == border_bin && q > 0.0) list.add(key_of(v[j]), at + j);
        }
        sum = all<64>(sum, Add());
        if (lane == 0) part_mass[part] = sum;
    };
    parts.each(part_sum);
    __syncthreads();
    wide_key edge = ~0ull;          // the last place of the border's bin that stays
    if (by_p) {
        const int have = list.count;
        if (have > LIST) {
            // thousands of places in the border's bin: of one value, or there is no help but the general form
            unsigned highest = 0u, lowest = 0xFFFFFFFFu;
            each_place(row, [&](int, float v) {
                if (v > -__builtin_inff() && bin_of(v) == border_bin) {
                    highest = max(highest, key_of(v));
                    lowest = min(lowest, key_of(v));
                }
            });
            highest = block.all(highest, Max());
            lowest = block.all(lowest, Min());
            if (highest != lowest) return general_draws<T>(x, a);
            const double q = weight(value_of(highest));
            int keep = (int)fmin((p - above) / q, (double)n);          // places i = 0, 1, .. stay while above + i q < p
            while (keep > 0 && !(above + (double)(keep - 1) * q < p)) --keep;
            while (keep < n && above + (double)keep * q < p) ++keep;
            int* ties = reinterpret_cast<int*>(list.q);
            if (t == 0) list.sorted[0] = 0ull;
            parts.ties_of(value_of(highest), keep, ties, ties + PARTS, block, [&](int place, int number, int) {
                if (number == keep - 1) list.sorted[0] = with_place(highest, place);
            });
            edge = list.sorted[0];            // (0: fewer ties than would stay, all of them do)
            if (t < parts.count() && q >= least) part_mass[t] += q * (double)min(max(keep - ties[PARTS + t], 0), ties[t]);
            __syncthreads();
        } else {
            list.sort(have);
            const wide_key mine = t < have ? list.sorted[t] : 0ull;
            const double q = t < have ? weight(value_of((unsigned)(mine >> 32))) : 0.0;
            double sum;
            const double front = above + block.before(q, sum);
            const bool stays = t < have && (front == 0.0 || front < p);
            const int keep = block.all((int)stays, Add());
            if (keep > 0) edge = list.sorted[keep - 1];
            if (stays && q >= least) unsafeAtomicAdd(&part_mass[parts.of((int)~(unsigned)mine)], q);
            __syncthreads();
        }
    }
    for (int d = 0; d < a.draws; ++d) {
        const double mass = t < parts.count() ? part_mass[t] : 0.0;
        double total;
        const double upto = block.before(mass, total);
        if (!(total > 0.0)) return none(d);
        const double u = (double)a.uniform(r, d) * total;
        if (upto <= u && u < upto + mass) {
            found[0] = upto;
            found_at = t;
        }
        __syncthreads();
        if (wave == 0) {
            const int part = found_at;
            int at;
            const int here = parts.places(part, lane, at);
            float v[PER];
            parts.load(at, here, v);
            double q[PER], sum = 0.0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int b = bin_of(v[j]);
                // (selections, no branches; a chain of || gives the same picks)
                const bool stays = (b < border_bin) | ((b == border_bin) & (with_place(key_of(v[j]), at + j) >= edge));
                const double w = weight(v[j]);
                bool taken = j >= here;
                for (int i = 0; i < d; ++i) taken |= picked[i] == at + j;
                q[j] = (stays & !taken & (w >= least)) ? w : 0.0;
                sum += q[j];
            }
            double end = found[0] + before<64>(sum);
            const double left = part_mass[part];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (end <= u && u < end + q[j]) {
                    picked[d] = at + j;
                    part_mass[part] = left - q[j];
                }
                end += q[j];
            }
        }
        __syncthreads();
        if (t == 0) a.store(r, d, d < want ? picked[d] : -1, first, n);
    }
}

// ---------------------------------------------------------------- the largest logits
struct TopArgs {
    long long rows, ld;
    int width, m, vec;
    const int* counts;
    float temperature, per;      // per: log2(e) / temperature
    float* values;
    int* index;
    float* lse;
    __device__ __forceinline__ int count(long long r) const { return counts ? min(max(counts[r], 0), width) : width; }
};

// The group's row sorted with its places, whole (M = 0; bf16's key and place share 32 bits), or a list of G M places that holds
// the m largest picked out first and sorted alone.  Bound by the issue of vector instructions: 100,000 x 64, m 16, 18 us, 15 of
// them issue of 726 instructions a wave (39 MB read and written: 9 us at the rate of a copy); sorted whole 23 us.
template <typename T, int G, int E, int M>
__global__ __launch_bounds__(256) void k_top(const T* __restrict__ x, TopArgs a) {
    constexpr int TRIES = 5;
    constexpr bool WHOLE = M == 0, PACKED = WHOLE && std::is_same<T, __hip_bfloat16>::value;
    __shared__ wide_key lds[WHOLE ? 1 : 256 / G][WHOLE ? 1 : G * (M ? M : 1)];
    const long long r = ((long long)blockIdx.x * 256 + threadIdx.x) / G;
    if (r >= a.rows) return;
    const int lane = threadIdx.x & (G - 1), n = a.count(r);
    float v[E], m = -__builtin_inff();
    load_values<T, E>(x + r * a.ld, n, a.width, a.vec, lane, v);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = or_nothing(v[e]);
        m = fmaxf(m, v[e]);
    }
    m = all<G>(m, Max());
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += v[e] == m ? 1.0f : __builtin_amdgcn_exp2f((v[e] - m) * a.per);
    s = all<G>(s, Add());
    if (lane == 0) a.lse[r] = m > -__builtin_inff() ? m / a.temperature + logf(s) : -__builtin_inff();

    float* values = a.values + r * a.m;
    int* index = a.index + r * a.m;
    if constexpr (PACKED) {
        unsigned k[E];
#pragma unroll
        for (int e = 0; e < E; ++e) k[e] = (key_of(v[e]) & 0xFFFF0000u) | (unsigned)(0xFFFF - (lane * E + e));
        sort_keys<G, E>(k, lane);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int rank = lane * E + e;
            if (rank < a.m) {
                // (a bf16's low half: zeros under a key of a positive value, ones under one of a negative)
                const unsigned key = (k[e] & 0xFFFF0000u) | ((int)k[e] < 0 ? 0u : 0xFFFFu);
                values[rank] = value_of(key);
                index[rank] = key > NO_KEY ? 0xFFFF - (int)(k[e] & 0xFFFFu) : -1;
            }
        }
        for (int j = G * E + lane; j < a.m; j += G) {
            values[j] = -__builtin_inff();
            index[j] = -1;
        }
    } else {
        auto write = [&](wide_key k, int rank) {
            const unsigned key = (unsigned)(k >> 32);
            values[rank] = key > NO_KEY ? value_of(key) : -__builtin_inff();
            index[rank] = key > NO_KEY ? (int)~(unsigned)k : -1;
        };
        constexpr int PER = WHOLE ? E : M;
        wide_key k[PER];
        if constexpr (WHOLE) {
#pragma unroll
            for (int e = 0; e < E; ++e) k[e] = with_place(key_of(v[e]), lane * E + e);
        } else {
            wide_key* list = lds[threadIdx.x / G];
#pragma unroll
            for (int e = 0; e < M; ++e) list[lane * M + e] = 0;
            // What lies between the smallest and the largest logit is halved until the places from lo on are at least m and at
            // most the list's (the first try: what lies far below the largest at this temperature is most likely masked).  A few
            // tries on the next value below hi is looked at itself: if there are enough of it, the first by place do.
            float least = __builtin_inff();
#pragma unroll
            for (int e = 0; e < E; ++e) least = v[e] > -__builtin_inff() ? fminf(least, v[e]) : least;
            least = all<G>(least, Min());
            float lo = least, hi = m, mid = fmaxf(0.5f * lo + 0.5f * m, m - 16.0f * a.temperature);
            bool all_below = true;                        // (no hi yet that places are left out from)
            int count = n, over = 0, quota = G * E;       // places from lo on; from hi on (fewer than m); of those at lo that go on the list
            for (int round = 0; count > G * M; ++round) {
                int c = 0;
                const bool look = round >= TRIES && (round & 1);
                if (!look) {
#pragma unroll
                    for (int e = 0; e < E; ++e) c += v[e] >= mid;
                } else {
                    mid = -__builtin_inff();
#pragma unroll
                    for (int e = 0; e < E; ++e) mid = all_below | (v[e] < hi) ? fmaxf(mid, v[e]) : mid;
                    mid = all<G>(mid, Max());
#pragma unroll
                    for (int e = 0; e < E; ++e) c += v[e] >= mid;
                }
                c = all<G>(c, Add());
                if (c >= a.m) {
                    lo = mid;
                    count = c;
                    if (look) {
                        quota = a.m - over;
                        break;
                    }
                } else {
                    hi = mid;
                    over = c;
                    all_below = false;
                    if (!(mid > least)) break;            // (all that is held is fewer than m)
                }
                mid = 0.5f * lo + 0.5f * hi;
            }
            int here = 0;
            if (quota == G * E) {
#pragma unroll
                for (int e = 0; e < E; ++e) here += v[e] >= lo;
                int at = before<G>(here);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (v[e] >= lo) list[at++] = with_place(key_of(v[e]), lane * E + e);
            } else {
                int ties = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    here += v[e] > lo;
                    ties += v[e] == lo;
                }
                int at = before<G>(here), tie = before<G>(ties);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (v[e] > lo) list[at++] = with_place(key_of(v[e]), lane * E + e);
                    if (v[e] == lo && tie++ < quota) list[over + tie - 1] = with_place(key_of(v[e]), lane * E + e);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int e = 0; e < M; ++e) k[e] = list[lane * M + e];
        }
        sort_keys<G, PER>(k, lane);
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (lane * PER + e < a.m) write(k[e], lane * PER + e);
        for (int j = G * PER + lane; j < a.m; j += G) write(0, j);
    }
}

// A workgroup per row: the places that can be among the m largest are picked out into a list and ranked there.  96 x 32,771
// IEEE halfs, m 64: 9.8 us, two reads of a row by one CU and a sort of some eighty places; the 6.3 MB themselves would take 1.4.
template <typename T>
__global__ __launch_bounds__(WIDE_T) void k_top_wide(const T* __restrict__ x, TopArgs a) {
    __shared__ double hist[256], found[2], red[WIDE_T / 64 + 1];
    __shared__ List list;
    __shared__ unsigned shared_key;
    const Block block{red};
    const long long r = blockIdx.x;
    const int n = a.count(r), t = threadIdx.x;
    const Span<T> row(x + r * a.ld, n);
    float m = -__builtin_inff();
    each_place(row, [&](int, float v) { m = fmaxf(m, or_nothing(v)); });
    unsigned low = bound_of_top(key_of(m), a.m, reinterpret_cast<unsigned*>(list.key), &shared_key);
    m = block.all(m, Max());
    if (t == 0) list.count = 0;
    __syncthreads();
    double s = 0.0;
    const float low_value = value_of(low);
    auto one = [&](int i, float v) {
        if (v >= low_value) list.add(key_of(v), i);
        return __builtin_amdgcn_exp2f((or_nothing(v) - m) * a.per);
    };
    if (n <= BY_PLACE) {
        for (int i = t; i < n; i += WIDE_T) s += (double)one(i, as_float(row.x[i]));
    } else {
        row.each(t, WIDE_T, [&](int i, const float (&v)[Span<T>::PER], int count) {
            float of_vector = 0.0f;
#pragma unroll
            for (int j = 0; j < Span<T>::PER; ++j)
                if (j < count) of_vector += one(i + j, v[j]);
            s += (double)of_vector;
        });
    }
    s = block.all(s, Add());
    // (beside an infinite largest logit there is nothing to sum)
    if (t == 0) a.lse[r] = fabsf(m) < __builtin_inff() ? m / a.temperature + logf((float)s) : m;
    int have = list.count;
    if (have > LIST) {
        list_with_ties(row, Parts<T>(row), list, low, a.m, block);
        have = list.count;
    }
    if (have > LIST) {
        int held = 0;
        each_place(row, [&](int, float v) { held += v > -__builtin_inff(); });
        held = block.all(held, Add());
        // thousands of equal logits at the border, or a row of few threads' places: the border bit by bit, then the list by place
        double above;
        const unsigned thr = held > a.m ? border_key(n, (double)a.m, hist, found, [&](int i) { return key_of(or_nothing(as_float(row.x[i]))); },
                                                     [](unsigned, int) { return 1.0; }, above)
                                        : NO_KEY;
        const int quota = held > a.m ? a.m - (int)above : 0;
        int ties_so_far = 0, kept_so_far = 0;
        for (int tile = 0; tile * TILE < n; ++tile) {
            const int base = tile * TILE + t * WIDE_E;
            unsigned k[WIDE_E];
            int ties = 0, mine = 0, ties_here, kept_here;
#pragma unroll
            for (int e = 0; e < WIDE_E; ++e) {
                k[e] = base + e < n ? key_of(or_nothing(as_float(row.x[base + e]))) : 0u;
                ties += k[e] == thr;
            }
            int tie = ties_so_far + block.before(ties, ties_here);
            bool stays[WIDE_E];
#pragma unroll
            for (int e = 0; e < WIDE_E; ++e) {
                stays[e] = k[e] > thr || (k[e] == thr && tie < quota);
                tie += k[e] == thr;
                mine += stays[e];
            }
            int at = kept_so_far + block.before(mine, kept_here);
#pragma unroll
            for (int e = 0; e < WIDE_E; ++e)
                if (stays[e] && at < LIST) list.key[at++] = with_place(k[e], base + e);
            ties_so_far += ties_here;
            kept_so_far += kept_here;
        }
        have = min(held, a.m);
    }
    list.sort(have);
    for (int j = t; j < a.m; j += WIDE_T) {
        const wide_key k = j < have ? list.sorted[j] : 0ull;
        a.values[r * a.m + j] = j < have ? value_of((unsigned)(k >> 32)) : -__builtin_inff();
        a.index[r * a.m + j] = j < have ? (int)~(unsigned)k : -1;
    }
}

// ---------------------------------------------------------------- launches
template <typename T> int sample_rows(hipStream_t s, const T* x, SampleRows a) {
    // (a lane reads its places as vectors where every row starts on their alignment)
    auto vec = [&](int e) {
        const size_t align = e * sizeof(T) < 16 ? e * sizeof(T) : 16;
        return (int)(reinterpret_cast<uintptr_t>(x) % align == 0 && (a.ld * sizeof(T)) % align == 0);
    };
    auto blocks = [&](int g) { return dim3((unsigned)((a.rows * g + 255) / 256)); };
    if (a.width <= 16) {
        a.vec = vec(4);
        hipLaunchKernelGGL((k_sample<T, 4, 4>), blocks(4), dim3(256), 0, s, x, a);
    } else if (a.width <= 64) {
        a.vec = vec(8);
        hipLaunchKernelGGL((k_sample<T, 8, 8>), blocks(8), dim3(256), 0, s, x, a);
    } else if (a.width <= 256) {
        a.vec = vec(16);
        hipLaunchKernelGGL((k_sample<T, 16, 16>), blocks(16), dim3(256), 0, s, x, a);
    } else if (a.width <= 512) {
        a.vec = vec(8);
        hipLaunchKernelGGL((k_sample<T, 64, 8>), blocks(64), dim3(256), 0, s, x, a);
    } else if (a.width <= NARROW) {
        a.vec = vec(16);
        hipLaunchKernelGGL((k_sample<T, 64, 16>), blocks(64), dim3(256), 0, s, x, a);
    } else if (in_registers(a.rows, a.width)) {
        a.vec = vec(32);
        hipLaunchKernelGGL((k_sample<T, 64, 32>), blocks(64), dim3(256), 0, s, x, a);
    } else {
        hipLaunchKernelGGL(k_sample_wide<T>, dim3((unsigned)a.rows), dim3(WIDE_T), 0, s, x, a);
    }
    AIG_LAUNCH_CHECK();
    return AIG_OK;
}

template <typename T> int top_rows(hipStream_t s, const T* x, TopArgs a) {
    auto vec = [&](int e) {
        const size_t align = e * sizeof(T) < 16 ? e * sizeof(T) : 16;
        return (int)(reinterpret_cast<uintptr_t>(x) % align == 0 && (a.ld * sizeof(T)) % align == 0);
    };
    auto blocks = [&](int g) { return dim3((unsigned)((a.rows * g + 255) / 256)); };
    constexpr bool PACKED = std::is_same<T, __hip_bfloat16>::value;
    // Lists of G M places, the smallest that leave room over m (a list of exactly m needs its border exactly: 50k x 512, m 64,
    // 113 us on one place a lane, 60 on two; m 48: 54 and 60), and the whole row where that is as fast: 64 places from m = 17 on
    // (m 32: 24 us whole, 28 on four a lane), 32-bit keys from m = 65 on (100k x 256, m 200: 184 us packed, 240 listed).
#define LAUNCH_TOP(G, E, M) hipLaunchKernelGGL((k_top<T, G, E, M>), blocks(G), dim3(256), 0, s, x, a)
    if (a.width <= 16) {
        a.vec = vec(4);
        LAUNCH_TOP(4, 4, 0);
    } else if (a.width <= 64) {
        a.vec = vec(8);
        if constexpr (PACKED) LAUNCH_TOP(8, 8, 0);
        else if (a.m > 16) LAUNCH_TOP(8, 8, 0);
        else if (a.m > 8) LAUNCH_TOP(8, 8, 4);
        else LAUNCH_TOP(8, 8, 2);
    } else if (a.width <= 256) {
        a.vec = vec(16);
        if (a.m > (PACKED ? 64 : 128)) LAUNCH_TOP(16, 16, 0);
        else if (a.m > 32) LAUNCH_TOP(16, 16, 8);
        else if (a.m > 16) LAUNCH_TOP(16, 16, 4);
        else LAUNCH_TOP(16, 16, 2);
    } else if (a.width <= 512) {
        a.vec = vec(8);
        if (a.m <= 48) LAUNCH_TOP(64, 8, 1);
        else if (a.m > (PACKED ? 64 : 96)) LAUNCH_TOP(64, 8, PACKED ? 0 : 4);
        else LAUNCH_TOP(64, 8, 2);
    } else if (a.width <= NARROW) {
        a.vec = vec(16);
        if (a.m <= 48) LAUNCH_TOP(64, 16, 1);
        else if (a.m > (PACKED ? 64 : 96)) LAUNCH_TOP(64, 16, PACKED ? 0 : 4);
        else LAUNCH_TOP(64, 16, 2);
    } else if (in_registers(a.rows, a.width)) {
        a.vec = vec(32);
        if (a.m <= 48) LAUNCH_TOP(64, 32, 1);
        else if (a.m > 96) LAUNCH_TOP(64, 32, 4);
        else LAUNCH_TOP(64, 32, 2);
#undef LAUNCH_TOP
    } else {
        hipLaunchKernelGGL(k_top_wide<T>, dim3((unsigned)a.rows), dim3(WIDE_T), 0, s, x, a);
    }
    AIG_LAUNCH_CHECK();
    return AIG_OK;
}
}  // namespace

// (also the wiring's: every slot of a set of graphs gets an answer)
int launch_sample_rows(hipStream_t s, int64_t rows, int64_t width, int64_t ld, int dtype, const void* logits, const int32_t* counts,
                       const int32_t* want, int64_t period, const aig_sampling* how, int64_t draws, const float* u, bool fill,
                       int32_t* out) {
    SampleRows a{};
    a.rows = rows; a.ld = ld; a.width = (int)width; a.draws = (int)draws; a.fill = fill; a.period = period;
    a.counts = counts; a.want = want; a.u = u; a.out = out;
    a.how = Settings{how->temperature, how->top_p, how->min_p, (float)(rows::LOG2E / (double)how->temperature), how->top_k, how->temperature_rows, how->top_p_rows,
                     how->min_p_rows, how->top_k_rows};
    if (dtype == AIG_F32) return sample_rows(s, static_cast<const float*>(logits), a);
    if (dtype == AIG_F16) return sample_rows(s, static_cast<const __half*>(logits), a);
    return sample_rows(s, static_cast<const __hip_bfloat16*>(logits), a);
}
}  // namespace aig

using namespace aig;

int aig::check_row_limits(const char* what, int64_t rows, int64_t width) {
    if (width > AIG_ROWS_MAX_WIDTH) return fail(AIG_ELIMIT, "%s: rows of %lld: at most %d", what, (long long)width, AIG_ROWS_MAX_WIDTH);
    // (a launch has fewer than 2^32 threads: a wave a row, four of them a workgroup; one of 1024 for rows beyond a wave's registers)
    const int64_t most = width <= rows::NARROW ? (1ll << 26) - 4 : (1ll << 22) - 1;
    if (rows > most) return fail(AIG_ELIMIT, "%s: %lld rows of %lld: at most %lld", what, (long long)rows, (long long)width, (long long)most);
    return AIG_OK;
}

static int check_rows(const char* what, int64_t rows, int64_t width, int64_t ld, int dtype) {
    AIG_REQUIRE(rows >= 0 && width >= 1 && ld >= 0, "%s: bad sizes rows=%lld width=%lld ld=%lld", what, (long long)rows,
                (long long)width, (long long)ld);
    AIG_REQUIRE(dtype == AIG_F32 || dtype == AIG_F16 || dtype == AIG_BF16, "%s: unknown dtype %d", what, dtype);
    return check_row_limits(what, rows, width);
}

extern "C" int aig_sample_rows(int64_t rows, int64_t width, int64_t ld, int dtype, const void* logits, const int32_t* counts,
                               const int32_t* want, const aig_sampling* how, int64_t draws, const float* u, int32_t* out,
                               void* stream) {
    if (const int rc = check_rows("aig_sample_rows", rows, width, ld, dtype)) return rc;
    AIG_REQUIRE(draws >= 1 && draws <= AIG_ROWS_MAX_DRAWS, "aig_sample_rows: draws=%lld is not in 1..%d", (long long)draws,
                AIG_ROWS_MAX_DRAWS);
    AIG_REQUIRE(how, "aig_sample_rows: null settings");
    if (rows == 0) return AIG_OK;
    AIG_REQUIRE(logits && u && out, "aig_sample_rows: null pointer");
    return launch_sample_rows(static_cast<hipStream_t>(stream), rows, width, ld, dtype, logits, counts, want, 0, how, draws, u,
                              false, out);
}

extern "C" int aig_top_rows(int64_t rows, int64_t width, int64_t ld, int dtype, const void* logits, const int32_t* counts,
                            int64_t m, float temperature, float* values, int32_t* index, float* lse, void* stream) {
    if (const int rc = check_rows("aig_top_rows", rows, width, ld, dtype)) return rc;
    AIG_REQUIRE(m >= 1 && m <= AIG_ROWS_MAX_TOP, "aig_top_rows: m=%lld is not in 1..%d", (long long)m, AIG_ROWS_MAX_TOP);
    AIG_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, "aig_top_rows: the temperature %g is not in 1e-6..1e6", (double)temperature);
    if (rows == 0) return AIG_OK;
    AIG_REQUIRE(logits && values && index && lse, "aig_top_rows: null pointer");
    TopArgs a{};
    a.rows = rows; a.ld = ld; a.width = (int)width; a.m = (int)m; a.counts = counts; a.temperature = temperature;
    a.per = (float)(rows::LOG2E / (double)temperature);
    a.values = values; a.index = index; a.lse = lse;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == AIG_F32) return top_rows(s, static_cast<const float*>(logits), a);
    if (dtype == AIG_F16) return top_rows(s, static_cast<const __half*>(logits), a);
    return top_rows(s, static_cast<const __hip_bfloat16*>(logits), a);
}
