// Routing matrices of language models: choice of the experts, the matrix by
// its columns (a stable counting sort), the gradient of the scores, and the
// product of the matrix with the experts' rows (combination) with its
// gradients.
#include "mpspmm_routing.hpp"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kRouteBlock = 256;

// ---------------------------------------------------------------------------
// Choice of the experts
// ---------------------------------------------------------------------------

// Order-preserving integers: a larger key is a better choice, 0 = never
// chosen (-inf), NaN above everything.
__device__ __forceinline__ unsigned key_of(float c)
{
    const unsigned u = float_bits(c);
    if (c != c) return 0xFFFFFFFFu;
    if (u == 0xFF800000u) return 0;
    if (u == 0x80000000u) return 0x80000000u;  // -0 ranks as +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(double c)
{
    const unsigned long long u = __builtin_bit_cast(unsigned long long, c);
    if (c != c) return ~0ull;
    if (u == 0xFFF0000000000000ull) return 0;
    if (u == 0x8000000000000000ull) return u;
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ float of_key(unsigned k)
{
    if (k == 0) return -__builtin_inff();
    return bits_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ double of_key(unsigned long long k)
{
    if (k == 0) return -__builtin_inf();
    return __builtin_bit_cast(double, k >> 63 ? k & 0x7FFFFFFFFFFFFFFFull : ~k);
}
struct RouteShape {
    int T, E, k, score, groups, group_size, top_groups, group_score, renormalise;
    float scale;
    int group_lanes;  // lanes that hold a group's experts, a power of two; 0: groups and lanes do not fit each other
};

// exp(x), x <= 0 in the softmax: the rounding of x * log2(e) is made good by
// its remainder, so that the relative error stays near 2^-23 for any x.
__device__ __forceinline__ float exp_near(float x)
{
    const float log2e = 1.4426950408889634f, log2e_low = 1.9259629911266175e-8f;
    const float hi = x * log2e;
    const float lo = __builtin_fmaf(x, log2e, -hi) + x * log2e_low;
    const float p = __builtin_amdgcn_exp2f(hi);
    // an overflowed or vanished power must not meet an infinite remainder
    return p == 0.0f || p == __builtin_inff() || p != p ? p : __builtin_fmaf(p, lo * 0.6931471805599453f, p);
}
__device__ __forceinline__ float sigmoid_near(float l)
{
    const float e = exp_near(-__builtin_fabsf(l));  // never overflows
    const float r = 1.0f / (1.0f + e);
    return l != l ? l : (l >= 0.0f ? r : e * r);
}

// What a chosen score l counts beside the others, up to a factor that is the
// same for all of a token; top = the largest of them.  0 for a slot without one.
__device__ __forceinline__ float chosen_share(float l, float top, bool soft)
{
    if (l == -__builtin_inff()) return 0.0f;
    if (l != l) return l;
    float p = l == top ? 1.0f : exp_near(l - top);  // infinite ones too
    // sigmoid(l), or where all are small sigmoid(l) * exp(-top): neither overflows, nor vanishes at the top
    if (!soft) p = top > 0.0f ? sigmoid_near(l) : p / (1.0f + exp_near(l));
    return p;
}

// LDS that only one wavefront uses: its operations happen in order.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// As written, without the steps that the compiler adds for NaN.
__device__ __forceinline__ double max_f64(double a, double b)
{
    double r;
    asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ double min_f64(double a, double b)
{
    double r;
    asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

// exp(x) for x <= 0 to about 2^-46 of itself: 2^n times the first twelve terms of
// the series at |r| <= log(2) / 2, whose remainder is r^12 / 12! < 7e-15.  r comes
// from Cody and Waite's reduction: n times a head of log(2) that is short enough
// for the product to be exact, then n times the rest of it.  No
// branches, so that a lane's exponentials go side by side and share their
// constants.  Below -700, and for NaN, exp(-700): the caller sees to NaN.
__device__ __forceinline__ double exp_wide(double x)
{
    x = max_f64(x, -700.0);
    const double n = __builtin_rint(x * 1.4426950408889634074);
    double r = __builtin_fma(n, -6.93147180369123816490e-01, x);  // the first 32 bits of log(2), and the rest
    r = __builtin_fma(n, -1.90821492927058770002e-10, r);
    double p = 1.0 / 39916800.0;
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)n);
}
// 1 / x, 1 <= x <= 2^11: the instruction's estimate, and two of Newton's steps.
__device__ __forceinline__ double reciprocal_wide(double x)
{
    double y = __builtin_amdgcn_rcp(x);
    y = __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
    return __builtin_fma(__builtin_fma(-x, y, 1.0), y, y);
}

// A choice score and its expert in one double, so that one maximum finds the
// larger score and, of equal ones, the lower expert.  The last 10 bits hold the
// expert or its complement, whichever counts the right way round for the sign;
// a score made from one float has zeros there.  NaN and the infinities, which a
// maximum of doubles would not order, become the largest numbers there are.
constexpr unsigned kNeverChosen = 0xFFEFFFFFu;  // high word of -inf's stand-in
constexpr unsigned kInfinite = 0x7FEFFFFEu, kNotANumber = 0x7FEFFFFFu;
__device__ __forceinline__ double from_words(unsigned hi, unsigned lo)
{
    return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ unsigned high_word(double v) { return (unsigned)(__builtin_bit_cast(unsigned long long, v) >> 32); }
__device__ __forceinline__ unsigned low_word(double v) { return (unsigned)__builtin_bit_cast(unsigned long long, v); }
__device__ __forceinline__ double pack_choice(double c, int expert)
{
    c += 0.0;  // -0 ranks as +0
    unsigned hi = high_word(c), lo = low_word(c);
    if (!(__builtin_fabs(c) < __builtin_inf())) {
        hi = c != c ? kNotANumber : c > 0.0 ? kInfinite : kNeverChosen;
        lo = 0;
    }
    const unsigned tag = (unsigned)(hi >> 31 ? expert : ~expert) & 1023u;
    return from_words(hi, (lo & ~1023u) | tag);
}
__device__ __forceinline__ int expert_of(double v)
{
    return (int)((high_word(v) >> 31 ? low_word(v) : ~low_word(v)) & 1023u);
}
// How near a packed choice score may be to this one and still not be told apart:
// a score is off by 2^-44 of one at most, the tag by 2^-42 of the whole.
__device__ __forceinline__ double doubt(double a) { return 0x1p-38 * max_f64(1.0, __builtin_fabs(a)); }

// The sum of a group's two largest packed choice scores.  Stand-ins are no
// numbers to add: the sum is that of the values which they stand for (-inf where
// the group has one expert or none, inf - inf = NaN), one stand-in for each, so
// that groups with the same sum tie.
__device__ __forceinline__ double sum_of_two(double first, double second)
{
    const unsigned a = high_word(first), b = high_word(second);
    const unsigned stands = a == kNotANumber || (a == kInfinite && b == kNeverChosen) ? kNotANumber
                            : b == kNeverChosen                                       ? kNeverChosen
                            : a == kInfinite                                          ? kInfinite
                                                                                      : 0;
    return stands ? from_words(stands, 0) : first + second;
}
// How near another group's score may be to this one and still not be told apart.
// What a stand-in stands for is known: nothing is near it.
__device__ __forceinline__ double group_doubt(double own) { return __builtin_fabs(own) > 1e300 ? -1.0 : 2.0 * doubt(own); }

// The k best of a token's packed choice scores, held by L lanes with IPL experts
// each (expert lane * IPL + i).  The j-th choice ends up in lane j.  With
// WATCH the (k + 1)-th too; returned are the places j whose choice is too near
// the one before it.
template <int IPL, int L, bool WATCH>
__device__ __forceinline__ unsigned long long choose(double (&v)[IPL], int k, int lane, int &chosen_expert)
{
    unsigned long long close = 0;
    double last = 0.0;
    chosen_expert = -1;
    for (int j = 0; j < k + (WATCH ? 1 : 0); ++j) {
        double m[IPL];
#pragma unroll
        for (int i = 0; i < IPL; ++i) m[i] = v[i];
#pragma unroll
        for (int step = 1; step < IPL; step *= 2)
#pragma unroll
            for (int i = 0; i + step < IPL; i += 2 * step) m[i] = max_f64(m[i], m[i + step]);
        const double best = fold_group<L>(m[0], max_f64);
        const bool is = high_word(best) != kNeverChosen;
        if constexpr (WATCH) {
            if (j > 0 && is && last - best <= doubt(best)) close |= 1ull << j;
            last = best;
        }
        const int e = expert_of(best);
        if (lane == j) chosen_expert = is ? e : -1;
        const int mine = e - lane * IPL;
#pragma unroll
        for (int i = 0; i < IPL; ++i) v[i] = from_words(i == mine ? kNeverChosen : high_word(v[i]), low_word(v[i]));
    }
    return close;
}

// Drops the experts outside the top_groups best groups where a group's experts
// lie in group_lanes whole lanes.  Returns whether that was too near to tell.
template <int IPL, int L, bool WATCH>
__device__ __forceinline__ bool keep_group_lanes(double (&v)[IPL], const RouteShape &sh, int lane,
                                                 double *__restrict__ of_group)
{
    double first = v[0], second = from_words(kNeverChosen, 0);
#pragma unroll
    for (int i = 1; i < IPL; ++i) {
        second = max_f64(second, min_f64(first, v[i]));
        first = max_f64(first, v[i]);
    }
#define MPS_MERGE_STEP(STEP)                                                                              \
    if constexpr (L > STEP) {                                                                             \
        if (sh.group_lanes > STEP) {                                                                      \
            const double low = fold<STEP>(first, min_f64);                                                \
            second = max_f64(low, fold<STEP>(second, max_f64));                                           \
            first = fold<STEP>(first, max_f64);                                                           \
        }                                                                                                 \
    }
    MPS_MERGE_STEP(1) MPS_MERGE_STEP(2) MPS_MERGE_STEP(4) MPS_MERGE_STEP(8) MPS_MERGE_STEP(16) MPS_MERGE_STEP(32)
#undef MPS_MERGE_STEP
    // the largest members carry their experts' numbers, so that of equal groups the lower is larger
    const double own = sh.group_score == MPS_GROUP_TOP2 ? sum_of_two(first, second) : first;
    const int group = lane / sh.group_lanes;
    if (group < sh.groups && lane % sh.group_lanes == 0) of_group[group] = own;
    wave_sync();
    const double apart = group_doubt(own);
    int better = 0, near = 0;
    for (int h = 0; h < sh.groups; ++h) {
        const double x = of_group[h];
        better += x > own || (x == own && h < group);
        if constexpr (WATCH) near += h != group && __builtin_fabs(x - own) <= apart;
    }
    wave_sync();
    if (better >= sh.top_groups || group >= sh.groups) {
#pragma unroll
        for (int i = 0; i < IPL; ++i) v[i] = from_words(kNeverChosen, low_word(v[i]));
    }
    // a kept group that might be behind the border; a group behind it that might be kept is near one
    return WATCH && group < sh.groups && better < sh.top_groups && near > 0 && better + near >= sh.top_groups;
}

// The same where groups and lanes do not fit each other: a group's scores are
// read back from LDS by one lane.  `all`: sh.E values of LDS, `of_group`: sh.groups.
template <int IPL, int L, bool WATCH>
__device__ __forceinline__ bool keep_groups_apart(double (&v)[IPL], const RouteShape &sh, int lane,
                                                  double *__restrict__ all, double *__restrict__ of_group)
{
#pragma unroll
    for (int i = 0; i < IPL; ++i)
        if (lane * IPL + i < sh.E) all[lane * IPL + i] = v[i];
    wave_sync();
    for (int g = lane; g < sh.groups; g += L) {
        double first = from_words(kNeverChosen, 0), second = first;
        for (int i = 0; i < sh.group_size; ++i) {
            const double x = all[g * sh.group_size + i];
            second = max_f64(second, min_f64(first, x));
            first = max_f64(first, x);
        }
        of_group[g] = sh.group_score == MPS_GROUP_TOP2 ? sum_of_two(first, second) : first;
    }
    wave_sync();
    bool close = false;
    for (int g = lane; g < sh.groups; g += L) {
        const double own = of_group[g], apart = group_doubt(own);
        int better = 0, near = 0;
        for (int h = 0; h < sh.groups; ++h) {
            const double x = of_group[h];
            better += x > own || (x == own && h < g);
            if constexpr (WATCH) near += h != g && __builtin_fabs(x - own) <= apart;
        }
        all[g] = better < sh.top_groups ? 1.0 : 0.0;  // groups <= E; the scores have been read
        close |= WATCH && better < sh.top_groups && near > 0 && better + near >= sh.top_groups;
    }
    wave_sync();
    int g = lane * IPL / sh.group_size, left = (g + 1) * sh.group_size - lane * IPL;
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        if (left == 0) {
            ++g;
            left = sh.group_size;
        }
        --left;
        if (g >= sh.groups || all[min(g, sh.groups - 1)] == 0.0) v[i] = from_words(kNeverChosen, low_word(v[i]));
    }
    wave_sync();
    return close;
}

// The same choice without shortcuts, with scores in 64 bits and ties by index,
// for tokens that the above leaves in doubt.  `all`: sh.E scores of LDS,
// `of_group`: sh.groups.
template <typename T, int IPL, int L>
__device__ __forceinline__ int choose_again(const T *__restrict__ row, bool live, const float *__restrict__ bias,
                                            const RouteShape &sh, int lane, bool plain, float largest,
                                            unsigned long long *__restrict__ all, unsigned long long *__restrict__ of_group)
{
    const bool soft = sh.score == MPS_SCORE_SOFTMAX;
    const float minus_inf = -__builtin_inff();
    double sum = 0.0;
    if (soft && !plain) {
#pragma unroll 1
        for (int i = 0; i < IPL; ++i) {
            const int x = lane * IPL + i;
            const float l = live && x < sh.E ? (float)row[x] : minus_inf;
            if (l != minus_inf) sum += exp((double)l - (double)largest);
        }
        sum = group_sum<L>(sum);
    }
    unsigned long long key[IPL];
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        const int x = lane * IPL + i;
        const float l = live && x < sh.E ? (float)row[x] : minus_inf;
        double c = (double)l;
        if (!plain && l != minus_inf) {
            c = soft ? exp(c - (double)largest) / sum : 1.0 / (1.0 + exp(-c));
            if (bias) c = bias[x] == minus_inf ? -__builtin_inf() : c + (double)bias[x];
        }
        key[i] = key_of(c);
    }
    if (sh.groups > 1) {
#pragma unroll
        for (int i = 0; i < IPL; ++i)
            if (lane * IPL + i < sh.E) all[lane * IPL + i] = key[i];
        wave_sync();
        for (int g = lane; g < sh.groups; g += L) {
            unsigned long long first = 0, second = 0;
            for (int i = 0; i < sh.group_size; ++i) {
                const unsigned long long v = all[g * sh.group_size + i];
                second = max(second, min(first, v));
                first = max(first, v);
            }
            of_group[g] = sh.group_score == MPS_GROUP_TOP2 ? key_of(of_key(first) + of_key(second)) : first;
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            const int g = min((lane * IPL + i) / sh.group_size, sh.groups - 1);
            const unsigned long long own = of_group[g];
            int better = 0;
            for (int h = 0; h < sh.groups; ++h) better += of_group[h] > own || (of_group[h] == own && h < g);
            if (better >= sh.top_groups) key[i] = 0;
        }
        wave_sync();
    }
    const int group_base = (threadIdx.x & 63) & ~(L - 1);
    int chosen_expert = -1;
    for (int j = 0; j < sh.k; ++j) {
        unsigned long long m = key[0];
#pragma unroll
        for (int i = 1; i < IPL; ++i) m = max(m, key[i]);
        const unsigned long long best = group_max<L>(m);
        const unsigned long long has = __ballot(m == best) >> group_base;
        const int owner = __ffsll(L == 64 ? has : has & ((1ull << L) - 1)) - 1;
        int at = -1;
        if (lane == owner && best != 0) {
#pragma unroll
            for (int i = IPL - 1; i >= 0; --i)
                if (key[i] == best) at = i;
#pragma unroll
            for (int i = 0; i < IPL; ++i)
                if (i == at) key[i] = 0;
        }
        const int e = __shfl(lane * IPL + at, group_base + owner, 64);
        if (lane == j) chosen_expert = best != 0 ? e : -1;
    }
    return chosen_expert;
}

// One token by L > k lanes; lane j gets the j-th choice and its weight.  The
// scores are read once.  Without a bias and without sums over a group c orders
// as l does, which is exact; else c is formed to 2^-44, and a token where two
// choices are nearer than that and have not the same l and bias, which makes
// them equal, is done again with every bit of a double.
template <typename T, int IPL, int L>
__device__ __forceinline__ void route_token(const T *__restrict__ row, bool live, const float *__restrict__ bias,
                                            const RouteShape &sh, int lane, unsigned long long *__restrict__ mine, int &e,
                                            float &w)
{
    const float minus_inf = -__builtin_inff();
    float l[IPL];
    {
        const int valid = live ? sh.E - lane * IPL : 0;
        if (valid >= IPL) {
            load_vec<T, IPL>(l, row + lane * IPL, valid);
        } else {
#pragma unroll
            for (int i = 0; i < IPL; ++i) l[i] = i < valid ? (float)row[lane * IPL + i] : minus_inf;
        }
    }
    const bool plain = bias == nullptr && (sh.groups <= 1 || sh.group_score == MPS_GROUP_MAX);
    const bool soft = sh.score == MPS_SCORE_SOFTMAX;
    float largest = 0.0f, total = 1.0f;
    if (soft) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < IPL; ++i) m = max(m, key_of(l[i]));
        largest = of_key(group_max<L>(m));
    }
    const bool broken = soft && !(largest < __builtin_inff());  // no softmax over NaN or an infinite score
    double v[IPL];
    if (plain) {
#pragma unroll
        for (int i = 0; i < IPL; ++i) v[i] = (double)l[i];
        if (soft && !sh.renormalise) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < IPL; ++i) sum += l[i] == minus_inf ? 0.0f : exp_near(l[i] - largest);
            total = group_sum<L>(sum);
        }
    } else {
        float b[IPL];
        load_vec<float, IPL>(b, bias + (bias ? lane * IPL : 0), bias ? sh.E - lane * IPL : 0);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            // -inf counts as exp(-700) in the sum, far below its last bit; it is never chosen
            v[i] = exp_wide(soft ? (double)l[i] - (double)largest : -__builtin_fabs((double)l[i]));
            sum += v[i];
        }
        double scale = 1.0;
        if (soft) {
            sum = group_sum<L>(sum);
            scale = 1.0 / sum;
            total = (float)sum;
        }
#pragma unroll
        for (int i = 0; i < IPL; ++i) {
            const double r = soft ? scale : reciprocal_wide(1.0 + v[i]);
            const double s = soft || l[i] < 0.0f ? v[i] * r : r;
            // a mask counts before a NaN, its own or that of the row
            v[i] = l[i] == minus_inf || b[i] == minus_inf ? -__builtin_inf()
                   : broken || l[i] != l[i]               ? __builtin_nan("")
                                                          : s + (double)b[i];
        }
    }
#pragma unroll
    for (int i = 0; i < IPL; ++i) v[i] = pack_choice(v[i], lane * IPL + i);
    bool again = false;
    {
        double *all = reinterpret_cast<double *>(mine), *of_group = all + sh.E;
        if (plain) {
            if (sh.groups > 1 && sh.group_lanes) keep_group_lanes<IPL, L, false>(v, sh, lane, of_group);
            else if (sh.groups > 1) keep_groups_apart<IPL, L, false>(v, sh, lane, all, of_group);
            choose<IPL, L, false>(v, sh.k, lane, e);
        } else {
            if (sh.groups > 1 && sh.group_lanes) again = keep_group_lanes<IPL, L, true>(v, sh, lane, of_group);
            else if (sh.groups > 1) again = keep_groups_apart<IPL, L, true>(v, sh, lane, all, of_group);
            const unsigned long long close = choose<IPL, L, true>(v, sh.k, lane, e);
            if (__any(close != 0)) {
                const float le = e >= 0 ? (float)row[e] : 0.0f, be = e >= 0 && bias ? bias[e] : 0.0f;
                const float lp = __shfl_up(le, 1, L), bp = __shfl_up(be, 1, L);
                again |= (close >> lane & 1) && !(le == lp && be == bp);
            }
            if (lane >= sh.k) e = -1;
        }
    }
    // All tokens of the wavefront go along; one that is not in doubt keeps what it has.
    if (__any(again && live)) {
        const int other = choose_again<T, IPL, L>(row, live, bias, sh, lane, plain, largest, mine, mine + sh.E);
        if (group_max<L>((unsigned)again)) e = other;
    }
    // Lane j weighs the j-th choice.
    const float lj = live && lane < sh.k && e >= 0 ? (float)row[e] : minus_inf;
    if (sh.renormalise) {
        // Relative to the largest chosen score, so that no sum vanishes: softmax
        // is exp(l) up to a factor; so is the sigmoid, times 1 / (1 + exp(l)).
        const float top = of_key(group_max<L>(key_of(lj)));
        const float p = chosen_share(lj, top, soft);
        const float sum = group_sum<L>(p);
        w = p == 0.0f ? 0.0f : p / sum;
    } else {
        w = lj == minus_inf ? 0.0f : (soft ? exp_near(lj - largest) / total : sigmoid_near(lj));
    }
    if (broken) w = __builtin_nanf("");
    w = e < 0 ? 0.0f : w * sh.scale;
}

template <typename T, int IPL, int L>
__global__ __launch_bounds__(kRouteBlock) void route_kernel(const T *__restrict__ scores, const float *__restrict__ bias,
                                                            RouteShape sh, int *__restrict__ expert,
                                                            float *__restrict__ weight)
{
    extern __shared__ unsigned long long route_lds[];
    const int lane = threadIdx.x & (L - 1), in_block = threadIdx.x / L;
    const long long t = block_number() * (kRouteBlock / L) + in_block;
    const bool live = t < sh.T;
    int e;
    float w;
    route_token<T, IPL, L>(scores + (live ? t : 0) * sh.E, live, bias, sh, lane, route_lds + in_block * (sh.E + sh.groups),
                           e, w);
    if (live && lane < sh.k) {
        expert[t * sh.k + lane] = e;
        weight[t * sh.k + lane] = w;
    }
}

// ---------------------------------------------------------------------------
// The matrix by its columns: a stable counting sort of the slots
// ---------------------------------------------------------------------------
constexpr int kSortBlock = 1024;
constexpr int kSortWaves = kSortBlock / 64;
constexpr int kSortMaxChunks = 256;
constexpr int kSortMinChunk = 2048;  // slots of one workgroup
constexpr int kSortAlone = 8192;     // up to here one workgroup alone, in one launch in place of two

inline int sort_chunk(long long M)
{
    const long long least = M <= kSortAlone ? M : kSortMinChunk, share = (M + kSortMaxChunks - 1) / kSortMaxChunks;
    return (int)((std::max(least, std::max(share, 1ll)) + kSortBlock - 1) / kSortBlock * kSortBlock);
}
// wavefronts of a workgroup that count by themselves: as many as fit 64 KB of counters and have slots
inline int sort_waves(int E, int slots)
{
    return std::max(1, std::min(E < 512 ? kSortWaves : kSortWaves / 2, ceil_div(slots, 64)));
}

__device__ __forceinline__ int id_of(int e, int E) { return (unsigned)e < (unsigned)E ? e : E; }

__global__ __launch_bounds__(kSortBlock) void columns_count_kernel(const int *__restrict__ expert, int M, int E, int chunk,
                                                                   int *__restrict__ counts)
{
    extern __shared__ int count_lds[];
    for (int e = threadIdx.x; e <= E; e += kSortBlock) count_lds[e] = 0;
    __syncthreads();
    const long long first = (long long)blockIdx.x * chunk;
    const long long end = min(first + chunk, (long long)M);
    for (long long s = first + threadIdx.x; s < end; s += kSortBlock) atomicAdd(&count_lds[id_of(expert[s], E)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= E; e += kSortBlock) counts[(size_t)blockIdx.x * (E + 1) + e] = count_lds[e];
}

// Exclusive sum of one value per thread over the workgroup (kSortBlock).
__device__ __forceinline__ int block_exclusive_sum(int v, int *__restrict__ wave_sum)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
    }
    if (lane == 63) wave_sum[wave] = x;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < kSortWaves; ++w) before += w < wave ? wave_sum[w] : 0;
    __syncthreads();
    return before + x - v;
}

// Every workgroup places its own chunk of slots.  The place of a slot is the
// number of slots with a smaller expert, plus those of the same expert in
// earlier chunks, in earlier wavefronts of the chunk, and in earlier lanes: no
// order depends on timing.  counts == nullptr: the only chunk there is.
__device__ __forceinline__ void place_chunk(const int *__restrict__ expert, int M, int E, int chunk, int chunks,
                                            const int *__restrict__ counts, int waves, int *__restrict__ expert_ptr,
                                            int *__restrict__ slot, int *__restrict__ pos,
                                            int *__restrict__ place_lds /* waves x (E + 1) */)
{
    __shared__ int wave_sum[kSortWaves];
    __shared__ int part_total[kSortBlock + 1], part_before[kSortBlock + 1];
    const int E1 = E + 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < waves * E1; i += kSortBlock) place_lds[i] = 0;
    __syncthreads();
    const long long block_first = (long long)blockIdx.x * chunk;
    const long long block_end = min(block_first + chunk, (long long)M);
    const int share = ((chunk + waves - 1) / waves + 63) & ~63;
    const long long first = min(block_first + (long long)wave * share, block_end);
    const long long end = wave < waves ? min(first + share, block_end) : first;
    int *hist = place_lds + (wave < waves ? wave : 0) * E1;
    for (long long s = first + lane; s < end; s += 64) atomicAdd(&hist[id_of(expert[s], E)], 1);
    __syncthreads();
    // The other chunks' counts are added up by as many threads as there are, each
    // a share of the chunks of one expert.
    const int parts = max(kSortBlock / E1, 1);
    if (counts) {
        for (int x = threadIdx.x; x < parts * E1; x += kSortBlock) {
            const int part = x / E1, e = x - part * E1;
            int total = 0, before = 0;
#pragma unroll 8
            for (int b = part; b < chunks; b += parts) {
                const int c = counts[(size_t)b * E1 + e];
                total += c;
                before += b < (int)blockIdx.x ? c : 0;
            }
            part_total[x] = total;
            part_before[x] = before;
        }
        __syncthreads();
    }
    // E1 <= 1025: thread x has expert x, the last thread also the 1025th
    int total = 0, before = 0;
    const int e = threadIdx.x;
    if (e < E1) {
        if (counts) {
            for (int x = e; x < parts * E1; x += E1) {
                total += part_total[x];
                before += part_before[x];
            }
        } else {
            for (int w = 0; w < waves; ++w) total += place_lds[w * E1 + e];
        }
    }
    const int base = block_exclusive_sum(e < E1 ? total : 0, wave_sum);
    if (e < E1) {
        if (blockIdx.x == 0) expert_ptr[e] = base;  // [E] = where the slots without an expert begin
        int at = base + before;
        for (int w = 0; w < waves; ++w) {
            const int c = place_lds[w * E1 + e];
            place_lds[w * E1 + e] = at;
            at += c;
        }
    }
    if (E1 > kSortBlock && threadIdx.x == kSortBlock - 1) {  // E = 1024: the slots without an expert
        const int last = base + total;
        if (blockIdx.x == 0) expert_ptr[E] = last;
        int at = last + (counts ? part_before[E] : 0);
        for (int w = 0; w < waves; ++w) {
            const int c = place_lds[w * E1 + E];
            place_lds[w * E1 + E] = at;
            at += c;
        }
    }
    __syncthreads();
    int bits = 32 - __clz(E);  // ids 0 .. E
    for (long long s0 = first; s0 < end; s0 += 64) {
        const long long s = s0 + lane;
        const bool in = s < end;
        const int id = in ? id_of(expert[s], E) : 0;
        unsigned long long same = __ballot(in);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long set = __ballot((id >> b) & 1);
            same &= (id >> b) & 1 ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int at = in ? hist[id] : 0;
        wave_sync();
        if (in && rank == 0) hist[id] = at + __popcll(same);
        wave_sync();
        if (in) {
            slot[at + rank] = (int)s;
            pos[s] = id < E ? at + rank : -1;
        }
    }
}

__global__ __launch_bounds__(kSortBlock) void columns_place_kernel(const int *__restrict__ expert, int M, int E, int chunk,
                                                                   int chunks, const int *__restrict__ counts, int waves,
                                                                   int *__restrict__ expert_ptr, int *__restrict__ slot,
                                                                   int *__restrict__ pos)
{
    extern __shared__ int place_lds[];
    place_chunk(expert, M, E, chunk, chunks, counts, waves, expert_ptr, slot, pos, place_lds);
}

// Rows and columns of a few tokens in one launch, where launches and latency are
// the time: one workgroup, a wavefront for every token in turn, so that a lane
// has few experts; the choices stay in LDS for the columns.
constexpr int kFewTokens = 16;

template <typename T, int IPL>
__global__ __launch_bounds__(kSortBlock) void route_few_kernel(const T *__restrict__ scores, const float *__restrict__ bias,
                                                               RouteShape sh, int *__restrict__ expert,
                                                               float *__restrict__ weight, int waves,
                                                               int *__restrict__ expert_ptr, int *__restrict__ slot,
                                                               int *__restrict__ pos)
{
    extern __shared__ unsigned long long route_lds[];
    __shared__ int ids[kFewTokens * MPS_ROUTE_MAX_K];
    const int lane = threadIdx.x & 63, t = threadIdx.x >> 6;
    if (t < sh.T) {
        int e;
        float w;
        route_token<T, IPL, 64>(scores + (size_t)t * sh.E, true, bias, sh, lane, route_lds + t * (sh.E + sh.groups), e, w);
        if (lane < sh.k) {
            expert[t * sh.k + lane] = e;
            weight[t * sh.k + lane] = w;
            ids[t * sh.k + lane] = e;
        }
    }
    __syncthreads();
    place_chunk(ids, sh.T * sh.k, sh.E, sh.T * sh.k, 1, nullptr, waves, expert_ptr, slot, pos,
                reinterpret_cast<int *>(route_lds));
}
static_assert(kFewTokens <= kSortWaves, "a wavefront for every token");

int launch_columns(const int *expert, int M, int E, int *expert_ptr, int *slot, int *pos, void *workspace,
                   hipStream_t st)
{
    const int chunk = sort_chunk(M);
    const int chunks = M > 0 ? ceil_div(M, chunk) : 1;
    const int waves = sort_waves(E, chunk);
    int *counts = chunks > 1 ? static_cast<int *>(workspace) : nullptr;
    if (counts) {
        hipLaunchKernelGGL(columns_count_kernel, dim3(chunks), dim3(kSortBlock), (E + 1) * sizeof(int), st, expert, M, E,
                           chunk, counts);
        MPS_HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL(columns_place_kernel, dim3(chunks), dim3(kSortBlock), (size_t)waves * (E + 1) * sizeof(int), st,
                       expert, M, E, chunk, chunks, counts, waves, expert_ptr, slot, pos);
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

size_t columns_workspace(int M, int E)
{
    const int chunks = M > 0 ? ceil_div(M, sort_chunk(M)) : 1;
    return chunks > 1 ? (size_t)chunks * (E + 1) * sizeof(int) : 0;
}

// ---------------------------------------------------------------------------
// Gradient of the scores
// ---------------------------------------------------------------------------

// One token by 64 lanes.  With s the scores, w = scale * s / sum or scale * s,
// g = dL/dw:
//   softmax      dl_e = s_e (scale g_e - D),  D = sum_j scale s_j g_j
//   sigmoid      dl_j = scale g_j s_j (1 - s_j)
//   renormalised dlog s_j = w_j (g_j - D / scale),  D = sum_j w_j g_j
//                dl_j = dlog s_j (softmax), dlog s_j (1 - s_j) (sigmoid)
// Only the first touches experts that were not chosen, and only it reads the
// whole row.
template <typename T>
__global__ __launch_bounds__(kRouteBlock) void route_backward_kernel(const T *__restrict__ scores,
                                                                     const int *__restrict__ expert,
                                                                     const float *__restrict__ dweight, RouteShape sh,
                                                                     T *__restrict__ dscores)
{
    const int lane = threadIdx.x & 63;
    const long long t = block_number() * (kRouteBlock / 64) + (threadIdx.x >> 6);
    if (t >= sh.T) return;
    const T *row = scores + t * sh.E;
    T *out = dscores + t * sh.E;
    const bool soft = sh.score == MPS_SCORE_SOFTMAX;
    const bool whole = soft && !sh.renormalise;
    const float minus_inf = -__builtin_inff();
    int e = lane < sh.k ? expert[t * sh.k + lane] : -1;
    if ((unsigned)e >= (unsigned)sh.E) e = -1;
    const float lj = e >= 0 ? (float)row[e] : minus_inf;
    const float g = e >= 0 ? dweight[t * sh.k + lane] : 0.0f;
    float largest = 0.0f, total = 1.0f;
    if (whole) {
        unsigned m = 0;
        for (int i = lane; i < sh.E; i += 64) m = max(m, key_of((float)row[i]));
        largest = of_key(group_max<64>(m));
        float sum = 0.0f;
        for (int i = lane; i < sh.E; i += 64) {
            const float l = (float)row[i];
            sum += l == minus_inf ? 0.0f : exp_near(l - largest);
        }
        total = group_sum<64>(sum);
    }
    float part;  // of dl at this lane's choice
    float mean = 0.0f;
    if (sh.renormalise) {
        const float top = of_key(group_max<64>(key_of(lj)));
        const float p = chosen_share(lj, top, soft);
        const float sum = group_sum<64>(p);
        const float w = p == 0.0f ? 0.0f : p / sum;
        mean = group_sum<64>(w == 0.0f ? 0.0f : w * g);
        part = w == 0.0f ? 0.0f : sh.scale * w * (g - mean);
        if (!soft && part != 0.0f) part *= sigmoid_near(-lj);
    } else if (soft) {
        const float s = lj == minus_inf ? 0.0f : exp_near(lj - largest) / total;
        mean = group_sum<64>(s == 0.0f ? 0.0f : s * g);
        part = s == 0.0f ? 0.0f : sh.scale * s * g;
    } else {
        part = lj == minus_inf ? 0.0f : sh.scale * g * sigmoid_near(lj) * sigmoid_near(-lj);
    }
    for (int i0 = 0; i0 < sh.E; i0 += 64) {
        const int i = i0 + lane;
        float d = 0.0f;
        if (whole && i < sh.E) {
            const float l = (float)row[i];
            d = l == minus_inf ? 0.0f : -(exp_near(l - largest) / total) * (sh.scale * mean);
        }
        for (int j = 0; j < sh.k; ++j) {
            const int ej = __builtin_amdgcn_readlane(e, j);
            const float pj = bits_float(__builtin_amdgcn_readlane(float_bits(part), j));
            if (ej == i) d += pj;
        }
        if (i < sh.E) out[i] = (T)d;
    }
}

// ---------------------------------------------------------------------------
// Combination
// ---------------------------------------------------------------------------

// Y[t] = base[t] + sum_j w[t, j] Z[pos[t, j]]: one lane per 16 bytes of a row
// of Y.  Bound by the bytes of Z and Y: 8192 tokens, k = 6, 2048 bf16 take 52 us,
// 4.3 TB/s.  A lane has one of its k loads on its way at a time, since the compiler
// waits for each at the end of the branch that tells whole chunks from a row's
// last part; the other wavefronts fill the time.
template <typename T>
__global__ __launch_bounds__(256) void combine_kernel(const T *__restrict__ Z, const int *__restrict__ pos,
                                                      const float *__restrict__ weight, const T *base, T *Y, int T_,
                                                      int k, int M, int N, int per_row)
{
    constexpr int V = 16 / sizeof(T);
    const long long item = block_number() * 256 + threadIdx.x;
    const long long t = item / per_row;
    if (t >= T_) return;
    const int col = (int)(item - t * per_row) * V;
    const int valid = N - col;
    float acc[V];
    if (base) load_vec<T, V>(acc, base + t * N + col, valid);
    else {
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    }
    for (int j0 = 0; j0 < k; j0 += 4) {
        int p[4];
        float w[4], z[4][V];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            p[j] = j0 + j < k ? pos[t * k + j0 + j] : -1;
            if ((unsigned)p[j] >= (unsigned)M) p[j] = -1;
            w[j] = p[j] < 0 ? 0.0f : weight ? weight[t * k + j0 + j] : 1.0f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (p[j] >= 0) load_vec<T, V>(z[j], Z + (long long)p[j] * N + col, valid);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (p[j] >= 0) {
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = __builtin_fmaf(w[j], z[j][i], acc[i]);
            }
    }
    store_vec<T, V>(Y + t * N + col, acc, valid);
}

// L lanes per place, a wavefront or for narrow rows less: they read the row of Z
// and the token's row of dY, write the row of dZ and the product of the two
// rows.  Places are in order, so Z and dZ stream; the k reads of a row of dY meet
// in the caches.  4099 tokens, k = 8, fp16, the same buffers in every call: rows of
// 1024 35.8 us (4.0 TB/s), 1032 40.6, 1030 48.0 (3.0 TB/s): the last part of a row
// is a turn of its own, and rows that are not whole 16 bytes cost a fifth more.
template <typename T, int L>
__global__ __launch_bounds__(256) void combine_backward_kernel(const T *__restrict__ dY, const T *__restrict__ Z,
                                                               const float *__restrict__ weight,
                                                               const int *__restrict__ expert_ptr, int E,
                                                               const int *__restrict__ slot, T *__restrict__ dZ,
                                                               float *__restrict__ dweight, int k, int M, int N)
{
    constexpr int V = 16 / sizeof(T);
    const int lane = threadIdx.x & (L - 1);
    const long long at = block_number() * (256 / L) + threadIdx.x / L;
    if (at >= M) return;
    const int p = (int)at;
    const int s = slot[p];
    const bool known = (unsigned)s < (unsigned)M;
    const bool routed = known && p < expert_ptr[E];
    const float w = routed ? (weight ? weight[s] : 1.0f) : 0.0f;
    const T *y_row = dY + (long long)(routed ? s / k : 0) * N;
    const T *z_row = Z + (long long)p * N;
    T *out = dZ + (long long)p * N;
    // A load behind a store waits for it, so that several chunks of both rows are
    // loaded before any is stored.  (One after the other: see combine_kernel.)
    constexpr int U = L == 64 ? 4 : 1;
    float dot = 0.0f;
    for (int first = lane * V; first < N; first += U * L * V) {
        float y[U][V], z[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = first + u * L * V;
            load_vec<T, V>(y[u], y_row + col, routed ? N - col : 0);
            load_vec<T, V>(z[u], z_row + col, routed && dweight ? N - col : 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = first + u * L * V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dot = __builtin_fmaf(y[u][i], z[u][i], dot);
                y[u][i] = routed ? y[u][i] * w : 0.0f;
            }
            if (col < N) store_vec<T, V>(out + col, y[u], N - col);
        }
    }
    if (dweight && known) {
        dot = group_sum<L>(dot);
        if (lane == 0) dweight[s] = routed ? dot : 0.0f;
    }
}

int check_options(const mps_route_options *o, int T, int E, bool choice)
{
    if (!o || T < 0 || E < 1 || o->k < 1 || o->k > E) return MPS_ERR_INVALID_ARG;
    if (o->score != MPS_SCORE_SOFTMAX && o->score != MPS_SCORE_SIGMOID) return MPS_ERR_INVALID_ARG;
    if (E > MPS_ROUTE_MAX_EXPERTS || o->k > MPS_ROUTE_MAX_K || (long long)T * o->k > INT_MAX - 65536)
        return MPS_ERR_UNSUPPORTED;
    if (choice && o->groups > 1) {
        if (o->groups > MPS_ROUTE_MAX_GROUPS) return MPS_ERR_UNSUPPORTED;
        if (E % o->groups || o->top_groups < 1 || o->top_groups > o->groups) return MPS_ERR_INVALID_ARG;
        if (o->group_score != MPS_GROUP_MAX && o->group_score != MPS_GROUP_TOP2) return MPS_ERR_INVALID_ARG;
        if (o->group_score == MPS_GROUP_TOP2 && E / o->groups < 2) return MPS_ERR_INVALID_ARG;
        if ((long long)o->top_groups * (E / o->groups) < o->k) return MPS_ERR_INVALID_ARG;
    }
    return MPS_OK;
}

RouteShape make_shape(const mps_route_options &o, int T, int E)
{
    const int groups = o.groups > 1 && o.top_groups < o.groups ? o.groups : 1;
    return RouteShape{T, E, o.k, o.score, groups, E / groups, o.top_groups, o.group_score, o.renormalise, o.scale, 0};
}

// Lanes and experts per lane for a token: 16 lanes do four tokens in a wavefront,
// and their maxima cross lanes in four cheap steps (16384 tokens of 256 experts
// with a bias and groups: 21 us on the GPU, 43 with 64 lanes and scores in 32
// bits); more where the experts or the choices need them.
template <typename F>
int with_route_lanes(const RouteShape &sh, F &&f)
{
#define MPS_LANES(IPL, L) f(std::integral_constant<int, IPL>{}, std::integral_constant<int, L>{})
    if (sh.k < 16) {
        if (sh.E <= 16) return MPS_LANES(1, 16);
        if (sh.E <= 64) return MPS_LANES(4, 16);
        if (sh.E <= 128) return MPS_LANES(8, 16);
        if (sh.E <= 256) return MPS_LANES(16, 16);
    } else if (sh.k < 32 && sh.E <= 256) {
        return MPS_LANES(8, 32);
    }
    if (sh.k < 32 && sh.E <= 512) return MPS_LANES(16, 32);
    return MPS_LANES(16, 64);
#undef MPS_LANES
}

// `columns`: where rows and columns were made by one launch.
template <typename T>
int launch_route(const T *scores, const float *bias, RouteShape sh, int *expert, float *weight, int *expert_ptr,
                 int *slot, int *pos, bool &columns, hipStream_t st)
{
    const size_t per_token = (size_t)(sh.groups > 1 ? sh.E + sh.groups : 0) * sizeof(unsigned long long);
    auto fit_groups = [&](int ipl) {
        const int lanes = sh.group_size / ipl;
        sh.group_lanes = sh.groups > 1 && sh.group_size % ipl == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    };
    if (expert_ptr && sh.T <= (sh.E <= 256 ? kFewTokens : kFewTokens / 4)) {
        const int waves = sort_waves(sh.E, sh.T * sh.k);
        const size_t lds = std::max(per_token * (sh.T + 1), (size_t)waves * (sh.E + 1) * sizeof(int));
        columns = true;
#define MPS_LAUNCH_FEW(IPL)                                                                                         \
    fit_groups(IPL);                                                                                                \
    hipLaunchKernelGGL((route_few_kernel<T, IPL>), dim3(1), dim3(kSortBlock), lds, st, scores, bias, sh, expert,    \
                       weight, waves, expert_ptr, slot, pos)
        if (sh.E <= 64) { MPS_LAUNCH_FEW(1); }
        else if (sh.E <= 256) { MPS_LAUNCH_FEW(4); }
        else { MPS_LAUNCH_FEW(16); }
#undef MPS_LAUNCH_FEW
        MPS_HIP_TRY(hipGetLastError());
        return MPS_OK;
    }
    return with_route_lanes(sh, [&](auto ipl, auto lanes) -> int {
        constexpr int IPL = decltype(ipl)::value, L = decltype(lanes)::value;
        fit_groups(IPL);
        hipLaunchKernelGGL((route_kernel<T, IPL, L>), grid_of(ceil_div(sh.T, kRouteBlock / L)), dim3(kRouteBlock),
                           per_token * (kRouteBlock / L), st, scores, bias, sh, expert, weight);
        MPS_HIP_TRY(hipGetLastError());
        return MPS_OK;
    });
}

template <typename T>
int launch_combine(const void *Z, const int *pos, const float *weight, const void *base, void *Y, int T_, int k, int M,
                   int N, hipStream_t st)
{
    const int per_row = ceil_div(N, 16 / (int)sizeof(T));
    const long long blocks = ((long long)T_ * per_row + 255) / 256;
    if (blocks > INT_MAX) return MPS_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((combine_kernel<T>), grid_of(blocks), dim3(256), 0, st, static_cast<const T *>(Z), pos, weight,
                       static_cast<const T *>(base), static_cast<T *>(Y), T_, k, M, N, per_row);
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

template <typename T>
int launch_combine_backward(const void *dY, const void *Z, const float *weight, const int *expert_ptr, int E,
                            const int *slot, void *dZ, float *dweight, int k, int M, int N, hipStream_t st)
{
    // as many lanes as a row has chunks (34076 places of 39 columns bf16: 10.6 us a call, 29.7 with 64)
    const int chunks = ceil_div(N, 16 / (int)sizeof(T));
#define MPS_LAUNCH_LANES(L)                                                                                            \
    hipLaunchKernelGGL((combine_backward_kernel<T, L>), grid_of(ceil_div(M, 256 / L)), dim3(256), 0, st,               \
                       static_cast<const T *>(dY), static_cast<const T *>(Z), weight, expert_ptr, E, slot,             \
                       static_cast<T *>(dZ), dweight, k, M, N)
    if (chunks <= 8) MPS_LAUNCH_LANES(8);
    else if (chunks <= 16) MPS_LAUNCH_LANES(16);
    else if (chunks <= 32) MPS_LAUNCH_LANES(32);
    else MPS_LAUNCH_LANES(64);
#undef MPS_LAUNCH_LANES
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

}  // namespace

extern "C" {

int mps_route_workspace_bytes(int T, int E, int k, size_t *bytes_out)
{
    if (!bytes_out || T < 0 || E < 1 || k < 1) return MPS_ERR_INVALID_ARG;
    if (E > MPS_ROUTE_MAX_EXPERTS || (long long)T * k > INT_MAX - 65536) return MPS_ERR_UNSUPPORTED;
    *bytes_out = columns_workspace(T * k, E);
    return MPS_OK;
}

int mps_route_columns(const int *d_expert, int T, int E, int k, int *d_expert_ptr, int *d_slot, int *d_pos,
                      void *d_workspace, size_t workspace_bytes, void *stream)
{
    size_t need = 0;
    const int rc = mps_route_workspace_bytes(T, E, k, &need);
    if (rc != MPS_OK) return rc;
    if (!d_expert_ptr || (T > 0 && (!d_expert || !d_slot || !d_pos))) return MPS_ERR_INVALID_ARG;
    if (!aligned_to(d_expert, 4) || !aligned_to(d_expert_ptr, 4) || !aligned_to(d_slot, 4) || !aligned_to(d_pos, 4) ||
        (need > 0 && !aligned_to(d_workspace, 16)))
        return MPS_ERR_ALIGNMENT;
    if (need > 0 && (!d_workspace || workspace_bytes < need)) return MPS_ERR_WORKSPACE;
    return launch_columns(d_expert, T * k, E, d_expert_ptr, d_slot, d_pos, d_workspace,
                          static_cast<hipStream_t>(stream));
}

int mps_route(const void *d_scores, int dtype, const float *d_bias, int T, int E, const mps_route_options *options,
              int *d_expert, float *d_weight, int *d_expert_ptr, int *d_slot, int *d_pos, void *d_workspace,
              size_t workspace_bytes, void *stream)
{
    const int rc = check_options(options, T, E, true);
    if (rc != MPS_OK) return rc;
    const int eb = dtype_bytes(dtype);
    if (!eb || (T > 0 && (!d_scores || !d_expert || !d_weight))) return MPS_ERR_INVALID_ARG;
    const bool columns = d_expert_ptr || d_slot || d_pos;
    if (columns && (!d_expert_ptr || (T > 0 && (!d_slot || !d_pos)))) return MPS_ERR_INVALID_ARG;
    if (!aligned_to(d_scores, eb) || !aligned_to(d_bias, 4) || !aligned_to(d_expert, 4) || !aligned_to(d_weight, 4) ||
        !aligned_to(d_expert_ptr, 4) || !aligned_to(d_slot, 4) || !aligned_to(d_pos, 4))
        return MPS_ERR_ALIGNMENT;
    const int M = T * options->k;
    if (columns) {
        const size_t need = columns_workspace(M, E);
        if (need > 0 && (!d_workspace || workspace_bytes < need)) return MPS_ERR_WORKSPACE;
        if (need > 0 && !aligned_to(d_workspace, 16)) return MPS_ERR_ALIGNMENT;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    bool done = false;
    if (T > 0) {
        const RouteShape sh = make_shape(*options, T, E);
        auto run = [&](auto *scores) {
            return launch_route(scores, d_bias, sh, d_expert, d_weight, d_expert_ptr, d_slot, d_pos, done, st);
        };
        const int r = dtype == MPS_F32   ? run(static_cast<const float *>(d_scores))
                      : dtype == MPS_F16 ? run(static_cast<const half_t *>(d_scores))
                                         : run(static_cast<const bf16_t *>(d_scores));
        if (r != MPS_OK || done) return r;
    }
    return columns ? launch_columns(d_expert, M, E, d_expert_ptr, d_slot, d_pos, d_workspace, st) : MPS_OK;
}

int mps_route_backward(const void *d_scores, int dtype, const int *d_expert, const float *d_dweight, int T, int E,
                       const mps_route_options *options, void *d_dscores, void *stream)
{
    const int rc = check_options(options, T, E, false);
    if (rc != MPS_OK) return rc;
    const int eb = dtype_bytes(dtype);
    if (!eb || (T > 0 && (!d_scores || !d_expert || !d_dweight || !d_dscores))) return MPS_ERR_INVALID_ARG;
    if (!aligned_to(d_scores, eb) || !aligned_to(d_expert, 4) || !aligned_to(d_dweight, 4) || !aligned_to(d_dscores, eb))
        return MPS_ERR_ALIGNMENT;
    if (T == 0) return MPS_OK;
    RouteShape sh = make_shape(*options, T, E);
    hipStream_t st = static_cast<hipStream_t>(stream);
#define MPS_LAUNCH_BACKWARD(TYPE)                                                                                  \
    hipLaunchKernelGGL((route_backward_kernel<TYPE>), grid_of(ceil_div(T, kRouteBlock / 64)), dim3(kRouteBlock), 0, st, \
                       static_cast<const TYPE *>(d_scores), d_expert, d_dweight, sh, static_cast<TYPE *>(d_dscores))
    if (dtype == MPS_F32) MPS_LAUNCH_BACKWARD(float);
    else if (dtype == MPS_F16) MPS_LAUNCH_BACKWARD(half_t);
    else MPS_LAUNCH_BACKWARD(bf16_t);
#undef MPS_LAUNCH_BACKWARD
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

int mps_combine(const void *d_Z, const int *d_pos, const float *d_weight, const void *d_base, void *d_Y, int dtype,
                int T, int k, int M, int N, void *stream)
{
    const int eb = dtype_bytes(dtype);
    if (!eb || T < 0 || k < 1 || M < 0 || N < 1) return MPS_ERR_INVALID_ARG;
    if ((long long)T * k > INT_MAX - 65536) return MPS_ERR_UNSUPPORTED;
    if (T > 0 && (!d_pos || !d_Y || (M > 0 && !d_Z))) return MPS_ERR_INVALID_ARG;
    if (!aligned_to(d_Z, eb) || !aligned_to(d_pos, 4) || !aligned_to(d_weight, 4) || !aligned_to(d_base, eb) ||
        !aligned_to(d_Y, eb))
        return MPS_ERR_ALIGNMENT;
    if (T == 0) return MPS_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == MPS_F32) return launch_combine<float>(d_Z, d_pos, d_weight, d_base, d_Y, T, k, M, N, st);
    if (dtype == MPS_F16) return launch_combine<half_t>(d_Z, d_pos, d_weight, d_base, d_Y, T, k, M, N, st);
    return launch_combine<bf16_t>(d_Z, d_pos, d_weight, d_base, d_Y, T, k, M, N, st);
}

int mps_combine_backward(const void *d_dY, const void *d_Z, const float *d_weight, const int *d_expert_ptr, int E,
                         const int *d_slot, void *d_dZ, float *d_dweight, int dtype, int T, int k, int N, void *stream)
{
    const int eb = dtype_bytes(dtype);
    if (!eb || T < 0 || E < 1 || k < 1 || N < 1) return MPS_ERR_INVALID_ARG;
    if ((long long)T * k > INT_MAX - 65536) return MPS_ERR_UNSUPPORTED;
    if (T > 0 && (!d_dY || !d_expert_ptr || !d_slot || !d_dZ || (d_dweight && !d_Z))) return MPS_ERR_INVALID_ARG;
    if (!aligned_to(d_dY, eb) || !aligned_to(d_Z, eb) || !aligned_to(d_weight, 4) || !aligned_to(d_expert_ptr, 4) ||
        !aligned_to(d_slot, 4) || !aligned_to(d_dZ, eb) || !aligned_to(d_dweight, 4))
        return MPS_ERR_ALIGNMENT;
    if (T == 0) return MPS_OK;
    const int M = T * k;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == MPS_F32)
        return launch_combine_backward<float>(d_dY, d_Z, d_weight, d_expert_ptr, E, d_slot, d_dZ, d_dweight, k, M, N, st);
    if (dtype == MPS_F16)
        return launch_combine_backward<half_t>(d_dY, d_Z, d_weight, d_expert_ptr, E, d_slot, d_dZ, d_dweight, k, M, N, st);
    return launch_combine_backward<bf16_t>(d_dY, d_Z, d_weight, d_expert_ptr, E, d_slot, d_dZ, d_dweight, k, M, N, st);
}

}  // extern "C"
