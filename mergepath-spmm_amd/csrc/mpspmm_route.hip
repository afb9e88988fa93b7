// Routing matrices of language models: choice of the experts, the matrix by
// its columns (a stable counting sort), the gradient of the scores, and the
// product of the matrix with the experts' rows (combination) with its
// gradients.
#include "mpspmm_routing.hpp"

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
template <typename S>
struct KeyOf;
template <>
struct KeyOf<float> {
    using type = unsigned;
};
template <>
struct KeyOf<double> {
    using type = unsigned long long;
};

struct RouteShape {
    int T, E, k, score, groups, group_size, top_groups, group_score, renormalise;
    float scale;
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
__device__ __forceinline__ double sigmoid_f64(double l) { return 1.0 / (1.0 + exp(-l)); }

// How far two choice scores formed in 32 bits may be off together: the score
// itself by less than 2^-22 (see exp_near; sigmoid and softmax are at most
// 1), the sum with the bias by half a step.  Twice that, for both sides, and
// some room.
__device__ __forceinline__ float doubt(float a, float b)
{
    return 0x1p-20f * fmaxf(1.0f, fmaxf(__builtin_fabsf(a), __builtin_fabsf(b)));
}

// The k best of a token's keys, held by L lanes with IPL experts each (expert
// lane * IPL + i).  The j-th choice ends up in lane j.  With WATCH, returns
// true where a decision was closer than 32 bits can tell.
template <typename S, int IPL, int L, bool WATCH>
__device__ __forceinline__ bool choose(typename KeyOf<S>::type (&key)[IPL], const RouteShape &sh, int lane,
                                       int &chosen_expert)
{
    using Key = typename KeyOf<S>::type;
    const int group_base = (threadIdx.x & 63) & ~(L - 1);
    bool close = false;
    Key last = 0;
    chosen_expert = -1;
    for (int j = 0; j < sh.k + (WATCH ? 1 : 0); ++j) {
        Key m = key[0];
#pragma unroll
        for (int i = 1; i < IPL; ++i) m = max(m, key[i]);
        const Key best = group_max<L>(m);
        if constexpr (WATCH) {
            if (j > 0 && best != 0) {
                const float a = (float)of_key(last), b = (float)of_key(best);
                close |= a - b <= doubt(a, b);
            }
            last = best;
            if (j == sh.k) break;
        }
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
    return close;
}

// Zeroes the keys of the experts outside the top_groups best groups.  `mine`:
// this token's part of LDS, 2 * groups values of S.
template <typename S, int IPL, int L, bool WATCH>
__device__ __forceinline__ bool keep_groups(typename KeyOf<S>::type (&key)[IPL], const RouteShape &sh, int lane,
                                            typename KeyOf<S>::type *__restrict__ all,
                                            typename KeyOf<S>::type *__restrict__ of_group)
{
    using Key = typename KeyOf<S>::type;
#pragma unroll
    for (int i = 0; i < IPL; ++i)
        if (lane * IPL + i < sh.E) all[lane * IPL + i] = key[i];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    for (int g = lane; g < sh.groups; g += L) {
        Key first = 0, second = 0;
        for (int i = 0; i < sh.group_size; ++i) {
            const Key v = all[g * sh.group_size + i];
            second = max(second, min(first, v));
            first = max(first, v);
        }
        of_group[g] = sh.group_score == MPS_GROUP_TOP2 ? key_of((S)(of_key(first) + of_key(second))) : first;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    bool close = false;
    unsigned long long kept = 0;
    for (int g = lane; g < sh.groups; g += L) {
        const Key own = of_group[g];
        int better = 0, surely = 0;
        for (int h = 0; h < sh.groups; ++h) {
            const Key v = of_group[h];
            better += v > own || (v == own && h < g);
            if constexpr (WATCH) {
                // groups that are better by more than the doubt; the others might be worse
                const float a = (float)of_key(v), b = (float)of_key(own);
                surely += h != g && v != 0 && own != 0 && __builtin_fabsf(a - b) <= 2.0f * doubt(a, b);
            }
        }
        // in doubt where a group near this one might change its side of the border
        if (WATCH && surely != 0 && better <= sh.top_groups && better + surely >= sh.top_groups - 1) close = true;
        if (better < sh.top_groups) kept |= 1ull << g;
    }
    unsigned lo = (unsigned)kept, hi = (unsigned)(kept >> 32);
#define MPS_OR_STEP(STEP)                                  \
    if constexpr (L > STEP) {                              \
        lo |= lane_partner<STEP>(lo);                      \
        hi |= lane_partner<STEP>(hi);                      \
    }
    MPS_OR_STEP(1) MPS_OR_STEP(2) MPS_OR_STEP(4) MPS_OR_STEP(8) MPS_OR_STEP(16) MPS_OR_STEP(32)
#undef MPS_OR_STEP
    kept = ((unsigned long long)hi << 32) | lo;
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        const int g = min((lane * IPL + i) / sh.group_size, sh.groups - 1);
        if (!((kept >> g) & 1)) key[i] = 0;
    }
    return close;
}

// One token by L lanes.  The scores are read once.  Without a bias and without
// sums over a group c orders as l does, which is exact; else c is formed in 32
// bits, and a token in which a decision falls by less than their error is done
// again in 64 bits: the choice is that of 64 bits, at the cost of 32.
template <typename T, int IPL, int L>
__global__ __launch_bounds__(kRouteBlock) void route_kernel(const T *__restrict__ scores, const float *__restrict__ bias,
                                                            RouteShape sh, int *__restrict__ expert,
                                                            float *__restrict__ weight)
{
    extern __shared__ unsigned long long route_lds[];
    constexpr int kTokens = kRouteBlock / L;
    const int lane = threadIdx.x & (L - 1);
    const int in_block = threadIdx.x / L;
    const long long t = (long long)blockIdx.x * kTokens + in_block;
    const bool live = t < sh.T;
    const T *row = scores + (live ? t : 0) * sh.E;
    unsigned long long *mine = route_lds + in_block * (sh.E + sh.groups);

    float l[IPL];
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        const int e = lane * IPL + i;
        l[i] = live && e < sh.E ? (float)row[e] : -__builtin_inff();
    }
    const bool plain = bias == nullptr && (sh.groups <= 1 || sh.group_score == MPS_GROUP_MAX);
    const bool soft = sh.score == MPS_SCORE_SOFTMAX;
    float largest = 0.0f, total = 1.0f;
    if (soft) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < IPL; ++i) m = max(m, key_of(l[i]));
        largest = of_key(group_max<L>(m));
        if (!plain || !sh.renormalise) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < IPL; ++i) sum += l[i] == -__builtin_inff() ? 0.0f : exp_near(l[i] - largest);
            total = group_sum<L>(sum);
        }
    }
    unsigned key[IPL];
#pragma unroll
    for (int i = 0; i < IPL; ++i) {
        float c = l[i];
        if (!plain && c != -__builtin_inff()) {
            c = soft ? exp_near(c - largest) / total : sigmoid_near(c);
            if (bias) c += bias[lane * IPL + i];
        }
        key[i] = key_of(c);
    }
    int e;
    bool close = false;
    if (plain) {
        if (sh.groups > 1)
            keep_groups<float, IPL, L, false>(key, sh, lane, reinterpret_cast<unsigned *>(mine),
                                              reinterpret_cast<unsigned *>(mine) + sh.E);
        choose<float, IPL, L, false>(key, sh, lane, e);
    } else {
        if (sh.groups > 1)
            close = keep_groups<float, IPL, L, true>(key, sh, lane, reinterpret_cast<unsigned *>(mine),
                                                     reinterpret_cast<unsigned *>(mine) + sh.E);
        close |= choose<float, IPL, L, true>(key, sh, lane, e);
        if (__any(close && live)) {
            double sum = 1.0;
            if (soft) {
                sum = 0.0;
#pragma unroll
                for (int i = 0; i < IPL; ++i)
                    if (l[i] != -__builtin_inff()) sum += exp((double)l[i] - (double)largest);
                sum = group_sum<L>(sum);
            }
            unsigned long long key2[IPL];
#pragma unroll
            for (int i = 0; i < IPL; ++i) {
                double c = -__builtin_inf();
                if (l[i] != -__builtin_inff()) {
                    c = soft ? exp((double)l[i] - (double)largest) / sum : sigmoid_f64((double)l[i]);
                    if (bias) c += (double)bias[lane * IPL + i];
                }
                key2[i] = key_of(c);
            }
            if (sh.groups > 1) keep_groups<double, IPL, L, false>(key2, sh, lane, mine, mine + sh.E);
            int e2;
            choose<double, IPL, L, false>(key2, sh, lane, e2);
            e = e2;
        }
    }
    // Lane j weighs the j-th choice.
    const float lj = live && lane < sh.k && e >= 0 ? (float)row[e] : -__builtin_inff();
    float w;
    if (sh.renormalise) {
        // Relative to the largest chosen score, so that no sum vanishes: softmax
        // is exp(l) up to a factor; so is the sigmoid, times 1 / (1 + exp(l)).
        unsigned m = lane < sh.k ? key_of(lj) : 0;
        const float top = of_key(group_max<L>(m));
        float p = 0.0f;
        if (lj != -__builtin_inff()) {
            p = exp_near(lj - top);
            if (lj == top) p = 1.0f;  // infinite ones too
            if (!soft) {
                // s / sigmoid(top) * (1 + exp(-|top|)) in two ranges, neither of which overflows
                p = top > 0.0f ? sigmoid_near(lj) : p / (1.0f + exp_near(lj));
            }
            if (lj != lj) p = lj;
        }
        const float sum = group_sum<L>(p);
        w = p == 0.0f ? 0.0f : p / sum;
    } else {
        w = lj == -__builtin_inff() ? 0.0f : (soft ? exp_near(lj - largest) / total : sigmoid_near(lj));
    }
    if (soft && !(largest < __builtin_inff())) w = __builtin_nanf("");  // no softmax over NaN or an infinite score
    if (live && lane < sh.k) {
        expert[t * sh.k + lane] = e;
        weight[t * sh.k + lane] = e < 0 ? 0.0f : w * sh.scale;
    }
}

// ---------------------------------------------------------------------------
// The matrix by its columns: a stable counting sort of the slots
// ---------------------------------------------------------------------------
constexpr int kSortBlock = 1024;
constexpr int kSortWaves = kSortBlock / 64;
constexpr int kSortMaxChunks = 256;
constexpr int kSortMinChunk = 2048;  // slots of one workgroup

inline int sort_chunk(long long M)
{
    const long long c = (M + kSortMaxChunks - 1) / kSortMaxChunks;
    return (int)((c < kSortMinChunk ? kSortMinChunk : c) + kSortBlock - 1) / kSortBlock * kSortBlock;
}
// wavefronts that count by themselves: as many as fit 64 KB of counters
inline int sort_waves(int E) { return E < 512 ? kSortWaves : kSortWaves / 2; }

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
__global__ __launch_bounds__(kSortBlock) void columns_place_kernel(const int *__restrict__ expert, int M, int E, int chunk,
                                                                   int chunks, const int *__restrict__ counts, int waves,
                                                                   int *__restrict__ expert_ptr, int *__restrict__ slot,
                                                                   int *__restrict__ pos)
{
    extern __shared__ int place_lds[];  // waves x (E + 1)
    __shared__ int wave_sum[kSortWaves];
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
    // E1 <= 1025: thread x has expert x, thread 0 the last one too
    int total = 0, before = 0;
    const int e = threadIdx.x;
    if (e < E1) {
        if (counts) {
            for (int b = 0; b < chunks; ++b) {
                const int c = counts[(size_t)b * E1 + e];
                total += c;
                before += b < (int)blockIdx.x ? c : 0;
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
        int at = last;
        if (counts)
            for (int b = 0; b < (int)blockIdx.x; ++b) at += counts[(size_t)b * E1 + E];
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
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (in && rank == 0) hist[id] = at + __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (in) {
            slot[at + rank] = (int)s;
            pos[s] = id < E ? at + rank : -1;
        }
    }
}

int launch_columns(const int *expert, int M, int E, int *expert_ptr, int *slot, int *pos, void *workspace,
                   hipStream_t st)
{
    const int chunk = sort_chunk(M);
    const int chunks = M > 0 ? ceil_div(M, chunk) : 1;
    const int waves = sort_waves(E);
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
    const long long t = (long long)blockIdx.x * (kRouteBlock / 64) + (threadIdx.x >> 6);
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
        float p = 0.0f;
        if (lj != minus_inf) {
            p = lj == top ? 1.0f : exp_near(lj - top);
            if (!soft) p = top > 0.0f ? sigmoid_near(lj) : p / (1.0f + exp_near(lj));
            if (lj != lj) p = lj;
        }
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
            const int ej = __shfl(e, j, 64);
            const float pj = __shfl(part, j, 64);
            if (ej == i) d += pj;
        }
        if (i < sh.E) out[i] = (T)d;
    }
}

// ---------------------------------------------------------------------------
// Combination
// ---------------------------------------------------------------------------

// Y[t] = base[t] + sum_j w[t, j] Z[pos[t, j]]: one lane per 16 bytes of a row
// of Y.  Bound by the bytes of Z and Y; the k rows of a token are asked for
// together, four at a time.
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void combine_kernel(const T *__restrict__ Z, const int *__restrict__ pos,
                                                      const float *__restrict__ weight, const T *base, T *Y, int T_,
                                                      int k, int M, int N, int per_row)
{
    constexpr int V = 16 / sizeof(T);
    const long long item = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long t = item / per_row;
    if (t >= T_) return;
    const int col = (int)(item - t * per_row) * V;
    const int valid = N - col;
    float acc[V];
    if (base) load_vec<T, V, ALIGNED>(acc, base + t * N + col, valid);
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
            if (p[j] >= 0) load_vec<T, V, ALIGNED>(z[j], Z + (long long)p[j] * N + col, valid);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (p[j] >= 0) {
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = __builtin_fmaf(w[j], z[j][i], acc[i]);
            }
    }
    store_vec<T, V, ALIGNED>(Y + t * N + col, acc, valid);
}

// One wavefront per place: reads the row of Z and the token's row of dY, writes
// the row of dZ and the product of the two rows.  Places are in order, so Z and
// dZ stream; the k reads of a row of dY meet in the caches.
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void combine_backward_kernel(const T *__restrict__ dY, const T *__restrict__ Z,
                                                               const float *__restrict__ weight,
                                                               const int *__restrict__ expert_ptr, int E,
                                                               const int *__restrict__ slot, T *__restrict__ dZ,
                                                               float *__restrict__ dweight, int k, int M, int N)
{
    constexpr int V = 16 / sizeof(T);
    const int lane = threadIdx.x & 63;
    const int p = (int)min((long long)blockIdx.x * 4 + (threadIdx.x >> 6), (long long)M);
    if (p >= M) return;
    const int s = slot[p];
    const bool known = (unsigned)s < (unsigned)M;
    const bool routed = known && p < expert_ptr[E];
    const float w = routed ? (weight ? weight[s] : 1.0f) : 0.0f;
    const T *y_row = dY + (long long)(routed ? s / k : 0) * N;
    const T *z_row = Z + (long long)p * N;
    T *out = dZ + (long long)p * N;
    float dot = 0.0f;
    for (int col = lane * V; col < N; col += 64 * V) {
        float y[V], z[V];
        if (routed) {
            load_vec<T, V, ALIGNED>(y, y_row + col, N - col);
            if (dweight) {
                load_vec<T, V, ALIGNED>(z, z_row + col, N - col);
#pragma unroll
                for (int i = 0; i < V; ++i) dot = __builtin_fmaf(y[i], z[i], dot);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] *= w;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = 0.0f;
        }
        store_vec<T, V, ALIGNED>(out + col, y, N - col);
    }
    if (dweight && known) {
        dot = group_sum<64>(dot);
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
    return RouteShape{T, E, o.k, o.score, groups, E / groups, o.top_groups, o.group_score, o.renormalise, o.scale};
}

template <typename T>
int launch_route(const T *scores, const float *bias, const RouteShape &sh, int *expert, float *weight, hipStream_t st)
{
    const size_t per_token = (size_t)(sh.groups > 1 ? sh.E + sh.groups : 0) * sizeof(unsigned long long);
#define MPS_LAUNCH_ROUTE(IPL, L)                                                                                   \
    hipLaunchKernelGGL((route_kernel<T, IPL, L>), dim3(ceil_div(sh.T, kRouteBlock / L)), dim3(kRouteBlock),        \
                       per_token * (kRouteBlock / L), st, scores, bias, sh, expert, weight)
    if (sh.E <= 64) MPS_LAUNCH_ROUTE(1, 64);
    else if (sh.E <= 128) MPS_LAUNCH_ROUTE(2, 64);
    else if (sh.E <= 256) MPS_LAUNCH_ROUTE(4, 64);
    else if (sh.E <= 512) MPS_LAUNCH_ROUTE(8, 64);
    else MPS_LAUNCH_ROUTE(16, 64);
#undef MPS_LAUNCH_ROUTE
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

template <typename T>
int launch_combine(const void *Z, const int *pos, const float *weight, const void *base, void *Y, int T_, int k, int M,
                   int N, hipStream_t st)
{
    const int per_row = ceil_div(N, 16 / (int)sizeof(T));
    const long long blocks = ((long long)T_ * per_row + 255) / 256;
    if (blocks > INT_MAX) return MPS_ERR_UNSUPPORTED;
    const bool fast = rows_of_16(Z, N, sizeof(T)) && rows_of_16(Y, N, sizeof(T)) && rows_of_16(base, N, sizeof(T));
#define MPS_LAUNCH_COMBINE(ALIGNED)                                                                               \
    hipLaunchKernelGGL((combine_kernel<T, ALIGNED>), dim3((unsigned)blocks), dim3(256), 0, st,                    \
                       static_cast<const T *>(Z), pos, weight, static_cast<const T *>(base), static_cast<T *>(Y), \
                       T_, k, M, N, per_row)
    if (fast) MPS_LAUNCH_COMBINE(true);
    else MPS_LAUNCH_COMBINE(false);
#undef MPS_LAUNCH_COMBINE
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

template <typename T>
int launch_combine_backward(const void *dY, const void *Z, const float *weight, const int *expert_ptr, int E,
                            const int *slot, void *dZ, float *dweight, int k, int M, int N, hipStream_t st)
{
    const bool fast = rows_of_16(dY, N, sizeof(T)) && rows_of_16(Z, N, sizeof(T)) && rows_of_16(dZ, N, sizeof(T));
#define MPS_LAUNCH_COMBINE(ALIGNED)                                                                                \
    hipLaunchKernelGGL((combine_backward_kernel<T, ALIGNED>), dim3(ceil_div(M, 4)), dim3(256), 0, st,              \
                       static_cast<const T *>(dY), static_cast<const T *>(Z), weight, expert_ptr, E, slot,         \
                       static_cast<T *>(dZ), dweight, k, M, N)
    if (fast) MPS_LAUNCH_COMBINE(true);
    else MPS_LAUNCH_COMBINE(false);
#undef MPS_LAUNCH_COMBINE
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
    if (T > 0) {
        const RouteShape sh = make_shape(*options, T, E);
        int r;
        if (dtype == MPS_F32) r = launch_route(static_cast<const float *>(d_scores), d_bias, sh, d_expert, d_weight, st);
        else if (dtype == MPS_F16) r = launch_route(static_cast<const half_t *>(d_scores), d_bias, sh, d_expert, d_weight, st);
        else r = launch_route(static_cast<const bf16_t *>(d_scores), d_bias, sh, d_expert, d_weight, st);
        if (r != MPS_OK) return r;
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
    hipLaunchKernelGGL((route_backward_kernel<TYPE>), dim3(ceil_div(T, kRouteBlock / 64)), dim3(kRouteBlock), 0, st, \
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
