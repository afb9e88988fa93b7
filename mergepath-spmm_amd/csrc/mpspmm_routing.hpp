// Shared by the sparse-routing translation units (mpspmm_route.hip: routing
// matrices, their gradient, combination; mpspmm_experts.hip: the experts'
// products; mpspmm_adapters.hip: low-rank adapters).  Everything lives in an
// anonymous namespace.
#ifndef MPSPMM_ROUTING_HPP
#define MPSPMM_ROUTING_HPP

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <cstring>

#include "mpspmm.h"

#define MPS_HIP_TRY(expr)                                       \
    do {                                                        \
        hipError_t e_ = (expr);                                 \
        if (e_ != hipSuccess) return MPS_ERR_HIP + (int)e_;     \
    } while (0)

namespace {

using half_t = _Float16;
using bf16_t = __bf16;

inline int dtype_bytes(int dtype) { return dtype == MPS_F32 ? 4 : (dtype == MPS_F16 || dtype == MPS_BF16) ? 2 : 0; }

inline bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

inline int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// A launch holds fewer than 2^32 threads in a dimension, which a wavefront for
// every one of 2^26 tokens reaches; of more only the rest is run, without an
// error.  More workgroups than kGridRow go into rows of a second dimension.
// Numbers from `blocks` on occur then; a kernel has nothing to do for them.
constexpr int kGridRow = 1 << 22;
inline dim3 grid_of(long long blocks)
{
    return blocks <= kGridRow ? dim3((unsigned)blocks) : dim3(kGridRow, (unsigned)ceil_div(blocks, kGridRow));
}
__device__ __forceinline__ long long block_number() { return (long long)blockIdx.y * kGridRow + blockIdx.x; }

// Whether a x b workgroups fit one dimension; a b may be beyond 64 bits.
inline bool fits_launch(long long a, long long b, int threads)
{
    const long long most = 0xFFFFFFFFll / threads;
    return a <= most && b <= most && a * b <= most;
}

// A matrix whose rows are loaded 16 bytes at a time: aligned base, rows of whole 16 bytes.
inline bool rows_of_16(const void *p, long long row_elems, int elem_bytes)
{
    return aligned_to(p, 16) && row_elems * elem_bytes % 16 == 0;
}

// V elements of T at an address that is only aligned to the element, of which
// `valid` exist.  Global memory takes one wide access at any such address, so that
// rows of whole 16 bytes have no variant of their own: it was the same instructions.
template <typename T, int V>
__device__ __forceinline__ void load_vec(float (&out)[V], const T *p, int valid)
{
    if (valid >= V) {
        T raw[V];
        __builtin_memcpy(raw, __builtin_assume_aligned(p, sizeof(T)), V * sizeof(T));
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = (float)raw[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) out[i] = i < valid ? (float)p[i] : 0.0f;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[V], int valid)
{
    if (valid >= V) {
        T raw[V];
#pragma unroll
        for (int i = 0; i < V; ++i) raw[i] = (T)v[i];
        __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), raw, V * sizeof(T));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < valid) p[i] = (T)v[i];
    }
}

typedef float float4v __attribute__((ext_vector_type(4)));
typedef half_t half8v __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8v __attribute__((ext_vector_type(8)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

// acc += p q^T for 16 rows p and q of one matrix step, 16 bytes of the summed
// index in every lane: lane l holds row l % 16, chunk l / 16.  The result: lane l
// holds q = l % 16 and four neighbouring p from (l / 16) * 4 on.
template <typename T>
__device__ __forceinline__ float4v mma(uint4v p, uint4v q, float4v acc)
{
    if constexpr (sizeof(T) == 4) {
        // instruction j sums element j of every chunk
        const float4v a = __builtin_bit_cast(float4v, p), b = __builtin_bit_cast(float4v, q);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
        return acc;
    } else if constexpr (__is_same(T, half_t)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, p), __builtin_bit_cast(half8v, q), acc,
                                                      0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8v, p), __builtin_bit_cast(bf16x8v, q),
                                                       acc, 0, 0, 0);
    }
}

// 16 bytes from p, of which `valid` elements exist; zeros for the others.
template <typename T>
__device__ __forceinline__ uint4v load_chunk(const T *p, int valid)
{
    constexpr int V = 16 / sizeof(T);
    uint4v v = {0, 0, 0, 0};
    if (valid >= V) {
        __builtin_memcpy(&v, __builtin_assume_aligned(p, sizeof(T)), 16);
    } else if (valid > 0) {
        T part[V];
#pragma unroll
        for (int i = 0; i < V; ++i) part[i] = i < valid ? p[i] : (T)0.0f;
        __builtin_memcpy(&v, part, 16);
    }
    return v;
}

// ---------------------------------------------------------------------------
// Segments.  ptr[0 .. E] cuts the places 0 .. M - 1 into the experts' runs.
// Values are clamped so that no caller's table reaches outside the arrays.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int clamp_place(int v, int M) { return min(max(v, 0), M); }

// Row tiles of the segments, BM rows each.  Expert e's tiles get the numbers
// ptr[e] / BM + e + i, i = 0 .. ceil(rows / BM) - 1.  Because
//   floor(ptr[e] / BM) + ceil(rows / BM) <= floor(ptr[e + 1] / BM) + 1
// no two experts share a number, so that a tile finds its expert as the last e
// with ptr[e] / BM + e <= number, without a prefix sum over the experts: the
// path that merges the ends of the experts with the tiles' rows.  Numbers
// below M / BM + E; those in a gap belong to nobody (rows = 0).
// One wavefront looks the expert up, 64 candidates at a time.
struct RowTile {
    int expert, first, rows;  // rows <= BM; 0 = nothing to do
};
template <int BM>
__device__ __forceinline__ RowTile find_row_tile(const int *__restrict__ ptr, int E, int M, int number)
{
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = E - 1;  // the expert lies in [lo, hi]
    while (hi > lo) {
        const int step = (hi - lo + 64) >> 6;
        const int e = lo + (lane + 1) * step;
        const bool below = e <= hi && clamp_place(ptr[e], M) / BM + e <= number;
        const int n = __popcll(__ballot(below));
        lo += n * step;
        hi = min(hi, lo + step - 1);
    }
    const int a = clamp_place(ptr[lo], M), b = clamp_place(ptr[lo + 1], M);
    RowTile t;
    t.expert = lo;
    const long long first = a + ((long long)number - a / BM - lo) * BM;
    t.rows = first < a || first >= b ? 0 : min(b - (int)first, BM);
    t.first = t.rows ? (int)first : a;
    return t;
}
// Workgroups are dealt to the 8 dies in turn, each with an L2 of its own.  Runs
// of kRun tiles go to one die, so that tiles that share an expert's weights and
// rows meet in one L2; the runs are dealt in turn, so that a long segment is
// shared by all dies.  Whole eighths of the tiles for a die: gradient of the
// weights of 32 uneven experts 599 us, 458 without runs, 285 with runs of 64;
// with 256 x 256 tiles runs of 8, 16, 32, 64 and 128: 210, 209, 237, 202 - 245, 268.
__device__ __forceinline__ int xcd_tile(int block, int blocks)
{
    constexpr int kRun = 16;
    if (block >= blocks / (8 * kRun) * (8 * kRun)) return block;
    const int xcd = block & 7, nth = block >> 3;
    return ((nth / kRun) * 8 + xcd) * kRun + nth % kRun;
}
inline long long num_row_tiles(int M, int E, int BM) { return (long long)M / BM + E; }

// ---------------------------------------------------------------------------
// Reductions over groups of L neighbouring lanes; every lane gets the result.
// ---------------------------------------------------------------------------
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned v)
{
    return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
// op(own value, that of the lane STEP further round), within 8 and 16 lanes by
// moving data between lanes; across 16 and 32 by exchanging rows of lanes
// between two copies, which leaves the two values side by side.  The lanes
// below STEP agree already, so the mirrored halves do for 4 and 8.
template <int STEP, typename V, typename F>
__device__ __forceinline__ V fold(V v, F op)
{
    static_assert(sizeof(V) == 4 || sizeof(V) == 8, "one or two registers");
    constexpr int WORDS = sizeof(V) / 4;
    unsigned own[WORDS], other[WORDS];
    __builtin_memcpy(own, &v, sizeof(V));
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
        if constexpr (STEP == 1) other[i] = dpp<0xB1>(own[i]);        // quad_perm 1,0,3,2
        else if constexpr (STEP == 2) other[i] = dpp<0x4E>(own[i]);   // quad_perm 2,3,0,1
        else if constexpr (STEP == 4) other[i] = dpp<0x141>(own[i]);  // mirrored within 8 lanes
        else if constexpr (STEP == 8) other[i] = dpp<0x140>(own[i]);  // mirrored within 16 lanes
        else {
            const auto both = STEP == 16 ? __builtin_amdgcn_permlane16_swap(own[i], own[i], false, false)
                                         : __builtin_amdgcn_permlane32_swap(own[i], own[i], false, false);
            own[i] = both[0];
            other[i] = both[1];
        }
    }
    V a, b;
    __builtin_memcpy(&a, own, sizeof(V));
    __builtin_memcpy(&b, other, sizeof(V));
    return op(a, b);
}
template <int L, typename V, typename F>
__device__ __forceinline__ V fold_group(V v, F op)
{
    if constexpr (L > 1) v = fold<1>(v, op);
    if constexpr (L > 2) v = fold<2>(v, op);
    if constexpr (L > 4) v = fold<4>(v, op);
    if constexpr (L > 8) v = fold<8>(v, op);
    if constexpr (L > 16) v = fold<16>(v, op);
    if constexpr (L > 32) v = fold<32>(v, op);
    return v;
}
template <int L, typename V>
__device__ __forceinline__ V group_max(V v)
{
    return fold_group<L>(v, [](V a, V b) { return max(a, b); });
}
template <int L, typename V>
__device__ __forceinline__ V group_sum(V v)
{
    return fold_group<L>(v, [](V a, V b) { return a + b; });
}
__device__ __forceinline__ float bits_float(unsigned u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ unsigned float_bits(float f) { return __builtin_bit_cast(unsigned, f); }

}  // namespace

#endif
