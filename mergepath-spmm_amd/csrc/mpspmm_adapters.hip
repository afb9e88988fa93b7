// Low-rank adapters of many requests beside a shared projection:
//   Y[t] = base[t] + scale[a] * (X[t] * A[a]^T) * B[a]^T
// for the tokens t of adapter a, which the columns of a routing matrix list.
// Two launches: the first makes V = X A^T (places x rank, fp32, in the
// workspace; the sum over K is cut into `splits` parts so that a few tokens
// fill the GPU), the second adds up the parts, multiplies with B and adds the
// base.  Both read each operand from memory into the matrix instructions'
// registers, without LDS between: the weights of an adapter are used by one
// tile of tokens, or found in the caches by the next.
#include "mpspmm_routing.hpp"

namespace {

typedef float float4v __attribute__((ext_vector_type(4)));
typedef half_t half8v __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8v __attribute__((ext_vector_type(8)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kRows = 16;  // tokens of a tile

template <typename T>
__device__ __forceinline__ float4v mma(uint4v p, uint4v q, float4v acc)
{
    if constexpr (sizeof(T) == 4) {
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
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4v load_chunk(const T *p, int valid)
{
    constexpr int V = 16 / sizeof(T);
    uint4v v = {0, 0, 0, 0};
    if (valid >= V) {
        __builtin_memcpy(&v, __builtin_assume_aligned(p, ALIGNED ? 16 : sizeof(T)), 16);
    } else if (valid > 0) {
        T part[V];
#pragma unroll
        for (int i = 0; i < V; ++i) part[i] = i < valid ? p[i] : (T)0.0f;
        __builtin_memcpy(&v, part, 16);
    }
    return v;
}

struct AdaptersShape {
    int T, E, R, K, N;
    int padded;       // the rank that the kernels are made for, 16, 32, 64, 128 or 256: the pitch of V
    int splits, per_split;  // parts of the sum over K, and their length
};

// V[split][place][r] = sum over the split's part of K.  One workgroup per tile
// of 16 tokens and part; its four wavefronts take the 64-byte steps of the part
// in turn and add up through LDS.
template <typename T, int RT, bool ALIGNED>
__global__ __launch_bounds__(64 * kWaves) void adapters_shrink_kernel(const T *__restrict__ X, const T *__restrict__ A,
                                                                      const int *__restrict__ ptr,
                                                                      const int *__restrict__ row_of,
                                                                      float *__restrict__ V, AdaptersShape sh)
{
    constexpr int C = 16 / sizeof(T), STEP = 4 * C;
    __shared__ float4v join[kWaves - 1][RT][64];
    const RowTile t = find_row_tile<kRows>(ptr, sh.E, sh.T, blockIdx.x);
    if (t.rows == 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = lane & 15, g = lane >> 4;
    int token = i < t.rows ? row_of[t.first + i] : -1;
    if ((unsigned)token >= (unsigned)sh.T) token = -1;
    const T *x = X + (size_t)(token < 0 ? 0 : token) * sh.K;
    const T *a = A + (size_t)t.expert * sh.R * sh.K;
    const int k0 = blockIdx.y * sh.per_split, k1 = min(k0 + sh.per_split, sh.K);
    float4v acc[RT] = {};
    for (int k = k0 + wave * STEP + g * C; k - g * C < k1; k += kWaves * STEP) {
        const uint4v q = load_chunk<T, ALIGNED>(x + k, token < 0 ? 0 : k1 - k);
#pragma unroll
        for (int n = 0; n < RT; ++n) {
            const int r = n * 16 + i;
            const uint4v p = load_chunk<T, ALIGNED>(a + (size_t)(r < sh.R ? r : 0) * sh.K + k, r < sh.R ? k1 - k : 0);
            acc[n] = mma<T>(p, q, acc[n]);
        }
    }
    if (wave > 0) {
#pragma unroll
        for (int n = 0; n < RT; ++n) join[wave - 1][n][lane] = acc[n];
    }
    __syncthreads();
    if (wave == 0 && i < t.rows) {
        float *out = V + ((size_t)blockIdx.y * sh.T + t.first + i) * sh.padded + g * 4;
#pragma unroll
        for (int n = 0; n < RT; ++n) {
            float4v sum = acc[n];
#pragma unroll
            for (int w = 0; w < kWaves - 1; ++w) sum += join[w][n][lane];
            *reinterpret_cast<float4v *>(out + n * 16) = sum;
        }
    }
}

// One workgroup per tile of 16 tokens and 256 columns, a wavefront 64 columns.
// V is made in fp32; for the product with B it is split into its rounding to T
// and the rounding of what that leaves, two instructions instead of one, so
// that it is not rounded to 8 or 11 bits on the way.  fp16 has no room for
// values from 65520 on: where a tile holds one, all of its V are taken down by
// 2^16 and the sums up again.  RANK: the largest rank, in units of 32.
template <typename T, int RANK, bool ALIGNED>
__global__ __launch_bounds__(64 * kWaves) void adapters_expand_kernel(const float *__restrict__ V,
                                                                      const T *__restrict__ B,
                                                                      const float *__restrict__ scale, const T *base,
                                                                      T *Y, const int *__restrict__ ptr,
                                                                      const int *__restrict__ row_of, AdaptersShape sh)
{
    constexpr int C = 16 / sizeof(T), STEP = 4 * C;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = lane & 15, g = lane >> 4;
    // The tokens without an adapter are one more segment, of which only the base is left.
    const int routed = clamp_place(ptr[sh.E], sh.T);
    const int tail_tiles = (sh.T - routed + kRows - 1) / kRows;
    RowTile t;
    if ((int)blockIdx.y < tail_tiles) {
        t.expert = -1;
        t.first = routed + blockIdx.y * kRows;
        t.rows = min(sh.T - t.first, kRows);
    } else {
        t = find_row_tile<kRows>(ptr, sh.E, sh.T, blockIdx.y - tail_tiles);
        if (t.rows == 0) return;
    }
    const int token = i < t.rows ? row_of[t.first + i] : -1;
    const bool live = (unsigned)token < (unsigned)sh.T;
    const int n0 = (blockIdx.x * kWaves + wave) * 64;
    if (n0 >= sh.N) return;
    float4v acc[4] = {};
    if (t.expert >= 0) {
        const float s = scale ? scale[t.expert] : 1.0f;
        const T *b = B + (size_t)t.expert * sh.N * sh.R;
        constexpr int STEPS = RANK * 32 / STEP;
        float v[STEPS][C];
        bool far = false;
#pragma unroll
        for (int m = 0; m < STEPS; ++m) {
            const int r = m * STEP + g * C;
#pragma unroll
            for (int c = 0; c < C; ++c) v[m][c] = 0.0f;
            if (live && r < sh.padded) {
                for (int part = 0; part < sh.splits; ++part) {
                    const float *from = V + ((size_t)part * sh.T + t.first + i) * sh.padded + r;
#pragma unroll
                    for (int c = 0; c < C; c += 4) {
                        const float4v f = *reinterpret_cast<const float4v *>(from + c);
#pragma unroll
                        for (int d = 0; d < 4; ++d) v[m][c + d] += f[d];
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < C; ++c) {
                v[m][c] = r + c < sh.R ? v[m][c] * s : 0.0f;  // infinite rows have NaN behind the rank
                far |= __builtin_fabsf(v[m][c]) > 65000.0f;
            }
        }
        const bool down = __is_same(T, half_t) && __any(far);
#pragma unroll
        for (int m = 0; m < STEPS; ++m) {
            const int r = m * STEP + g * C;
            if (m * STEP >= sh.R) break;
            uint4v high, low;
            T high_of[C], low_of[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const float x = down ? v[m][c] * 0x1p-16f : v[m][c];
                high_of[c] = (T)x;
                const float rest = x - (float)high_of[c];
                low_of[c] = (T)(__builtin_fabsf(rest) < __builtin_inff() ? rest : 0.0f);  // infinities stand in `high`
            }
            __builtin_memcpy(&high, high_of, 16);
            __builtin_memcpy(&low, low_of, 16);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int col = n0 + n * 16 + i;
                const uint4v p = load_chunk<T, ALIGNED>(b + (size_t)(col < sh.N ? col : 0) * sh.R + r,
                                                        col < sh.N ? sh.R - r : 0);
                acc[n] = mma<T>(p, high, acc[n]);
                if constexpr (sizeof(T) == 2) acc[n] = mma<T>(p, low, acc[n]);
            }
        }
        if (down) {
#pragma unroll
            for (int n = 0; n < 4; ++n) acc[n] *= 65536.0f;
        }
    }
    if (!live) return;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int col = n0 + n * 16 + g * 4;
        if (col >= sh.N) continue;
        float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (base) load_vec<T, 4, ALIGNED>(y, base + (size_t)token * sh.N + col, sh.N - col);
#pragma unroll
        for (int d = 0; d < 4; ++d) y[d] += acc[n][d];
        store_vec<T, 4, ALIGNED>(Y + (size_t)token * sh.N + col, y, sh.N - col);
    }
}

AdaptersShape make_shape(int T, int E, int R, int K, int N)
{
    int padded = 16;
    while (padded < R) padded *= 2;
    AdaptersShape sh{T, E, R, K, N, padded, 1, K};
    // Parts of the sum over K: about 1024 workgroups, each with at least 256 of K.
    const long long tiles = num_row_tiles(T, E < T ? E : T, kRows);
    long long splits = 1024 / (tiles > 0 ? tiles : 1);
    if (splits > K / 256) splits = K / 256;
    if (splits > 16) splits = 16;
    if (splits < 1) splits = 1;
    sh.per_split = (ceil_div(K, splits) + 63) / 64 * 64;
    sh.splits = ceil_div(K, sh.per_split);
    return sh;
}

template <typename T>
int launch_adapters(const void *X, const void *A, const void *B, const float *scale, const void *base, void *Y,
                    const int *ptr, const int *row_of, const AdaptersShape &sh, float *V, hipStream_t st)
{
    const long long tiles = num_row_tiles(sh.T, sh.E, kRows);
    const dim3 shrink((unsigned)tiles, sh.splits);
    const bool fast = rows_of_16(X, sh.K, sizeof(T)) && rows_of_16(A, sh.K, sizeof(T));
#define MPS_LAUNCH_SHRINK(RT)                                                                                       \
    if (fast)                                                                                                       \
        hipLaunchKernelGGL((adapters_shrink_kernel<T, RT, true>), shrink, dim3(64 * kWaves), 0, st,                 \
                           static_cast<const T *>(X), static_cast<const T *>(A), ptr, row_of, V, sh);               \
    else                                                                                                            \
        hipLaunchKernelGGL((adapters_shrink_kernel<T, RT, false>), shrink, dim3(64 * kWaves), 0, st,                \
                           static_cast<const T *>(X), static_cast<const T *>(A), ptr, row_of, V, sh)
    if (sh.padded <= 16) { MPS_LAUNCH_SHRINK(1); }
    else if (sh.padded <= 32) { MPS_LAUNCH_SHRINK(2); }
    else if (sh.padded <= 64) { MPS_LAUNCH_SHRINK(4); }
    else if (sh.padded <= 128) { MPS_LAUNCH_SHRINK(8); }
    else { MPS_LAUNCH_SHRINK(16); }
#undef MPS_LAUNCH_SHRINK
    MPS_HIP_TRY(hipGetLastError());
    const dim3 expand(ceil_div(sh.N, 64 * kWaves), (unsigned)tiles + 1);
    const bool fast2 = rows_of_16(B, sh.R, sizeof(T)) && rows_of_16(base, sh.N, sizeof(T)) && rows_of_16(Y, sh.N, sizeof(T));
#define MPS_LAUNCH_EXPAND(RANK, ALIGNED)                                                                             \
    hipLaunchKernelGGL((adapters_expand_kernel<T, RANK, ALIGNED>), expand, dim3(64 * kWaves), 0, st, V,                    \
                       static_cast<const T *>(B), scale, static_cast<const T *>(base), static_cast<T *>(Y), ptr, row_of, sh)
    if (sh.R <= 32) { if (fast2) MPS_LAUNCH_EXPAND(1, true); else MPS_LAUNCH_EXPAND(1, false); }
    else if (sh.R <= 64) { if (fast2) MPS_LAUNCH_EXPAND(2, true); else MPS_LAUNCH_EXPAND(2, false); }
    else { if (fast2) MPS_LAUNCH_EXPAND(8, true); else MPS_LAUNCH_EXPAND(8, false); }
#undef MPS_LAUNCH_EXPAND
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

int check_adapters(int T, int E, int R, int K)
{
    if (T < 0 || E < 1 || R < 1 || K < 1) return MPS_ERR_INVALID_ARG;
    if (R > MPS_ADAPTERS_MAX_RANK || E > MPS_ROUTE_MAX_EXPERTS || T > 65535 * 8 || K > INT_MAX / 4)
        return MPS_ERR_UNSUPPORTED;
    return MPS_OK;
}

}  // namespace

extern "C" {

int mps_adapters_workspace_bytes(int T, int E, int R, int K, size_t *bytes_out)
{
    if (!bytes_out) return MPS_ERR_INVALID_ARG;
    const int rc = check_adapters(T, E, R, K);
    if (rc != MPS_OK) return rc;
    const AdaptersShape sh = make_shape(T, E, R, K, 1);
    *bytes_out = (size_t)sh.splits * T * sh.padded * sizeof(float);
    return MPS_OK;
}

int mps_adapters_mm(const void *d_X, const void *d_A, const void *d_B, const float *d_scale, const void *d_base,
                    void *d_Y, int dtype, const int *d_adapter_ptr, const int *d_row, int T, int E, int R, int K, int N,
                    void *d_workspace, size_t workspace_bytes, void *stream)
{
    size_t need = 0;
    const int rc = mps_adapters_workspace_bytes(T, E, R, K, &need);
    if (rc != MPS_OK) return rc;
    const int eb = dtype_bytes(dtype);
    if (!eb || N < 1) return MPS_ERR_INVALID_ARG;
    if (N > INT_MAX / 4) return MPS_ERR_UNSUPPORTED;
    if (T == 0) return MPS_OK;
    if (!d_X || !d_A || !d_B || !d_Y || !d_adapter_ptr || !d_row) return MPS_ERR_INVALID_ARG;
    if (!aligned_to(d_X, eb) || !aligned_to(d_A, eb) || !aligned_to(d_B, eb) || !aligned_to(d_scale, 4) ||
        !aligned_to(d_base, eb) || !aligned_to(d_Y, eb) || !aligned_to(d_adapter_ptr, 4) || !aligned_to(d_row, 4) ||
        !aligned_to(d_workspace, 16))
        return MPS_ERR_ALIGNMENT;
    if (!d_workspace || workspace_bytes < need) return MPS_ERR_WORKSPACE;
    const AdaptersShape sh = make_shape(T, E, R, K, N);
    hipStream_t st = static_cast<hipStream_t>(stream);
    float *V = static_cast<float *>(d_workspace);
    if (dtype == MPS_F32) return launch_adapters<float>(d_X, d_A, d_B, d_scale, d_base, d_Y, d_adapter_ptr, d_row, sh, V, st);
    if (dtype == MPS_F16) return launch_adapters<half_t>(d_X, d_A, d_B, d_scale, d_base, d_Y, d_adapter_ptr, d_row, sh, V, st);
    return launch_adapters<bf16_t>(d_X, d_A, d_B, d_scale, d_base, d_Y, d_adapter_ptr, d_row, sh, V, st);
}

}  // extern "C"
