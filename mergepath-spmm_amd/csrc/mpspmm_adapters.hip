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

constexpr int kWaves = 4;

struct AdaptersShape {
    int T, E, R, K, N;
    int padded;             // the rank that the kernels are made for, 16, 32, 64, 128 or 256: the pitch of V
    int splits, per_split;  // parts of the sum over K, and their length
    bool tall;              // long segments: tiles of several times 16 tokens
};

// V[split][place][r] = sum over the split's part of K.  One workgroup per tile
// of 16 MT tokens and part; its four wavefronts take 128 bytes of a row in turn
// and add up through LDS.  A step of 64 bytes loads MT + RT chunks for MT * RT
// matrix instructions.
template <typename T, int RT, int MT>
__global__ __launch_bounds__(64 * kWaves) void adapters_shrink_kernel(const T *__restrict__ X, const T *__restrict__ A,
                                                                      const int *__restrict__ ptr,
                                                                      const int *__restrict__ row_of,
                                                                      float *__restrict__ V, AdaptersShape sh)
{
    constexpr int C = 16 / sizeof(T), STEP = 4 * C;
    __shared__ float4v join[kWaves][RT][64];
    const RowTile t = find_row_tile<16 * MT>(ptr, sh.E, sh.T, blockIdx.x);
    if (t.rows == 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = lane & 15, g = lane >> 4;
    const T *x[MT];
    bool live[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int token = 16 * m + i < t.rows ? row_of[t.first + 16 * m + i] : -1;
        live[m] = (unsigned)token < (unsigned)sh.T;
        x[m] = X + (size_t)(live[m] ? token : 0) * sh.K;
    }
    const T *a[RT];
#pragma unroll
    for (int n = 0; n < RT; ++n) {
        const int r = n * 16 + i;
        a[n] = A + ((size_t)t.expert * sh.R + (r < sh.R ? r : 0)) * sh.K;
    }
    const int k0 = blockIdx.y * sh.per_split, k1 = min(k0 + sh.per_split, sh.K);
    float4v acc[MT][RT] = {};
    for (int base = k0 + wave * 2 * STEP; base < k1; base += kWaves * 2 * STEP) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = base + half * STEP + g * C;
            uint4v q[MT], p[RT];
#pragma unroll
            for (int m = 0; m < MT; ++m) q[m] = load_chunk<T>(x[m] + k, live[m] ? k1 - k : 0);
#pragma unroll
            for (int n = 0; n < RT; ++n) p[n] = load_chunk<T>(a[n] + k, n * 16 + i < sh.R ? k1 - k : 0);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < RT; ++n) acc[m][n] = mma<T>(p[n], q[m], acc[m][n]);
        }
    }
    // The wavefronts' sums meet 16 tokens at a time; each wavefront adds a share of the ranks up.
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (m > 0) __syncthreads();
#pragma unroll
        for (int n = 0; n < RT; ++n) join[wave][n][lane] = acc[m][n];
        __syncthreads();
        if (16 * m + i < t.rows) {
            float *out = V + ((size_t)blockIdx.y * sh.T + t.first + 16 * m + i) * sh.padded + g * 4;
            for (int n = wave; n < RT; n += kWaves) {
                float4v sum = join[0][n][lane];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) sum += join[w][n][lane];
                *reinterpret_cast<float4v *>(out + n * 16) = sum;
            }
        }
    }
}

// One workgroup per tile of 16 MT tokens and `columns` columns; a wavefront takes
// 64 columns at a time, with the tokens' V in its registers throughout.  V is
// made in fp32; for the product with B it is split into its rounding to T and
// the rounding of what that leaves, two instructions instead of one, so that
// it is not rounded to 8 or 11 bits on the way but to 16 (bf16) or 22 (fp16).
// fp16 has neither room for values from 65520 on nor bits for those below 2^-14:
// a token's V are multiplied by the power of two that takes the largest of them to
// 2^14 or more, below 2^15, and its sums divided by it, so that each is kept to
// 2^-22 of itself or 2^-39 of the largest.  RANK: the largest rank, in units of 32.
// Row g * 4 + d of the b-th matrix instruction is the column that leaves a lane
// with 16 bytes of neighbouring columns, and the four lanes of a token with 64.
template <typename T, int RANK, int MT>
__global__ __launch_bounds__(64 * kWaves) void adapters_expand_kernel(const float *__restrict__ V,
                                                                      const T *__restrict__ B,
                                                                      const float *__restrict__ scale, const T *base,
                                                                      T *Y, const int *__restrict__ ptr,
                                                                      const int *__restrict__ row_of, int columns,
                                                                      AdaptersShape sh)
{
    constexpr int C = 16 / sizeof(T), STEP = 4 * C, STEPS = RANK * 32 / STEP, ROWS = 16 * MT;
    constexpr int PER = C / 4;  // matrix instructions that fill 16 bytes
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = lane & 15, g = lane >> 4;
    // The tokens without an adapter are one more segment, of which only the base is left.
    const int routed = clamp_place(ptr[sh.E], sh.T);
    const int tail_tiles = (sh.T - routed + ROWS - 1) / ROWS;
    RowTile t;
    if ((int)blockIdx.y < tail_tiles) {
        t.expert = -1;
        t.first = routed + blockIdx.y * ROWS;
        t.rows = min(sh.T - t.first, ROWS);
    } else {
        t = find_row_tile<ROWS>(ptr, sh.E, sh.T, blockIdx.y - tail_tiles);
        if (t.rows == 0) return;
    }
    int token[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        token[m] = 16 * m + i < t.rows ? row_of[t.first + 16 * m + i] : -1;
        if ((unsigned)token[m] >= (unsigned)sh.T) token[m] = -1;
    }
    uint4v high[MT][STEPS], low[MT][STEPS];
    float back[MT] = {};  // 1 / the factor on a token's V
    if (t.expert >= 0) {
        const float s = scale ? scale[t.expert] : 1.0f;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float v[STEPS][C];
            float largest = 0.0f;  // finite one
#pragma unroll
            for (int step = 0; step < STEPS; ++step) {
                const int r = step * STEP + g * C;
#pragma unroll
                for (int c = 0; c < C; ++c) v[step][c] = 0.0f;
                if (token[m] >= 0 && r < sh.padded) {
#pragma unroll 4
                    for (int part = 0; part < sh.splits; ++part) {
                        const float *from = V + ((size_t)part * sh.T + t.first + 16 * m + i) * sh.padded + r;
#pragma unroll
                        for (int c = 0; c < C; c += 4) {
                            const float4v f = *reinterpret_cast<const float4v *>(from + c);
#pragma unroll
                            for (int d = 0; d < 4; ++d) v[step][c + d] += f[d];
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    v[step][c] = r + c < sh.R ? v[step][c] * s : 0.0f;  // infinite rows have NaN behind the rank
                    const float size = __builtin_fabsf(v[step][c]);
                    if (size < __builtin_inff()) largest = max(largest, size);
                }
            }
            float factor = 1.0f;
            back[m] = 1.0f;
            if constexpr (__is_same(T, half_t)) {
                // a token's values lie in the four lanes i, i + 16, i + 32, i + 48; its sums come back to the same lanes
                const auto larger = [](float a, float b) { return max(a, b); };
                largest = fold<32>(fold<16>(largest, larger), larger);
                const int up = min(14 + 127 - (int)(float_bits(largest) >> 23), 126);  // -113 .. 126
                factor = bits_float((unsigned)(127 + up) << 23);
                back[m] = bits_float((unsigned)(127 - up) << 23);
            }
#pragma unroll
            for (int step = 0; step < STEPS; ++step) {
                T high_of[C], low_of[C];
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const float x = v[step][c] * factor;
                    high_of[c] = (T)x;
                    const float rest = x - (float)high_of[c];
                    low_of[c] = (T)(__builtin_fabsf(rest) < __builtin_inff() ? rest : 0.0f);  // infinities stand in `high`
                }
                __builtin_memcpy(&high[m][step], high_of, 16);
                __builtin_memcpy(&low[m][step], low_of, 16);
            }
        }
    }
    const T *b_of = B + (size_t)max(t.expert, 0) * sh.N * sh.R;
    // Stores are counted with the loads, in order, so that a load behind a store
    // waits for it: the next 64 columns are asked for before these are stored.
    // The two sets of operands change places by a copy, though, for which the
    // compiler waits until all of a turn's loads and stores are done, so that only
    // the stores' issue overlaps with the loads.  8192 tokens, rank 64, 4096 columns
    // fp16: 55 of the 91 us in all.
    // (Ranks over 64 have no registers for two, and one turn.)
    struct Operands {
        uint4v p[STEPS][4], y[MT][PER == 1 ? 4 : 2];
    };
    auto ask = [&](Operands &o, int n0) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int b = 0; b < 16 / C; ++b) {
                const int col = n0 + b * 4 * C + g * C;
                o.y[m][b] = load_chunk<T>(base + (base && token[m] >= 0 ? (size_t)token[m] * sh.N + col : 0),
                                                   base && token[m] >= 0 ? sh.N - col : 0);
            }
        if (t.expert < 0) return;
#pragma unroll
        for (int step = 0; step < STEPS; ++step) {
            const int r = step * STEP + g * C;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int col = n0 + b / PER * 4 * C + (i >> 2) * C + b % PER * 4 + (i & 3);
                o.p[step][b] = load_chunk<T>(b_of + (size_t)(col < sh.N ? col : 0) * sh.R + r,
                                                      col < sh.N ? sh.R - r : 0);
            }
        }
    };
    auto finish = [&](const Operands &o, int n0, auto next) {
        float4v acc[MT][4] = {};
        if (t.expert >= 0) {
#pragma unroll
            for (int step = 0; step < STEPS; ++step)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        acc[m][b] = mma<T>(o.p[step][b], high[m][step], acc[m][b]);
                        if constexpr (sizeof(T) == 2) acc[m][b] = mma<T>(o.p[step][b], low[m][step], acc[m][b]);
                    }
        }
        next();
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (token[m] < 0) continue;
            const float down = __is_same(T, half_t) && t.expert >= 0 ? back[m] : 1.0f;
#pragma unroll
            for (int b = 0; b < 16 / C; ++b) {
                const int col = n0 + b * 4 * C + g * C;
                T of_base[C];
                __builtin_memcpy(of_base, &o.y[m][b], 16);
                float part[C];
#pragma unroll
                for (int c = 0; c < C; ++c)
                    part[c] = __builtin_fmaf(acc[m][b * PER + c / 4][c % 4], down, (float)of_base[c]);
                store_vec<T, C>(Y + (size_t)token[m] * sh.N + col, part, sh.N - col);
            }
        }
    };
    const int end = min((int)(blockIdx.x + 1) * columns, sh.N);
    int n0 = blockIdx.x * columns + wave * 64;
    if (n0 >= end) return;
    Operands now;
    ask(now, n0);
    if constexpr (RANK > 2) {
        finish(now, n0, [] {});
    } else {
        for (;; n0 += kWaves * 64) {
            Operands ahead = now;
            const int n1 = n0 + kWaves * 64;
            finish(now, n0, [&] { if (n1 < end) ask(ahead, n1); });
            if (n1 >= end) break;
            now = ahead;
        }
    }
}

AdaptersShape make_shape(int T, int E, int R, int K, int N)
{
    int padded = 16;
    while (padded < R) padded *= 2;
    // Taller tiles from 128 tokens an adapter on.  Measured with and without, K = N =
    // 4096 fp16, us: rank 64, 12 adapters: 683 tokens each 91 / 106, 512: 83 / 83, 256:
    // 72 / 54, 128: 68 / 43, 64: 46 / 28; 4 adapters: 512: 72 / 43; rank 256, 4 adapters:
    // 512: 281 / 135; rank 16, 12 adapters: 512: 51 / 44.  So they gain at long segments of
    // many adapters alone, where the short tiles fill the GPU several times over.
    AdaptersShape sh{T, E, R, K, N, padded, 1, K, T >= 128LL * E};
    // Parts of the sum over K: about 512 workgroups, each with at least 256 of K.
    const long long tiles = num_row_tiles(T, E < T ? E : T, sh.tall ? 64 : 16);
    long long splits = (512 + tiles - 1) / (tiles > 0 ? tiles : 1);
    if (splits > K / 256) splits = K / 256;
    if (splits > 16) splits = 16;
    if (splits < 1) splits = 1;
    sh.per_split = (ceil_div(K, splits) + 63) / 64 * 64;
    sh.splits = ceil_div(K, sh.per_split);
    return sh;
}

// MT of the first kernel: what fits the registers beside the rank.
constexpr int shrink_tiles(int RT) { return RT <= 4 ? 4 : RT == 8 ? 2 : 1; }

template <typename T, int RT, int MT>
int launch_shrink(const T *X, const T *A, const int *ptr, const int *row_of, float *V, const AdaptersShape &sh,
                  hipStream_t st)
{
    const dim3 grid((unsigned)num_row_tiles(sh.T, sh.E, 16 * MT), sh.splits);
    hipLaunchKernelGGL((adapters_shrink_kernel<T, RT, MT>), grid, dim3(64 * kWaves), 0, st, X, A, ptr, row_of, V, sh);
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

template <typename T, int RANK, int MT>
int launch_expand(const float *V, const T *B, const float *scale, const T *base, T *Y, const int *ptr, const int *row_of,
                  const AdaptersShape &sh, hipStream_t st)
{
    const long long tiles = num_row_tiles(sh.T, sh.E, 16 * MT) + 1;
    // Columns of a workgroup: as many as leave about 1024 of them, at most 1024, so that V is not read too often.
    long long columns = (long long)sh.N * tiles / 1024 / 256 * 256;
    columns = columns < 256 || RANK > 2 ? 256 : columns > 1024 ? 1024 : columns;
    const dim3 grid(ceil_div(sh.N, columns), (unsigned)tiles);
    hipLaunchKernelGGL((adapters_expand_kernel<T, RANK, MT>), grid, dim3(64 * kWaves), 0, st, V, B, scale, base, Y, ptr,
                       row_of, (int)columns, sh);
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

template <typename T>
int launch_adapters(const void *X_, const void *A_, const void *B_, const float *scale, const void *base_, void *Y_,
                    const int *ptr, const int *row_of, const AdaptersShape &sh, float *V, hipStream_t st)
{
    const T *X = static_cast<const T *>(X_), *A = static_cast<const T *>(A_), *B = static_cast<const T *>(B_);
    const T *base = static_cast<const T *>(base_);
    T *Y = static_cast<T *>(Y_);
    int rc;
#define MPS_SHRINK(RT)                                                                                 \
    rc = sh.tall ? launch_shrink<T, RT, shrink_tiles(RT)>(X, A, ptr, row_of, V, sh, st)                \
                 : launch_shrink<T, RT, 1>(X, A, ptr, row_of, V, sh, st)
    if (sh.padded <= 16) MPS_SHRINK(1);
    else if (sh.padded <= 32) MPS_SHRINK(2);
    else if (sh.padded <= 64) MPS_SHRINK(4);
    else if (sh.padded <= 128) MPS_SHRINK(8);
    else MPS_SHRINK(16);
#undef MPS_SHRINK
    if (rc != MPS_OK) return rc;
#define MPS_EXPAND(RANK)                                                                                         \
    return sh.tall && RANK <= 2 ? launch_expand<T, RANK, RANK <= 2 ? 2 : 1>(V, B, scale, base, Y, ptr, row_of, sh, st) \
                                  : launch_expand<T, RANK, 1>(V, B, scale, base, Y, ptr, row_of, sh, st)
    // Tiles of 32 tokens: 8192 tokens, rank 64, 4096 columns take 91 us in all, 106 with 16, 156 with 64, which
    // leave one wavefront a SIMD.  Ranks from 65 to 256 share one kernel, with the matrix work of 256: 12 adapters of
    // 512 tokens take 83 us at rank 64, 229 at 128, 453 at 256.
    if (sh.R <= 32) MPS_EXPAND(1);
    if (sh.R <= 64) MPS_EXPAND(2);
    MPS_EXPAND(8);
#undef MPS_EXPAND
}

int check_adapters(int T, int E, int R, int K)
{
    if (T < 0 || E < 1 || R < 1 || K < 1) return MPS_ERR_INVALID_ARG;
    if (R > MPS_ADAPTERS_MAX_RANK || E > MPS_ROUTE_MAX_EXPERTS || T > MPS_ADAPTERS_MAX_TOKENS || K > INT_MAX / 4)
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
