// Products of the experts: a matrix for every expert, times the rows that the
// routing matrix sends there, with their two gradients.
//
// One scheme does all three.  A workgroup owns a tile of the result, of panels
// of S = 128 or 64: P counts its columns (contiguous in memory), Q its rows,
//   D[q, p] = sum_r Q[q, r] P[p, r],
// with r the summed index.  An operand is stored either with r contiguous
// (rows of 128 bytes of r are staged, one per q or p) or with p / q contiguous
// (rows of S elements are staged, one per r, and turned while they are read
// from LDS):
//                r             P                       Q
//   product      K             W[e], r contiguous      X, r contiguous
//   dX           N             W[e], p contiguous      dY, r contiguous
//   dW           places of e   X, p contiguous         dY, q contiguous
// P is the first operand of the matrix instruction, whose result gives a lane
// four neighbouring p of one q: stores of 8 or 16 bytes.
#include "mpspmm_routing.hpp"

#include <type_traits>

namespace {

typedef short short4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) short4v *lds_short4;

constexpr int kThreads = 256;

template <typename T>
struct Elem {
    static constexpr int kPerChunk = 16 / sizeof(T);
    static constexpr int kDepth = 128 / sizeof(T);      // r per stage
    static constexpr int kStep = 4 * kPerChunk;         // r per matrix step: lane group g takes chunk g
};

// Where chunk c of staged row `row` lies, so that the 16 lanes that read
// together meet 16 different chunks of the 256 bytes that LDS gives at once.
//   r contiguous: 8 chunks a row, lanes read the same chunk of 16 rows.
template <typename T>
__device__ __forceinline__ int place_rows(int row, int c)
{
    return (row * 8 + (c ^ ((row >> 1) & 7))) * 16;
}
//   p / q contiguous, 16-bit: the turning read takes 32 bytes of each of the rows
//   8 g + 0 .. 3 (or 4 .. 7), g = 0 .. 3; fp32: lanes take 64 bytes of the rows
//   4 g + j.
template <typename T, int S>
__device__ __forceinline__ int place_turned(int row, int c)
{
    constexpr int CHUNKS = S / Elem<T>::kPerChunk;  // of a staged row
    if constexpr (sizeof(T) == 4) return (row * CHUNKS + (c ^ (((row >> 2) & 3) << 2))) * 16;
    else if constexpr (S == 128) return (row * CHUNKS + (c ^ (((row & 3) | ((row >> 1) & 4)) << 1))) * 16;
    else return (row * CHUNKS + (c ^ (((row >> 1 & 1) | ((row >> 2) & 2)) << 1))) * 16;
}

// What a lane feeds to the matrix instruction for 16 neighbouring outer indices,
// the (first + n)-th 16 of a panel, and matrix step s.  The places above differ
// between n and s by sums and exclusive ors of constants only, so that a lane
// needs one base: `first` a multiple of a power of two above n.
template <typename T, bool TURNED, int S>
__device__ __forceinline__ int fragment_base(int first, int lane)
{
    const int i = lane & 15, g = lane >> 4;
    if constexpr (!TURNED) return place_rows<T>(first * 16 + i, g);
    else if constexpr (sizeof(T) == 2) return place_turned<T, S>(8 * g + (i >> 2), first * 2 + ((i & 3) >> 1)) + (i & 1) * 8;
    else return place_turned<T, S>(4 * g, first * 4 + (i >> 2)) + (i & 3) * 4;
}
template <typename T, bool TURNED, int S>
__device__ __forceinline__ uint4v fragment(const char *panel, int base, int n, int s)
{
    constexpr int ROW_BYTES = S * sizeof(T);  // of a staged row to be turned
    if constexpr (!TURNED) {
        return *reinterpret_cast<const uint4v *>(panel + (base ^ (s << 6)) + n * 2048);
    } else if constexpr (sizeof(T) == 2) {
        // 16 lanes read a block of 4 rows (r) by 16 elements, 8 bytes each, and get it turned
        const char *at = panel + (base ^ (n << 5)) + s * (32 * ROW_BYTES);
        union {
            short4v part[2];
            uint4v all;
        } u;
        u.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)at);
        u.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4)(at + 4 * ROW_BYTES));
        return u.all;
    } else {
        const char *at = panel + (base ^ (n << 6)) + s * (16 * ROW_BYTES);
        uint4v v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const unsigned *>(at + j * ROW_BYTES);
        return v;
    }
}

struct ExpertsShape {
    int M, E, N, K, k;
    int col_tiles, row_tiles;
    unsigned k_magic, k_shift;  // slot / k = slot * k_magic >> k_shift, see divide_by()
};

// s / k for 0 <= s < 2^31: with 2^(L - 1) < k <= 2^L and m = ceil(2^(31 + L) / k), m k exceeds 2^(31 + L) by less than
// k <= 2^L, so that s m / 2^(31 + L) exceeds s / k by less than 1 / k.  m < 2^32.
void divide_by(int k, unsigned &magic, unsigned &shift)
{
    unsigned L = 0;
    while ((1ll << L) < k) ++L;
    shift = 31 + L;
    magic = (unsigned)(((1ull << shift) + (unsigned)k - 1) / (unsigned)k);
}
__device__ __forceinline__ unsigned token_of(unsigned slot, const ExpertsShape &sh)
{
    return (unsigned)(((unsigned long long)slot * sh.k_magic) >> sh.k_shift);
}

enum Product { kForward, kRows, kWeights };

template <typename T, Product WHAT, int S>
__global__ __launch_bounds__(kThreads, 2) void experts_tile_kernel(const T *__restrict__ A, const T *__restrict__ B,
                                                                   T *__restrict__ out, const int *__restrict__ ptr,
                                                                   const int *__restrict__ slot, ExpertsShape sh)
{
    // product: A = X, B = W, out = Y; dX: A = dY, B = W, out = dX; dW: A = dY, B = X, out = dW
    constexpr bool PT = WHAT != kForward, QT = WHAT == kWeights;
    constexpr int V = Elem<T>::kPerChunk, DEPTH = Elem<T>::kDepth, ROW = S / V;
    constexpr int CHUNKS = S * 128 / 16 / kThreads;  // 16-byte chunks of an operand's stage per thread
    constexpr int F = S / 32;                        // 16s of a wavefront's share, either way
    __shared__ __attribute__((aligned(16))) char stage_p[2][S * 128];
    __shared__ __attribute__((aligned(16))) char stage_q[2][S * 128];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int cols = WHAT == kForward ? sh.N : sh.K;
    const int number = xcd_tile(blockIdx.x, gridDim.x);
    const int col0 = number % sh.col_tiles * S;
    const int rest = number / sh.col_tiles;
    int expert, row0, rows, first, depth;  // rows of the tile in the result; places summed over from `first` on
    if constexpr (WHAT == kWeights) {
        expert = rest / sh.row_tiles;
        row0 = rest % sh.row_tiles * S;
        rows = min(sh.N - row0, S);
        first = clamp_place(ptr[expert], sh.M);
        depth = max(clamp_place(ptr[expert + 1], sh.M) - first, 0);
    } else {
        const RowTile t = find_row_tile<S>(ptr, sh.E, sh.M, rest);
        if (t.rows == 0) return;
        expert = t.expert;
        row0 = first = t.first;
        rows = t.rows;
        depth = WHAT == kForward ? sh.K : sh.N;
    }
    const T *W = WHAT == kWeights ? nullptr : B + (size_t)expert * sh.N * sh.K;

    // The chunks that this thread stages.
    const T *p_src[CHUNKS], *q_src[CHUNKS];
    int p_valid[CHUNKS], q_valid[CHUNKS];  // turned: elements from the chunk's column on; else unused (row given or null)
#pragma unroll
    for (int n = 0; n < CHUNKS; ++n) {
        const int id = tid + n * kThreads;
        if constexpr (PT) {
            const int c = id % ROW;
            p_src[n] = (WHAT == kRows ? W : B) + col0 + c * V;
            p_valid[n] = cols - (col0 + c * V);
        } else {
            const int row = id / 8;
            p_src[n] = col0 + row < cols ? W + (size_t)(col0 + row) * sh.K : nullptr;
        }
        if constexpr (QT) {
            const int c = id % ROW;
            q_src[n] = A + row0 + c * V;
            q_valid[n] = sh.N - (row0 + c * V);
        } else {
            const int row = id / 8;
            q_src[n] = nullptr;
            if (row < rows) {
                int from = first + row;
                if (WHAT == kForward && slot) {
                    const int s = slot[from];
                    from = (unsigned)s < (unsigned)sh.M ? (int)token_of(s, sh) : -1;
                }
                if (from >= 0) q_src[n] = A + (size_t)from * (WHAT == kForward ? sh.K : sh.N);
            }
        }
    }
    uint4v p_hold[CHUNKS], q_hold[CHUNKS];
    auto fetch = [&](int r0) {
#pragma unroll
        for (int n = 0; n < CHUNKS; ++n) {
            const int id = tid + n * kThreads;
            if constexpr (PT) {
                const int r = r0 + id / ROW;
                long long from = -1;
                if (r < depth) {
                    from = r;
                    if constexpr (WHAT == kWeights) {
                        from = first + r;
                        if (slot) {
                            const int s = slot[from];
                            from = (unsigned)s < (unsigned)sh.M ? (int)token_of(s, sh) : -1;
                        }
                    }
                }
                p_hold[n] = load_chunk<T>(p_src[n] + (from < 0 ? 0 : from * sh.K), from < 0 ? 0 : p_valid[n]);
            } else {
                const int r = r0 + id % 8 * V;
                p_hold[n] = load_chunk<T>(p_src[n] + r, p_src[n] ? depth - r : 0);
            }
            if constexpr (QT) {
                const int r = r0 + id / ROW;
                q_hold[n] = load_chunk<T>(q_src[n] + (size_t)(first + (r < depth ? r : 0)) * sh.N,
                                                   r < depth ? q_valid[n] : 0);
            } else {
                const int r = r0 + id % 8 * V;
                q_hold[n] = load_chunk<T>(q_src[n] + r, q_src[n] ? depth - r : 0);
            }
        }
    };
    auto put = [&](int buffer) {
#pragma unroll
        for (int n = 0; n < CHUNKS; ++n) {
            const int id = tid + n * kThreads;
            const int p_at = PT ? place_turned<T, S>(id / ROW, id % ROW)
                                : place_rows<T>(id / 8, id % 8);
            const int q_at = QT ? place_turned<T, S>(id / ROW, id % ROW)
                                : place_rows<T>(id / 8, id % 8);
            *reinterpret_cast<uint4v *>(stage_p[buffer] + p_at) = p_hold[n];
            *reinterpret_cast<uint4v *>(stage_q[buffer] + q_at) = q_hold[n];
        }
    };

    float4v acc[F][F] = {};  // [q][p]
    const int p_base = (wave & 1) * (S / 2), q_base = (wave >> 1) * (S / 2);
    const int p_at = fragment_base<T, PT, S>(p_base / 16, lane), q_at = fragment_base<T, QT, S>(q_base / 16, lane);
    if (depth > 0) {
        fetch(0);
        put(0);
    }
    __syncthreads();
    int buffer = 0;
    for (int r0 = 0; r0 < depth; r0 += DEPTH) {
        const bool more = r0 + DEPTH < depth;
        if (more) fetch(r0 + DEPTH);
#pragma unroll
        for (int s = 0; s < DEPTH / Elem<T>::kStep; ++s) {
            uint4v p[F], q[F];
#pragma unroll
            for (int n = 0; n < F; ++n) {
                p[n] = fragment<T, PT, S>(stage_p[buffer], p_at, n, s);
                q[n] = fragment<T, QT, S>(stage_q[buffer], q_at, n, s);
            }
#pragma unroll
            for (int a = 0; a < F; ++a)
#pragma unroll
                for (int b = 0; b < F; ++b) acc[a][b] = mma<T>(p[b], q[a], acc[a][b]);
        }
        if (more) put(buffer ^ 1);
        __syncthreads();
        buffer ^= 1;
    }

    // Lane: q = lane % 16, four p from (lane / 16) * 4 on.
#pragma unroll
    for (int a = 0; a < F; ++a) {
        const int q = q_base + 16 * a + (lane & 15);
        if (q >= rows) continue;
        T *row = out + (WHAT == kWeights ? (size_t)expert * sh.N * sh.K + (size_t)(row0 + q) * sh.K
                                         : (size_t)(row0 + q) * cols);
#pragma unroll
        for (int b = 0; b < F; ++b) {
            const int p = col0 + p_base + 16 * b + (lane >> 4) * 4;
            const float v[4] = {acc[a][b][0], acc[a][b][1], acc[a][b][2], acc[a][b][3]};
            if (p < cols) store_vec<T, 4>(row + p, v, cols - p);
        }
    }
}

// The same products where rows are whole 16 bytes.  The stages come straight
// from memory into LDS, two of them in turn: while the matrix instructions work
// on one, the other is on its way.  Measured, 256 x 256 tiles, fp16: 1202 TFLOP/s
// for one expert of 8192 x 8192 x 8192 (a library product: 1414), 897 for 64
// experts of 768 rows, 1408 x 2048 (a last tile of half the columns), 820 - 840
// where their rows are uneven.  Four stages of one matrix step, for requests three
// ahead, and sums that begin at another place in every column tile gave nothing:
// neither the way from memory nor its channels bound it.
//   PP, QP  panels of S in the tile's columns and rows
//   WP, WQ  wavefronts that share them
typedef __attribute__((address_space(3))) void *lds_ptr;

template <typename T, Product WHAT, int S, int PP, int QP, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ, 2) void experts_stream_kernel(const T *__restrict__ A, const T *__restrict__ B,
                                                                         T *__restrict__ out,
                                                                         const int *__restrict__ ptr,
                                                                         const int *__restrict__ slot, ExpertsShape sh)
{
    constexpr bool PT = WHAT != kForward, QT = WHAT == kWeights;
    constexpr int V = Elem<T>::kPerChunk, DEPTH = Elem<T>::kDepth, ROW = S / V;
    constexpr int THREADS = 64 * WP * WQ, BP = PP * S, BQ = QP * S, PANEL = S * 128;
    constexpr int PC = PP * PANEL / 16 / THREADS, QC = QP * PANEL / 16 / THREADS;  // chunks of a thread
    constexpr int FP = BP / 16 / WP, FQ = BQ / 16 / WQ;                           // fragments of a wavefront
    __shared__ __attribute__((aligned(16))) char stage0[(PP + QP) * PANEL];
    __shared__ __attribute__((aligned(16))) char stage1[(PP + QP) * PANEL];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cols = WHAT == kForward ? sh.N : sh.K;
    const int number = xcd_tile(blockIdx.x, gridDim.x);
    const int col0 = number % sh.col_tiles * BP;
    const int rest = number / sh.col_tiles;
    int expert, row0, rows, first, depth;
    if constexpr (WHAT == kWeights) {
        expert = rest / sh.row_tiles;
        row0 = rest % sh.row_tiles * BQ;
        rows = min(sh.N - row0, BQ);
        first = clamp_place(ptr[expert], sh.M);
        depth = max(clamp_place(ptr[expert + 1], sh.M) - first, 0);
    } else {
        const RowTile t = find_row_tile<BQ>(ptr, sh.E, sh.M, rest);
        if (t.rows == 0) return;
        expert = __builtin_amdgcn_readfirstlane(t.expert);
        row0 = first = __builtin_amdgcn_readfirstlane(t.first);
        rows = __builtin_amdgcn_readfirstlane(t.rows);
        depth = WHAT == kForward ? sh.K : sh.N;
    }

    // Chunk n of this thread lies at (n * THREADS + tid) * 16 of its operand.  It
    // comes from the stage's base, which all threads share, plus an offset of 32
    // bits (the launcher sees to that).  A row or column that does not exist is
    // replaced by the last one that does: what is made of it is not stored.
    // Chunks behind the end of the sum, and rows whose slot is out of range, are
    // asked for behind the end of the buffer, which gives zeros.
    constexpr unsigned kBufferEnd = 0x80000000u;
    const char *p_now, *q_now;
    unsigned p_off[PC], q_off[QC];
    const long long p_step = (PT ? (long long)DEPTH * sh.K : DEPTH) * (long long)sizeof(T);
    const long long q_step = (QT ? (long long)DEPTH * sh.N : DEPTH) * (long long)sizeof(T);
    constexpr bool LIST = WHAT == kWeights;  // rows of P are looked up for every stage
    // where chunk n begins in its staged row, and the summed index it begins with in a stage
    auto turned_at = [&](int n) { return place_turned<T, S>(tid / ROW + n * THREADS / ROW % DEPTH, tid % ROW) / 16 % ROW * V; };
    const int row_at = place_rows<T>(tid / 8, tid % 8) / 16 % 8 * V;  // the same for all n
    static_assert(THREADS / 8 % 16 == 0, "rows of equal place");
    auto p_r = [&](int n) { return PT ? tid / ROW + n * THREADS / ROW % DEPTH : row_at; };
    auto q_r = [&](int n) { return QT ? tid / ROW + n * THREADS / ROW % DEPTH : row_at; };
#pragma unroll
    for (int n = 0; n < PC; ++n) {
        const int panel = n * THREADS / (PANEL / 16);
        if constexpr (PT) {
            const int col = min(col0 + panel * S + turned_at(n), cols - V);
            p_off[n] = (unsigned)((LIST ? 0u : (unsigned)p_r(n) * (unsigned)sh.K) + col) * (unsigned)sizeof(T);
        } else {
            const int col = min(col0 + (n * THREADS + tid) / 8, cols - 1);
            p_off[n] = ((unsigned)col * (unsigned)sh.K + row_at) * (unsigned)sizeof(T);
        }
    }
    p_now = reinterpret_cast<const char *>(LIST ? B : B + (size_t)expert * sh.N * sh.K);
#pragma unroll
    for (int n = 0; n < QC; ++n) {
        const int panel = n * THREADS / (PANEL / 16);
        if constexpr (QT) {
            const int at = min(row0 + panel * S + turned_at(n), sh.N - V);
            q_off[n] = ((unsigned)q_r(n) * (unsigned)sh.N + at) * (unsigned)sizeof(T);
        } else {
            const int at = min((n * THREADS + tid) / 8, rows - 1);
            int from = at;
            if constexpr (WHAT == kForward) {
                from += first;
                if (slot) {
                    const int s = slot[from];
                    const bool is = (unsigned)s < (unsigned)sh.M;
                    from = is ? (int)token_of(s, sh) : -1;
                }
            }
            q_off[n] = from < 0 ? kBufferEnd
                                : ((unsigned)from * (unsigned)(WHAT == kForward ? sh.K : sh.N) + row_at) * (unsigned)sizeof(T);
        }
    }
    q_now = reinterpret_cast<const char *>(WHAT == kForward ? A : A + (size_t)first * sh.N);
    // Rows of P for the next stage (dW): looked up one stage ahead.
    int row_of[PC];
    auto look_up = [&](int r0) {
#pragma unroll
        for (int n = 0; n < PC; ++n) {
            const int r = r0 + p_r(n);
            int from = r < depth ? first + r : -1;
            if (slot && from >= 0) from = slot[from];
            row_of[n] = from;
        }
    };
    auto request = [&](const char *base, unsigned off, char *stage, int n) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), 0, kBufferEnd, 0x00020000),
            (lds_ptr)(stage + (n * THREADS + wave * 64) * 16), 16, off, 0, 0, 0);
    };
    auto issue = [&](char *stage, int r0) {
#pragma unroll
        for (int n = 0; n < PC; ++n) {
            unsigned off;
            if constexpr (LIST) {
                const int s = row_of[n];
                const bool is = slot ? (unsigned)s < (unsigned)sh.M : s >= 0;
                const unsigned row = slot ? token_of(s, sh) : (unsigned)s;
                off = is ? p_off[n] + row * (unsigned)sh.K * (unsigned)sizeof(T) : kBufferEnd;
            } else {
                off = r0 + p_r(n) < depth ? p_off[n] : kBufferEnd;
            }
            request(p_now, off, stage, n);
        }
#pragma unroll
        for (int n = 0; n < QC; ++n)
            request(q_now, r0 + q_r(n) < depth ? q_off[n] : kBufferEnd, stage + PP * PANEL, n);
        if constexpr (!LIST) p_now += p_step;
        q_now += q_step;
    };

    float4v acc[FQ][FP] = {};
    // Wavefronts w and w + 4 share a SIMD.  Where there are 8 they take opposite
    // halves of both the columns and the rows, and one whose rows or columns do not
    // exist has no work: a tile that is half empty takes half the time.
    constexpr bool EIGHT = WP == 2 && WQ == 4;
    const int p_part = EIGHT ? (wave & 1) ^ (wave >> 2) : wave % WP;
    const int q_part = EIGHT ? (wave >> 1 & 1) | (wave >> 2) << 1 : wave / WP;
    const int p_base = p_part * (FP * 16), q_base = q_part * (FQ * 16);
    // Two loops, one of requests alone: branches within one make the compiler wait
    // for what is on its way to LDS.  dW has the branches (with two loops it has
    // not the registers: 436 us in place of 245, 32768 rows 1024 x 2048 bf16).
    const bool busy = q_base < rows && col0 + p_base < cols;
    static_assert(FP * 16 <= S && FQ * 16 <= S, "a wavefront's part of an operand lies in one panel");
    int p_at = p_base / S * PANEL + fragment_base<T, PT, S>(p_base % S / 16, lane);
    int q_at = (PP + q_base / S) * PANEL + fragment_base<T, QT, S>(q_base % S / 16, lane);
    auto arrive = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0): own chunks have come, own reads of LDS are done
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // A stage is two matrix steps, a step two halves of P: four groups of matrix
    // instructions.  What a group needs is read from LDS while the group before
    // it works, across the stages too: everybody has read all of a stage before
    // its last group, which the first reads of the next stage and the requests
    // for the one after that go along with.
    static_assert(DEPTH == 2 * Elem<T>::kStep, "a stage is two matrix steps");
    constexpr int HALF = FP / 2;
    uint4v q[2][FQ], p[2][HALF];
    auto read_q = [&](const char *stage, int s, int to) {
#pragma unroll
        for (int n = 0; n < FQ; ++n) q[to][n] = fragment<T, QT, S>(stage, q_at, n, s);
    };
    auto read_p = [&](const char *stage, int s, int half) {
#pragma unroll
        for (int n = 0; n < HALF; ++n) p[half][n] = fragment<T, PT, S>(stage, p_at, half * HALF + n, s);
    };
    auto group = [&](int of, int half) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int a = 0; a < FQ; ++a)
#pragma unroll
            for (int b = 0; b < HALF; ++b) acc[a][half * HALF + b] = mma<T>(p[half][b], q[of][a], acc[a][half * HALF + b]);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto turn = [&](auto works, char *now, const char *next, int r0) {
        const bool on = LIST ? busy : decltype(works)::value;
        // the places that follow from these are made anew in every turn, not kept in registers for all
        if constexpr (PT) asm volatile("" : "+v"(p_at));
        if constexpr (QT) asm volatile("" : "+v"(q_at));
        if (on) {
            read_p(now, 0, 1);
            group(0, 0);
            read_q(now, 1, 1);
            read_p(now, 1, 0);
            group(0, 1);
            read_p(now, 1, 1);
            group(1, 0);
        }
        arrive();  // the next stage has come, and everybody is done with this one
        if (on) {
            read_q(next, 0, 0);
            read_p(next, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        issue(now, r0 + 2 * DEPTH);
        if constexpr (LIST) look_up(r0 + 3 * DEPTH);
        if (on) group(1, 1);
    };

    // Two stages a turn, behind the end of the sum ones of zeros.
    if constexpr (LIST) look_up(0);
    issue(stage0, 0);
    if constexpr (LIST) look_up(DEPTH);
    arrive();
    issue(stage1, DEPTH);
    if constexpr (LIST) look_up(2 * DEPTH);
    if (LIST || busy) {
        read_q(stage0, 0, 0);
        read_p(stage0, 0, 0);
        for (int r0 = 0; r0 < depth; r0 += 2 * DEPTH) {
            turn(std::true_type{}, stage0, stage1, r0);
            turn(std::true_type{}, stage1, stage0, r0 + DEPTH);
        }
    } else {  // the same requests and barriers
        for (int r0 = 0; r0 < depth; r0 += 2 * DEPTH) {
            turn(std::false_type{}, stage0, stage1, r0);
            turn(std::false_type{}, stage1, stage0, r0 + DEPTH);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0070);  // nothing is on its way into LDS when the workgroup ends

#pragma unroll
    for (int a = 0; a < FQ; ++a) {
        const int q = q_base + 16 * a + (lane & 15);
        if (q >= rows) continue;
        T *row = out + (WHAT == kWeights ? (size_t)expert * sh.N * sh.K + (size_t)(row0 + q) * sh.K
                                         : (size_t)(row0 + q) * cols);
#pragma unroll
        for (int b = 0; b < FP; ++b) {
            const int p = col0 + p_base + 16 * b + (lane >> 4) * 4;
            const float v[4] = {acc[a][b][0], acc[a][b][1], acc[a][b][2], acc[a][b][3]};
            if (p < cols) store_vec<T, 4>(row + p, v, cols - p);
        }
    }
}

template <typename T, Product WHAT, int S, int PP, int QP, int WP, int WQ>
int launch_stream(const void *A, const void *B, void *out, const int *ptr, const int *slot, ExpertsShape sh, hipStream_t st)
{
    sh.col_tiles = ceil_div(WHAT == kForward ? sh.N : sh.K, PP * S);
    sh.row_tiles = ceil_div(sh.N, QP * S);
    const long long others = WHAT == kWeights ? (long long)sh.E * sh.row_tiles : num_row_tiles(sh.M, sh.E, QP * S);
    if (!fits_launch(others, sh.col_tiles, 64 * WP * WQ)) return MPS_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((experts_stream_kernel<T, WHAT, S, PP, QP, WP, WQ>), dim3((unsigned)(others * sh.col_tiles)),
                       dim3(64 * WP * WQ), 0, st, static_cast<const T *>(A), static_cast<const T *>(B),
                       static_cast<T *>(out), ptr, slot, sh);
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

// The product where experts have a few rows each, as in decoding: the weights'
// bytes are the time, and every one is used once.  One workgroup per tile of
// 16 MT rows and 64 columns; its four wavefronts take 128 bytes of the rows in
// turn, straight into the matrix instructions' registers, and add up through
// LDS.  No barrier until the end, so that many loads are on their way.
constexpr int kFewWaves = 4, kFewColumns = 4;  // in 16s

template <typename T, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void experts_few_kernel(const T *__restrict__ X, const T *__restrict__ W,
                                                                     T *__restrict__ Y, const int *__restrict__ ptr,
                                                                     const int *__restrict__ slot, ExpertsShape sh)
{
    constexpr int C = 16 / sizeof(T), STEP = 4 * C, RT = kFewColumns;
    __shared__ float4v join[kFewWaves][RT][64];
    const RowTile t = find_row_tile<16 * MT>(ptr, sh.E, sh.M, blockIdx.x / sh.col_tiles);
    if (t.rows == 0) return;
    const int col0 = blockIdx.x % sh.col_tiles * (16 * RT);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = lane & 15, g = lane >> 4;
    const T *x[MT], *w[RT];
    bool live[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        int from = 16 * m + i < t.rows ? t.first + 16 * m + i : -1;
        if (slot && from >= 0) {
            const int s = slot[from];
            from = (unsigned)s < (unsigned)sh.M ? (int)token_of(s, sh) : -1;
        }
        live[m] = from >= 0;
        x[m] = X + (size_t)max(from, 0) * sh.K;
    }
#pragma unroll
    for (int n = 0; n < RT; ++n) w[n] = W + ((size_t)t.expert * sh.N + min(col0 + n * 16 + i, sh.N - 1)) * sh.K;
    float4v acc[MT][RT] = {};
    for (int base = wave * 2 * STEP; base < sh.K; base += kFewWaves * 2 * STEP) {
        uint4v p[2][RT], q[2][MT];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k = base + half * STEP + g * C;
#pragma unroll
            for (int n = 0; n < RT; ++n) p[half][n] = load_chunk<T>(w[n] + k, sh.K - k);
#pragma unroll
            for (int m = 0; m < MT; ++m) q[half][m] = load_chunk<T>(x[m] + k, live[m] ? sh.K - k : 0);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < RT; ++n) acc[m][n] = mma<T>(p[half][n], q[half][m], acc[m][n]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (m > 0) __syncthreads();
#pragma unroll
        for (int n = 0; n < RT; ++n) join[wave][n][lane] = acc[m][n];
        __syncthreads();
        const int col = col0 + wave * 16 + g * 4;  // as many 16s of columns as wavefronts
        if (16 * m + i < t.rows && col < sh.N) {
            float4v sum = join[0][wave][lane];
#pragma unroll
            for (int other = 1; other < kFewWaves; ++other) sum += join[other][wave][lane];
            const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
            store_vec<T, 4>(Y + (size_t)(t.first + 16 * m + i) * sh.N + col, v, sh.N - col);
        }
    }
}
static_assert(kFewColumns == kFewWaves, "a wavefront adds up 16 columns");

template <typename T, int MT>
int launch_few(const void *X, const void *W, void *Y, const int *ptr, const int *slot, ExpertsShape sh, hipStream_t st)
{
    sh.col_tiles = ceil_div(sh.N, 16 * kFewColumns);
    const long long tiles = num_row_tiles(sh.M, sh.E, 16 * MT);
    if (!fits_launch(tiles, sh.col_tiles, 64 * kFewWaves)) return MPS_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((experts_few_kernel<T, MT>), dim3((unsigned)(tiles * sh.col_tiles)), dim3(64 * kFewWaves), 0, st,
                       static_cast<const T *>(X), static_cast<const T *>(W), static_cast<T *>(Y), ptr, slot, sh);
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

template <typename T, Product WHAT, int S>
int launch_tile(const void *A, const void *B, void *out, const int *ptr, const int *slot, ExpertsShape sh, hipStream_t st)
{
    sh.col_tiles = ceil_div(WHAT == kForward ? sh.N : sh.K, S);
    sh.row_tiles = ceil_div(sh.N, S);
    const long long others = WHAT == kWeights ? (long long)sh.E * sh.row_tiles : num_row_tiles(sh.M, sh.E, S);
    if (!fits_launch(others, sh.col_tiles, kThreads)) return MPS_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((experts_tile_kernel<T, WHAT, S>), dim3((unsigned)(others * sh.col_tiles)), dim3(kThreads), 0, st,
                       static_cast<const T *>(A), static_cast<const T *>(B), static_cast<T *>(out), ptr, slot, sh);
    MPS_HIP_TRY(hipGetLastError());
    return MPS_OK;
}

template <typename T, Product WHAT>
int launch_experts(const void *A, const void *B, void *out, const int *ptr, const int *slot, int k, int M, int E, int N,
                   int K, hipStream_t st)
{
    ExpertsShape sh{M, E, N, K, k, 0, 0, 0, 0};
    divide_by(k, sh.k_magic, sh.k_shift);
    // every operand's rows are N or K long
    const bool fast = rows_of_16(A, WHAT == kForward ? K : N, sizeof(T)) && rows_of_16(B, K, sizeof(T)) &&
                      rows_of_16(out, WHAT == kForward ? N : K, sizeof(T));
    if constexpr (WHAT == kForward) {
        // Few rows an expert: the tiles below would be nearly empty and their workgroups few (32 tokens, 6 of 64 experts,
        // 2048 x 1024 bf16: 56 - 59 us, 62 - 80 with tiles of 128).  Measured on experts of uneven length, K = 2048, us
        // with 16 rows / 32 rows / the tiles below, by the mean rows of an expert:
        //   64 of 1408 columns, bf16   4: 72 / 68 / 89   9: 93 / 87 / 97   16: 114 / 97 / 96   24: 136 / 111 / 96
        //                       fp32   8: 180 / 217 / 445   16: 242 / 258 / 469   25: 303 / 300 / 469   48: 476 / 431 / 472
        //   32 of 1024 columns, bf16   4: 33 / 37 / 29    8: 38 / 38 / 30    24: 54 / 51 / 36
        //                       fp32   8: 78 / 108 / 74   24: 121 / 146 / 97
        // Where the tiles below are those of 64 they are ahead from 4 rows on, those of 128 from 16 (bf16) or 64 (fp32):
        // 24 lies between.
        if (M <= 8LL * E) return launch_few<T, 1>(A, B, out, ptr, slot, sh, st);
        if (M <= 24LL * E) return launch_few<T, 2>(A, B, out, ptr, slot, sh, st);
    }
    // Tiles of 64 where tiles of 128 would leave compute units without one.
    const long long others = WHAT == kWeights ? (long long)E * ceil_div(N, 128) : (long long)M / 128 + (E < M ? E : M);
    const bool small = others < 512 && others * ceil_div(WHAT == kForward ? N : K, 128) < 512;
    // 256 x 256 tiles from 384 rows on.  Measured on uneven experts, bf16, us with them / with tiles of 128 or 64:
    //   product, 32 of 1024 x 2048    256: 63 / 74    384: 108 / 81    512: 110 / 110   768: 122 / 152
    //            64 of 1408 x 2048    256: 169 / 164  384: 223 / 220   512: 259 / 272   768: 333 / 385
    //   dX,      64 of 1408 x 2048    128: 122 / 126  256: 162 / 181   384: 208 / 236   768: 361 / 413
    //   dW,      32 of 1024 x 2048     96: 60 / 70    256: 81 / 95     384: 96 / 111    768: 149 / 176
    // The rule looks at the rows alone.  Narrow matrices of few experts make few such tiles, and dW is never cut along
    // its places: 65536 rows, 2 experts of 64 x 64: dW 526 / 242, 16 of 256 x 512: dW 110 / 44, product 43 / 35.
    // offsets of 32 bits inside X or dY and inside the matrix of an expert
    const long long far = INT_MAX / (long long)sizeof(T);
    const bool near = (long long)M * (WHAT == kForward ? K : N) <= far && (long long)N * K <= far &&
                      (WHAT != kWeights || (long long)M * K <= far);
    if (fast && near) {
        if constexpr (sizeof(T) == 2) {
            if ((long long)M >= 384LL * E) return launch_stream<T, WHAT, 128, 2, 2, 2, 4>(A, B, out, ptr, slot, sh, st);
        }
        return small ? launch_stream<T, WHAT, 64, 1, 1, 2, 2>(A, B, out, ptr, slot, sh, st)
                     : launch_stream<T, WHAT, 128, 1, 1, 2, 2>(A, B, out, ptr, slot, sh, st);
    }
    return small ? launch_tile<T, WHAT, 64>(A, B, out, ptr, slot, sh, st)
                 : launch_tile<T, WHAT, 128>(A, B, out, ptr, slot, sh, st);
}
template <Product WHAT>
int experts_entry(const void *A, const void *B, void *out, int dtype, const int *ptr, const int *slot, int k, int M,
                  int E, int N, int K, void *stream)
{
    const int eb = dtype_bytes(dtype);
    if (!eb || M < 0 || E < 1 || N < 1 || K < 1 || k < 1 || M % k) return MPS_ERR_INVALID_ARG;
    if (M > INT_MAX - 65536 || N > INT_MAX / 4 || K > INT_MAX / 4) return MPS_ERR_UNSUPPORTED;
    if (!ptr || (M > 0 && !A) || (M > 0 || WHAT == kWeights ? !out : false) || (M > 0 && !B)) return MPS_ERR_INVALID_ARG;
    if (!aligned_to(A, eb) || !aligned_to(B, eb) || !aligned_to(out, eb) || !aligned_to(ptr, 4) || !aligned_to(slot, 4))
        return MPS_ERR_ALIGNMENT;
    if (M == 0 && WHAT != kWeights) return MPS_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == MPS_F32) return launch_experts<float, WHAT>(A, B, out, ptr, slot, k, M, E, N, K, st);
    if (dtype == MPS_F16) return launch_experts<half_t, WHAT>(A, B, out, ptr, slot, k, M, E, N, K, st);
    return launch_experts<bf16_t, WHAT>(A, B, out, ptr, slot, k, M, E, N, K, st);
}

}  // namespace

extern "C" {

int mps_experts_mm(const void *d_X, const void *d_W, void *d_Y, int dtype, const int *d_expert_ptr, const int *d_slot,
                   int k, int M, int E, int N, int K, void *stream)
{
    return experts_entry<kForward>(d_X, d_W, d_Y, dtype, d_expert_ptr, d_slot, k, M, E, N, K, stream);
}

int mps_experts_mm_dx(const void *d_dY, const void *d_W, void *d_dX, int dtype, const int *d_expert_ptr, int M, int E,
                      int N, int K, void *stream)
{
    return experts_entry<kRows>(d_dY, d_W, d_dX, dtype, d_expert_ptr, nullptr, 1, M, E, N, K, stream);
}

int mps_experts_mm_dw(const void *d_dY, const void *d_X, void *d_dW, int dtype, const int *d_expert_ptr,
                      const int *d_slot, int k, int M, int E, int N, int K, void *stream)
{
    return experts_entry<kWeights>(d_dY, d_X, d_dW, dtype, d_expert_ptr, d_slot, k, M, E, N, K, stream);
}

}  // extern "C"
