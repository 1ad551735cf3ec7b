// bnn_grouped.hip.h -- kernels of the grouped linear layer: the product of ragged row groups with their members' matrices (forward and dX), and
// the product over the rows of a group (dW, db).  Used by bnn_ops_grouped.hip (float types) and bnn_ops_int8.hip (8-bit operands).
#pragma once
#include <type_traits>

#include "bnn_tile.hip.h"

namespace bnn {

struct RowsParams {            // y_r = act(W[g] x_r + b[g]) over the rows of every member g
    const char* x;             // rows; ldx bytes apart
    const char* w;             // element (g, i, j) at g * w_member + i * w_row (bytes) + j
    const void* bias;          // [G, N] in the output's type, or null
    char* y;                   // [.., N] rows of ldy bytes
    const int32_t* order;      // grouped row -> (row, copy) pair; null: the same
    const int32_t* offsets;    // [G + 1]; null: one member holds all rows
    const float* xs;           // 8-bit operands: scale per row of x, and per (member, output)
    const float* ws;
    int64_t ldx, w_member, w_row, ldy;
    int32_t P, G, N, K;        // grouped rows, members, output width, length of the reduction
    int32_t gather_div;        // 0: x is in grouped order; c >= 1: grouped row r reads row order[r] / c of x
    int32_t scatter;           // 1: grouped row r goes to row order[r] of y
    int32_t relu;
    int32_t nblk, tiles_n, band, block_rows;
    int32_t vec;               // N % 4 == 0 and rows of y aligned to four elements
};

struct ReduceParams {          // dW[g] = sum over rows r of member g of dy_r x_r^T;  db[g] = sum of dy_r
    const char* x;
    const char* dy;
    char* dw;                  // [G, N, K]
    void* db;                  // [G, N] or null
    float* part;               // [splits, G, N, K] then [splits, G, N] when splits > 1
    const int32_t* offsets;
    const int32_t* list;       // order, if either operand is gathered
    uint32_t ldx, lddy;
    int32_t P, G, N, K;
    int32_t m_x, m_dy;             // -1: row r of the grouped order is row order[r] / copies of x, row order[r] of dy; 0: row r
    uint32_t magic, shift;         // of the division by copies
    int32_t tiles_n, tiles_k, splits;
    int32_t by_size;               // 1: the members' tiles start in the order of their rows (at most 64 members)
    int32_t vec;                   // K % 4 == 0 and dw aligned to four elements
    __device__ __forceinline__ unsigned by_copies(int pair) const { return __umulhi(2u * (unsigned)pair, magic) >> shift; }
};

// ---- staging ------------------------------------------------------------------------------------------------------------------------------
// KC operand: W rows of 128 bytes per stage.  DMA: chunk-aligned rows, straight into LDS; otherwise through registers with any alignment.
template <typename T, int W, int NT, bool DMA>
struct KcStage {
    static constexpr int N = W * 8 / NT;
    static_assert(W * 8 % NT == 0 && NT % 128 == 0, "whole chunks per thread, one chunk column per thread");
    const char* p[N];
    u32x4 r[DMA ? 1 : N];
    int c;   // this thread's chunk of a row, in bytes
    __device__ __forceinline__ static int row_of(int i) { return (threadIdx.x + i * NT) >> 3; }
    __device__ __forceinline__ void init() { c = ((threadIdx.x & 7) ^ kc_swz(threadIdx.x >> 3)) * CHUNK; }
    __device__ __forceinline__ void issue(char* lds, int64_t k0, int64_t kbytes, int i) {   // the i-th of its N loads
        const int64_t at = k0 + c;
        if constexpr (DMA) load_to_lds(at < kbytes ? p[i] + at : (const char*)zero_chunk, lds + (__builtin_amdgcn_readfirstlane(threadIdx.x & ~63) + i * NT) * CHUNK);
        else r[i] = load_chunk<T>(p[i], at, kbytes, k0 + STAGE_BYTES <= kbytes);
    }
    __device__ __forceinline__ void commit(char* lds) {
        if constexpr (!DMA)
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4*>(lds + (threadIdx.x + i * NT) * CHUNK) = r[i];
    }
};

// FC operand: 128 / sizeof(T) rows of the reduction per stage, W columns each, from column byte `col0` of rows of `width` bytes.  A thread's rows are
// NT / CW apart.
template <typename T, int W, int NT, bool DMA>
struct FcStage {
    static constexpr int CW = W * (int)sizeof(T) / CHUNK, N = W * 8 / NT, KR = stage_k<T>(), STEP = NT / CW;
    static_assert(W * 8 % NT == 0 && NT % CW == 0 && STEP % 8 == 0, "whole chunks per thread, at most two chunk columns per thread");
    int at[2];         // byte of this thread's chunk in a row (below 2^26): of its even and odd loads
    bool inside;       // all of the tile's columns are the matrix's
    u32x4 r[DMA ? 1 : N];
    __device__ __forceinline__ static int k_of(int i) { return threadIdx.x / CW + i * STEP; }
    __device__ __forceinline__ void init(int64_t col0, int64_t width) {
        inside = col0 + W * (int64_t)sizeof(T) <= width;
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            at[o] = (int)col0 + (((int)threadIdx.x % CW) ^ fc_swz<T, W>(k_of(o))) * CHUNK;
            if (DMA && at[o] >= width) at[o] = 0;   // (columns behind the matrix: any, they are not stored)
        }
    }
    __device__ __forceinline__ void issue(char* lds, const char* row, bool live, int64_t width, int i) {   // the i-th of its N loads
        const int a = at[STEP % 16 == 0 ? 0 : i & 1];
        if constexpr (DMA) {
            const char* src = row + a;
            load_to_lds(live ? src : (const char*)zero_chunk, lds + (__builtin_amdgcn_readfirstlane(threadIdx.x & ~63) + i * NT) * CHUNK);
        } else {
            if (width >= CHUNK) r[i] = load_chunk<T>(live ? row : (const char*)zero_chunk, live ? a : 0, live ? width : CHUNK, inside);
            else r[i] = live ? load_short<T>(row, a, width) : u32x4{0, 0, 0, 0};
        }
    }
    __device__ __forceinline__ void commit(char* lds) {
        if constexpr (!DMA)
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4*>(lds + (threadIdx.x + i * NT) * CHUNK) = r[i];
    }
};

// ---- the loop over the reduction ----------------------------------------------------------------------------------------------------------
// acc += first . second over KT stages of 128 bytes, two LDS buffers.  A stage is two 64-byte steps with a register set of fragments each; the
// fragments of a step are read while the products of the step before run, across the stage border too.  Two barriers cut a stage into three parts:
//   1  the second step's fragments are read under the first step's products;                       then nobody reads this stage's buffer any more
//   2  the loads of the stage after next start into it, under products;                            then the next stage has landed
//   3  the next stage's first fragments are read under the rest of the products
// so that a load has one and a third stages to arrive.  The compiler keeps the order of loads into LDS and reads from it, so the parts are written as
// they should issue, the products spread between.
//   issue(kt, i)  load i of LOADS of stage kt; before(kt) comes ahead of the first; commit(kt) stores what loads through registers brought
//   read(kt, s, i, first, second)  fragment i of F1 + F2 of step s, READS LDS reads in all
// (stages behind the last are issued too: they read zeros into buffers that nobody reads)
constexpr int wait_loads(int n) { return (n & 15) | 0x0f70 | (n >> 4) << 14; }   // s_waitcnt vmcnt(n)
constexpr int WAIT_LDS = 0xc07f;                                                 // s_waitcnt lgkmcnt(0)

__device__ __forceinline__ void workgroup_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename T, int F1, int F2, int READS, int LOADS, bool DMA, class Before, class Issue, class Commit, class Read>
__device__ __forceinline__ void tile_loop(int KT, typename Mma<T>::Acc (&acc)[F1][F2], Before before, Issue issue, Commit commit, Read read) {
    constexpr int FR = F1 + F2, PR = F1 * F2, C1 = (PR + 1) / 2, C2 = PR / 4, MF = sizeof(T) == 4 ? 4 : 1, FLY = DMA ? LOADS : 63;
    u32x4 a0[F1], b0[F2], a1[F1], b1[F2];
    const auto products = [&](u32x4 (&a)[F1], u32x4 (&b)[F2], int lo, int hi) {
#pragma unroll
        for (int j = 0; j < F1; ++j)
#pragma unroll
            for (int f = 0; f < F2; ++f)
                if (j * F2 + f >= lo && j * F2 + f < hi) acc[j][f] = Mma<T>::mul(a[j], b[f], acc[j][f]);
    };
    before(0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) issue(0, i);
    commit(0);
    before(1);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) issue(1, i);
    __builtin_amdgcn_s_waitcnt(wait_loads(FLY));
    __builtin_amdgcn_s_waitcnt(WAIT_LDS);
    workgroup_barrier();
#pragma unroll
    for (int i = 0; i < FR; ++i) read(0, 0, i, a0, b0);
    for (int kt = 0; kt + 1 < KT; ++kt) {
        __builtin_amdgcn_s_waitcnt(WAIT_LDS);   // the fragments read in part 3, before more reads are in flight
#pragma unroll
        for (int i = 0; i < FR; ++i) read(kt, 1, i, a1, b1);
        products(a0, b0, 0, C1);
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        commit(kt + 1);
        __builtin_amdgcn_s_waitcnt(WAIT_LDS);
        workgroup_barrier();
        __builtin_amdgcn_sched_barrier(0);
        before(kt + 2);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) issue(kt + 2, i);
        products(a0, b0, C1, PR);
        products(a1, b1, 0, C2);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, (PR - C1 + C2) * MF / LOADS > 0 ? (PR - C1 + C2) * MF / LOADS : 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(wait_loads(FLY));   // all but the loads just issued (what came before them, too)
        workgroup_barrier();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FR; ++i) read(kt + 1, 0, i, a0, b0);
        products(a1, b1, C2, PR);
#pragma unroll
        for (int i = 0; i < READS; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < FR; ++i) read(KT - 1, 1, i, a1, b1);
    products(a0, b0, 0, PR);
    products(a1, b1, 0, PR);
    __builtin_amdgcn_s_waitcnt(0);   // (nothing is on its way into LDS when the wave ends)
}

// ---- stores -------------------------------------------------------------------------------------------------------------------------------
// four neighbours of a row of N, one rounding each, to nearest even, from the fp32 sums.  vec: N % 4 == 0 and rows aligned to four elements.
template <typename O>
__device__ __forceinline__ void store4(char* row, int n, int N, const float v[4], bool vec) {
    O* d = reinterpret_cast<O*>(row) + n;
    typedef O O4 __attribute__((ext_vector_type(4)));
    const O4 o = {(O)v[0], (O)v[1], (O)v[2], (O)v[3]};
    if (vec) {
        if (n < N) *reinterpret_cast<O4*>(d) = o;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < N) d[i] = o[i];
    }
}

// ---- forward / dX --------------------------------------------------------------------------------------------------------------------------
// Y = X W^T (or dX = dY W) of a member's rows.  Bound by the matrix pipe from a few hundred rows a member on: a 256 x 256 tile does 64 products per byte it
// loads in 16 bits.  Measured, launches back to back: 65 536 pairs x 4 096 -> 4 096 bf16 in 1.84 ms (1.20 PFLOP/s; matrix pipe 62-66 % busy), 16 384 x 4 096 -> 8 192
// in 8 bits 0.47 ms (2.3 POP/s).  The first 20 or so launches after a pause take up to a quarter longer, until the clock has settled.
// BM rows x BN outputs per workgroup, WM x WN waves.  WFC: the matrix is used the other way round (element (k, n) at k * w_row + n): dX.
template <typename T, typename O, int BM, int BN, int WM, int WN, bool WFC, bool DMA>
__device__ __forceinline__ void grouped_tile(const RowsParams& p, const RowTile rt, const int tn, char* smem) {
    constexpr int NT = WM * WN * 64, FM = BM / WM / 16, FN = BN / WN / 16, BUF = (BM + BN) * STAGE_BYTES;
    using M = Mma<T>;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
    const int n0 = tn * BN;
    auto out_row = [&](int m) -> char* {
        if (m >= rt.r1) return nullptr;
        int64_t o = m;
        if (p.scatter) {
            o = p.order[m];
            if (o < 0 || o >= p.P) return nullptr;
        }
        return p.y + o * p.ldy;
    };
    if (rt.g == p.G && p.offsets) {   // rows of nobody: zero
        const float z[4] = {0, 0, 0, 0};
        for (int f = 0; f < FM; ++f) {
            char* row = out_row(rt.r0 + wm * (BM / WM) + f * 16 + (lane & 15));
            if (!row) continue;
            for (int j = 0; j < FN; ++j) store4<O>(row, n0 + wn * (BN / WN) + j * 16 + (lane >> 4) * 4, p.N, z, DMA || p.vec);
        }
        return;
    }
    const int64_t kbytes = (int64_t)p.K * sizeof(T);
    KcStage<T, BM, NT, DMA> sa;
    sa.init();
#pragma unroll
    for (int i = 0; i < sa.N; ++i) {
        const int m = min(rt.r0 + sa.row_of(i), rt.r1 - 1);   // (rows behind the tile's end read its last row; they are not stored)
        int64_t src = m;
        if (p.gather_div) {
            const int o = p.order[m];
            src = o >= 0 && o < p.P ? (p.gather_div > 1 ? o / p.gather_div : o) : 0;
        }
        sa.p[i] = p.x + src * p.ldx;
    }
    const char* wg = p.w + rt.g * p.w_member;
    const char* wl = wg + (int64_t)FcStage<T, BN, NT, DMA>::k_of(0) * p.w_row;
    KcStage<T, BN, NT, DMA> sb;
    FcStage<T, BN, NT, DMA> sf;
    if constexpr (WFC) {
        sf.init((int64_t)n0 * sizeof(T), (int64_t)p.N * sizeof(T));
    } else {
        sb.init();
#pragma unroll
        for (int i = 0; i < sb.N; ++i) sb.p[i] = wg + (int64_t)min(n0 + sb.row_of(i), p.N - 1) * p.w_row;
    }
    auto issue = [&](int kt, int i) {
        char* buf = smem + (kt & 1) * BUF;
        if (i < sa.N) sa.issue(buf, (int64_t)kt * STAGE_BYTES, kbytes, i);
        else if constexpr (WFC) {
            const int k = kt * stage_k<T>() + (i - sa.N) * sf.STEP;   // of the wave's first rows
            sf.issue(buf + BM * STAGE_BYTES, wl + (int64_t)k * p.w_row, k + sf.k_of(0) < p.K, (int64_t)p.N * sizeof(T), i - sa.N);
        }
        else sb.issue(buf + BM * STAGE_BYTES, (int64_t)kt * STAGE_BYTES, kbytes, i - sa.N);
    };
    auto commit = [&](int kt) {
        char* buf = smem + (kt & 1) * BUF;
        sa.commit(buf);
        if constexpr (WFC) sf.commit(buf + BM * STAGE_BYTES);
        else sb.commit(buf + BM * STAGE_BYTES);
    };
    typename M::Acc acc[FN][FM];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int f = 0; f < FM; ++f) acc[j][f] = typename M::Acc{};
    const int KT = (int)((kbytes + STAGE_BYTES - 1) / STAGE_BYTES);
    tile_loop<T, FN, FM, FM + FN * (WFC ? (sizeof(T) == 4 ? 4 : 2) : 1), (BM + BN) * 8 / NT, DMA>(KT, acc, [](int) {}, issue, commit,
        [&](int kt, int st, int i, u32x4 (&fb)[FN], u32x4 (&fa)[FM]) {
        const char* a = smem + (kt & 1) * BUF;
        const char* b = a + BM * STAGE_BYTES;
        if (i < FM) fa[i] = frag_kc<T>(a, wm * (BM / WM) + i * 16, st, lane);
        else if constexpr (WFC) fb[i - FM] = frag_fc<T, BN>(b, wn * (BN / WN) + (i - FM) * 16, st, lane);
        else fb[i - FM] = frag_kc<T>(b, wn * (BN / WN) + (i - FM) * 16, st, lane);
    });
    tf32x4 bias[FN];   // of this lane's four outputs per fragment (outputs behind N: not stored)
    Scale ws[FN][4];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t col = (int64_t)rt.g * p.N + min(n0 + wn * (BN / WN) + j * 16 + (lane >> 4) * 4 + i, p.N - 1);
            bias[j][i] = 0.0f;
            if constexpr (sizeof(T) == 1) ws[j][i] = Scale(p.ws[col]);
        }
    if (p.bias)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                bias[j][i] = (float)reinterpret_cast<const O*>(p.bias)[(int64_t)rt.g * p.N + min(n0 + wn * (BN / WN) + j * 16 + (lane >> 4) * 4 + i, p.N - 1)];
#pragma unroll
    for (int f = 0; f < FM; ++f) {
        const int m = rt.r0 + wm * (BM / WM) + f * 16 + (lane & 15);
        char* row = out_row(m);
        if (!row) continue;
        Scale xs;
        if constexpr (sizeof(T) == 1) {
            int64_t src = m;
            if (p.gather_div) {
                const int o = p.order[m];
                src = o >= 0 && o < p.P ? o / p.gather_div : 0;
            }
            xs = Scale(p.xs[src]);
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = value_of(acc[j][f][i], xs, ws[j][i]) + bias[j][i];
                if (p.relu) v[i] = v[i] < 0.0f ? 0.0f : v[i];   // (NaN stays NaN, as in nn.ReLU)
            }
            store4<O>(row, n0 + wn * (BN / WN) + j * 16 + (lane >> 4) * 4, p.N, v, DMA || p.vec);
        }
    }
}

template <typename T, typename O, int BM, int BN, int WM, int WN, bool WFC, bool DMA>
__global__ __launch_bounds__(WM * WN * 64, WM * WN * 64 >= 512 ? 2 : 1) void bnn_grouped_kernel(RowsParams p) {
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    int tm, tn;
    tile_of_block(p.nblk, p.tiles_n, p.band, tm, tn);
    const RowTile rt = find_rows(p.offsets, p.G, p.P, tm, BM);
    if (rt.g < 0) return;
    // a member's last tile: half the rows take half the products (16 members of about 2 048 rows: one tile in nine)
    if (BM == 256 && rt.r1 - rt.r0 <= BM / 2) grouped_tile<T, O, BM == 256 ? BM / 2 : BM, BN, WM, WN, WFC, DMA>(p, rt, tn, smem);
    else grouped_tile<T, O, BM, BN, WM, WN, WFC, DMA>(p, rt, tn, smem);
}

// ---- forward of few rows --------------------------------------------------------------------------------------------------------------------
// 16 FM rows x 16 FN outputs per workgroup of eight waves.  With few rows per member the matrices are what is read: nothing is shared through LDS,
// every wave takes an eighth of the reduction and loads fragments of W and x as they lie in memory (64 bytes of 16 rows per load, U steps in
// flight), and the eight partial sums meet in LDS, in the waves' order.  Bound by the latency of a wave's loads: 15 rows of 30 members, 40 -> 40 fp32, 5.4 us.
template <typename T, typename O, int FM, int FN, int U, bool VEC>
__global__ __launch_bounds__(512) void bnn_grouped_few_kernel(RowsParams p) {
    constexpr int WAVES = 8, BM = 16 * FM, BN = 16 * FN, STEP = 64;
    using M = Mma<T>;
    using Acc = typename M::Acc;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    Acc* part = reinterpret_cast<Acc*>(smem);   // [WAVES][FM * FN][64]
    int tm, tn;
    tile_of_block(p.nblk, p.tiles_n, p.band, tm, tn);
    const RowTile rt = find_rows(p.offsets, p.G, p.P, tm, BM);
    if (rt.g < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n0 = tn * BN, q16 = (lane >> 4) * CHUNK;
    const bool nobody = rt.g == p.G && p.offsets;
    Acc acc[FM][FN];
#pragma unroll
    for (int f = 0; f < FM; ++f)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[f][j] = Acc{};
    if (!nobody) {
        const int64_t kbytes = (int64_t)p.K * sizeof(T);
        const char *px[FM], *pw[FN];
#pragma unroll
        for (int f = 0; f < FM; ++f) {
            const int m = min(rt.r0 + f * 16 + (lane & 15), rt.r1 - 1);
            int64_t src = m;
            if (p.gather_div) {
                const int o = p.order[m];
                src = o >= 0 && o < p.P ? (p.gather_div > 1 ? o / p.gather_div : o) : 0;
            }
            px[f] = p.x + src * p.ldx;
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) pw[j] = p.w + rt.g * p.w_member + (int64_t)min(n0 + j * 16 + (lane & 15), p.N - 1) * p.w_row;
        const int steps = (int)((kbytes + STEP - 1) / STEP), per = (steps + WAVES - 1) / WAVES, end = min(steps, (wave + 1) * per);
        const auto load = [&](const char* row, int step) -> u32x4 {   // past the wave's share or the row's end: zero
            const int64_t at = (int64_t)step * STEP + q16;
            if constexpr (VEC) return *reinterpret_cast<const u32x4*>(step < end && at < kbytes ? row + at : (const char*)zero_chunk);
            else if (kbytes >= CHUNK) return step < end ? load_chunk<T>(row, at, kbytes, ((int64_t)step + 1) * STEP <= kbytes) : u32x4{0, 0, 0, 0};
            else return load_short<T>(row, at, step < end ? kbytes : 0);
        };
        for (int s0 = wave * per; s0 < end; s0 += U) {
            u32x4 w[U][FN], x[U][FM];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < FN; ++j) w[u][j] = load(pw[j], s0 + u);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int f = 0; f < FM; ++f) x[u][f] = load(px[f], s0 + u);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int f = 0; f < FM; ++f)
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[f][j] = M::mul(w[u][j], x[u][f], acc[f][j]);
        }
    }
#pragma unroll
    for (int f = 0; f < FM; ++f)
#pragma unroll
        for (int j = 0; j < FN; ++j) part[(wave * FM * FN + f * FN + j) * 64 + lane] = acc[f][j];
    __syncthreads();
    for (int t = tid; t < FM * FN * 64; t += 512) {
        Acc a = part[t];
        for (int w = 1; w < WAVES; ++w) a = join(a, part[w * FM * FN * 64 + t]);
        const int frag = t >> 6, l = t & 63;
        const int m = rt.r0 + frag / FN * 16 + (l & 15), n = n0 + frag % FN * 16 + (l >> 4) * 4;
        if (m >= rt.r1) continue;
        int64_t o = m, src = m;
        if (p.order && (p.scatter || p.gather_div)) {
            const int pair = p.order[m];
            if (pair < 0 || pair >= p.P) continue;
            if (p.scatter) o = pair;
            if (p.gather_div) src = pair / p.gather_div;
        }
        float v[4] = {0, 0, 0, 0};
        if (!nobody) {
            float ws[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ws[i] = sizeof(T) == 1 ? p.ws[(int64_t)rt.g * p.N + min(n + i, p.N - 1)] : 1.0f;
            values_of(a, sizeof(T) == 1 ? p.xs[src] : 1.0f, ws, false, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (p.bias) v[i] += (float)reinterpret_cast<const O*>(p.bias)[(int64_t)rt.g * p.N + min(n + i, p.N - 1)];
                if (p.relu) v[i] = v[i] < 0.0f ? 0.0f : v[i];
            }
        }
        store4<O>(p.y + o * p.ldy, n, p.N, v, VEC || p.vec);
    }
}

// ---- forward of short rows --------------------------------------------------------------------------------------------------------------
// Rows of up to 64 ST bytes: the member's matrix stays in registers, FN x ST fragments a wave, while `block_rows` rows of the batch stream by,
// sixteen at a time -- no LDS, no barrier; what is read and written is the batch.  WN of the four waves share a row (each 16 FN outputs; its second
// to fourth reading comes from the first-level cache), so that a wave's part of the matrix is small and many waves fit.  The rows' places are
// fetched two steps ahead and the rows one step ahead of their products.  150 000 x 41 -> 128 fp32: 44 us (2.3 TB/s); its products alone would take 10-12,
// writing alone takes 14, so what is left is the latency of a row's way.
template <typename T, typename O, int FN, int ST, int WN>
__global__ __launch_bounds__(256) void bnn_grouped_short_kernel(RowsParams p) {
    constexpr int BN = 16 * FN * WN, STEP = 64, MSTEP = 16 * (4 / WN);
    using M = Mma<T>;
    using Acc = typename M::Acc;
    int tm, tn;
    tile_of_block(p.nblk, p.tiles_n, p.band, tm, tn);
    const RowTile rt = find_rows(p.offsets, p.G, p.P, tm, p.block_rows);
    if (rt.g < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n0 = tn * BN + wave % WN * 16 * FN, i16 = lane & 15, q = lane >> 4;
    if (n0 >= p.N) return;
    const bool nobody = rt.g == p.G && p.offsets;
    const int64_t kbytes = (int64_t)p.K * sizeof(T);
    const char* wg = p.w + (nobody ? 0 : rt.g) * p.w_member;
    const bool listed = p.gather_div || p.scatter;
    const auto place = [&](int m) -> int {   // the pair at grouped row m (m itself without an order)
        const int r = min(m, rt.r1 - 1);
        return listed ? p.order[r] : r;
    };
    int m = rt.r0 + wave / WN * 16 + i16;
    int pair = place(m), pair1 = place(m + MSTEP);   // (asked for ahead of the matrix: the rows wait for them)
    u32x4 w[FN][ST];
    float bias[FN][4], ws[FN][4];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            const int at = s * STEP + q * CHUNK, n = n0 + j * 16 + i16;
            w[j][s] = load_chunk<T>(wg + (int64_t)min(n, p.N - 1) * p.w_row, at, kbytes, (s + 1) * STEP <= kbytes);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t col = (int64_t)(nobody ? 0 : rt.g) * p.N + min(n0 + j * 16 + q * 4 + i, p.N - 1);
            bias[j][i] = p.bias && !nobody ? (float)reinterpret_cast<const O*>(p.bias)[col] : 0.0f;
            ws[j][i] = sizeof(T) == 1 ? p.ws[col] : 1.0f;
        }
    }
    const auto source = [&](int m, int pair) -> int64_t {   // row of x
        if (!p.gather_div) return min(m, rt.r1 - 1);
        const int o = pair >= 0 && pair < p.P ? pair : 0;
        return p.gather_div > 1 ? o / p.gather_div : o;
    };
    const auto fetch = [&](int64_t src, u32x4 (&x)[ST], float& xs) {
        const char* row = p.x + src * p.ldx;
        if constexpr (sizeof(T) == 1) xs = p.xs[src];   // (with the row: asked for in front of the output it is waited for there)
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            const int at = s * STEP + q * CHUNK;
            x[s] = load_chunk<T>(row, at, kbytes, (s + 1) * STEP <= kbytes);
        }
    };
    u32x4 x[ST];
    float xs = 1.0f;
    if (!nobody) fetch(source(m, pair), x, xs);
    for (; m - i16 < rt.r1; m += MSTEP) {
        u32x4 xn[ST];
        float xsn = 1.0f;
        const int64_t src1 = source(m + MSTEP, pair1);
        const int pair2 = place(m + 2 * MSTEP);
        if (!nobody) fetch(src1, xn, xsn);
        Acc acc[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[j] = Acc{};
        if (!nobody)
#pragma unroll
            for (int s = 0; s < ST; ++s)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[j] = M::mul(w[j][s], x[s], acc[j]);
        const int o = p.scatter ? pair : m;
        if (m < rt.r1 && o >= 0 && o < p.P) {
            char* row = p.y + (int64_t)o * p.ldy;
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                float v[4];
                values_of(acc[j], xs, ws[j], nobody, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] += bias[j][i];
                    if (p.relu) v[i] = v[i] < 0.0f ? 0.0f : v[i];
                }
                store4<O>(row, n0 + j * 16 + q * 4, p.N, v, p.vec);
            }
        }
        pair = pair1; pair1 = pair2; xs = xsn;
#pragma unroll
        for (int s = 0; s < ST; ++s) x[s] = xn[s];
    }
}

// the member with the r-th most rows, of up to 64
__device__ __forceinline__ int largest_member(const int32_t* __restrict__ off, int G, int P, int r) {
    const int lane = threadIdx.x & 63;
    int size = -1;
    if (lane < G) {
        const int s = min(max(off[lane], 0), P);
        size = min(max(off[lane + 1], s), P) - s;
    }
    int rank = 0;
    for (int j = 0; j < G; ++j) {
        const int other = __builtin_amdgcn_readlane(size, j);
        rank += other > size || (other == size && j < lane) ? 1 : 0;
    }
    return __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)__ballot(lane < G && rank == r)) - 1);
}

// ---- dW, db --------------------------------------------------------------------------------------------------------------------------------
// dW = dY^T X over a member's rows.  Bound by the matrix pipe where the member has a few hundred rows: 32 768 rows of 16 members, 2 048 x 2 048 bf16, 260 us
// with the bias (1.06 PFLOP/s).  Few tiles (30 000 rows of 30 members, 128 x 128 fp32: 120) would leave most CUs idle: their rows are split, 33 + 4 us.
// Every member's rows are cut into as many parts, so that the largest member is last where members are uneven.
// BT outputs x BT inputs of one member per workgroup, over split blockIdx.y of the member's rows; further workgroups sum dy's columns, the bias
// gradient.
// LISTED: rows of x or dy are found through the order (else both are in grouped order, and a load's row is the wave's plus a constant).
template <typename T, typename O, int BT, int WN, int WK, bool DMA, bool LISTED>
__global__ __launch_bounds__(WN * WK * 64, WN * WK * 64 >= 512 ? 2 : 1) void bnn_grouped_dw_kernel(ReduceParams p) {
    constexpr int NT = WN * WK * 64, FN = BT / WN / 16, FK = BT / WK / 16, BUF = 2 * BT * STAGE_BYTES, KR = stage_k<T>();
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wn = wave / WK, wk = wave % WK;
    // The workgroups that sum dy's columns come first.  Behind them the members' tiles, largest member first (a tile takes as long as its
    // member has rows; p.by_size), every member spread over all XCDs: XCD x takes the x-th eighth of its tiles, four output tiles side by side, which share their operands
    // in the XCD's L2.
    constexpr int BC = STAGE_BYTES / (int)sizeof(T);   // dy's columns per workgroup: 128 bytes of a row, for many rows in flight
    const int ncol = (p.N + BC - 1) / BC, nbias = p.db ? p.G * ncol : 0, first = (nbias + 7) / 8 * 8;
    const bool bias = (int)blockIdx.x < first;
    int g, tn, tk = 0;
    if (bias) {
        if ((int)blockIdx.x >= nbias) return;
        g = (int)blockIdx.x / ncol;
        tn = (int)blockIdx.x - g * ncol;
    } else {
        const int each = p.tiles_n * p.tiles_k, eighth = each < 8 ? 0 : (each + 7) / 8, slots = each < 8 ? each : 8 * eighth, b = (int)blockIdx.x - first;
        g = b / slots;
        const int j = b - g * slots, i = each < 8 ? j : (j + g) % 8 * eighth + j / 8;   // (the short last eighth goes round the XCDs)
        if (i >= each) return;
        const int band = i / (4 * p.tiles_k), at = i - band * 4 * p.tiles_k, rows = min(4, p.tiles_n - band * 4);
        tk = at / rows;
        tn = band * 4 + at - tk * rows;
        if (p.by_size) g = largest_member(p.offsets, p.G, p.P, g);
    }
    const int n0 = tn * (bias ? BC : BT), k0 = tk * BT;
    int r0 = min(max(p.offsets[g], 0), p.P), r1 = min(max(p.offsets[g + 1], r0), p.P);
    if (p.splits > 1) {   // whole stages per split
        const int64_t len = (((int64_t)(r1 - r0) + p.splits - 1) / p.splits + KR - 1) / KR * KR;
        const int64_t lo = r0 + len * blockIdx.y;
        r0 = (int)(lo < r1 ? lo : r1);
        r1 = (int)(lo + len < r1 ? lo + len : r1);
        r1 = max(r1, r0);
    }
    const bool whole = p.splits == 1;
    const int64_t nk = (int64_t)p.N * p.K, gnk = p.G * nk;
    if (bias) {   // a thread takes one chunk of every RL-th row, several at a time; the RL sums meet in LDS, in order
        constexpr int E = CHUNK / (int)sizeof(T), CW = BC / E, RL = NT / CW;
        float* part = reinterpret_cast<float*>(smem);   // [RL][BC]
        const int c = tid % CW, rl = tid / CW;
        const int64_t width = (int64_t)p.N * sizeof(T), byte = ((int64_t)n0 + c * E) * sizeof(T);
        const bool inside = (int64_t)(n0 + BC) * (int64_t)sizeof(T) <= width, tail = width >= CHUNK;
        float s[E];
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] = 0.0f;
        const auto add = [&](int r, auto count) {   // rows r, r + RL, ...
            constexpr int U = decltype(count)::value;
            int src[U];
            u32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int row = r + u * RL;
                src[u] = LISTED && p.m_dy ? p.list[min(row, r1 - 1)] : row;
                if (row >= r1 || src[u] >= p.P) src[u] = -1;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool live = src[u] >= 0;
                const char* row = live ? p.dy + (uint64_t)(unsigned)src[u] * p.lddy : (const char*)zero_chunk;
                if (tail) v[u] = load_chunk<T>(row, live ? byte : 0, live ? width : CHUNK, inside);
                else v[u] = load_short<T>(row, byte, live ? width : 0);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                T t[E];
                __builtin_memcpy(t, &v[u], CHUNK);
#pragma unroll
                for (int e = 0; e < E; ++e) s[e] += (float)t[e];
            }
        };
        int r = r0 + rl;
        for (; r + 8 * RL < r1; r += 16 * RL) add(r, std::integral_constant<int, 16>{});
        for (; r < r1; r += 4 * RL) add(r, std::integral_constant<int, 4>{});
#pragma unroll
        for (int e = 0; e < E; ++e) part[rl * BC + c * E + e] = s[e];
        __syncthreads();
        for (int i = tid; i < BC; i += NT) {
            const int n = n0 + i;
            float sum = part[i];
            for (int l = 1; l < RL; ++l) sum += part[l * BC + i];
            if (n < p.N) {
                if (whole) reinterpret_cast<O*>(p.db)[(int64_t)g * p.N + n] = (O)sum;
                else p.part[p.splits * gnk + ((int64_t)blockIdx.y * p.G + g) * p.N + n] = sum;
            }
        }
        return;
    }
    typename Mma<T>::Acc acc[FK][FN];
#pragma unroll
    for (int f = 0; f < FN; ++f)
#pragma unroll
        for (int j = 0; j < FK; ++j) acc[j][f] = typename Mma<T>::Acc{};
    const int KT = (r1 - r0 + KR - 1) / KR;
    if (KT > 0) {
        using S = FcStage<T, BT, NT, DMA>;
        S sy, sx;
        const int64_t wy = (int64_t)p.N * sizeof(T), wx = (int64_t)p.K * sizeof(T);
        sy.init((int64_t)n0 * sizeof(T), wy);
        sx.init((int64_t)k0 * sizeof(T), wx);
        int at[S::N], next[S::N];   // the pair at this thread's rows of the stage that is issued (negative: none), and what the list holds for the one behind it
        const auto row_of = [&](int kt, int i) { return r0 + kt * KR + S::k_of(i); };   // of the grouped order
        const auto pick = [](int mask, int a, int b) { return (a & mask) | (b & ~mask); };   // (masks, not conditions: the loop stays one block)
        const auto fetch = [&](int kt) {
#pragma unroll
            for (int i = 0; i < S::N; ++i) next[i] = p.list[min(row_of(kt, i), r1 - 1)];
        };
        const auto before = [&](int kt) {   // fetched a stage ahead; what is fetched now is older than the loads into LDS that follow
            if constexpr (!LISTED) return;
#pragma unroll
            for (int i = 0; i < S::N; ++i) {
                const int o = next[i];
                at[i] = row_of(kt, i) < r1 && o < p.P ? o : -1;
            }
            fetch(kt + 1);
        };
        const char* ly = p.dy + (uint64_t)(unsigned)(r0 + S::k_of(0)) * p.lddy;   // not LISTED: this thread's first rows
        const char* lx = p.x + (uint64_t)(unsigned)(r0 + S::k_of(0)) * p.ldx;
        if constexpr (!LISTED && DMA && S::STEP % 16 == 0) {   // ... and its chunk of them (fewer registers in the loop)
            ly += sy.at[0];
            lx += sx.at[0];
            sy.at[0] = sx.at[0] = 0;
        }
        const int below = r1 - r0 - S::k_of(0);
        const auto issue = [&](int kt, int i) {
            char* buf = smem + (kt & 1) * BUF;
            const int l = i % S::N;
            if constexpr (!LISTED) {
                const int k = kt * KR + l * S::STEP;
                const bool live = k < below;
                if (i < S::N) sy.issue(buf, ly + (uint64_t)(unsigned)k * p.lddy, live, wy, l);
                else sx.issue(buf + BT * STAGE_BYTES, lx + (uint64_t)(unsigned)k * p.ldx, live, wx, l);
                return;
            }
            const bool live = at[l] >= 0;
            if (i < S::N) sy.issue(buf, p.dy + (uint64_t)(unsigned)pick(p.m_dy, at[l], row_of(kt, l)) * p.lddy, live, wy, l);
            else sx.issue(buf + BT * STAGE_BYTES, p.x + (uint64_t)(unsigned)pick(p.m_x, p.by_copies(at[l]), row_of(kt, l)) * p.ldx, live, wx, l);
        };
        const auto commit = [&](int kt) {
            char* buf = smem + (kt & 1) * BUF;
            sy.commit(buf);
            sx.commit(buf + BT * STAGE_BYTES);
        };
        if constexpr (LISTED) fetch(0);
        tile_loop<T, FK, FN, (FK + FN) * (sizeof(T) == 4 ? 4 : 2), 2 * S::N, DMA>(KT, acc, before, issue, commit,
            [&](int kt, int st, int i, u32x4 (&fb)[FK], u32x4 (&fa)[FN]) {
                const char* a = smem + (kt & 1) * BUF;
                const char* b = a + BT * STAGE_BYTES;
                if (i < FN) fa[i] = frag_fc<T, BT>(a, wn * (BT / WN) + i * 16, st, lane);
                else fb[i - FN] = frag_fc<T, BT>(b, wk * (BT / WK) + (i - FN) * 16, st, lane);
            });
    }
    char* dst = whole ? p.dw + g * nk * (int64_t)sizeof(O) : reinterpret_cast<char*>(p.part + blockIdx.y * gnk + g * nk);
#pragma unroll
    for (int f = 0; f < FN; ++f) {
        const int n = n0 + wn * (BT / WN) + f * 16 + (lane & 15);
        if (n >= p.N) continue;
#pragma unroll
        for (int j = 0; j < FK; ++j) {
            const int k = k0 + wk * (BT / WK) + j * 16 + (lane >> 4) * 4;
            const float v[4] = {acc[j][f][0], acc[j][f][1], acc[j][f][2], acc[j][f][3]};
            if (whole) store4<O>(dst + (int64_t)n * p.K * sizeof(O), k, p.K, v, DMA || p.vec);
            else store4<float>(dst + (int64_t)n * p.K * sizeof(float), k, p.K, v, DMA || p.vec);
        }
    }
}

}  // namespace bnn
