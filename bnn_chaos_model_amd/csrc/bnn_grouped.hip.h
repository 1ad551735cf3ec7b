// bnn_grouped.hip.h -- kernels of the grouped linear layer: the product of ragged row groups with their members' matrices (forward and dX), and
// the product over the rows of a group (dW, db).  Used by bnn_ops_grouped.hip (float types) and bnn_ops_int8.hip (8-bit operands).
#pragma once
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
    int32_t nblk, tiles_n, band;
};

struct ReduceParams {          // dW[g] = sum over rows r of member g of dy_r x_r^T;  db[g] = sum of dy_r
    const char* x;
    const char* dy;
    char* dw;                  // [G, N, K]
    void* db;                  // [G, N] or null
    float* part;               // [splits, G, N, K] then [splits, G, N] when splits > 1
    const int32_t* order;
    const int32_t* offsets;
    int64_t ldx, lddy;
    int32_t P, G, N, K;
    int32_t x_div, dy_div;     // as gather_div
    int32_t tiles_k, splits;
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
    __device__ __forceinline__ void issue(char* lds, int64_t k0, int64_t kbytes) {
        const int64_t at = k0 + c;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (DMA) load_to_lds(at < kbytes ? p[i] + at : (const char*)zero_chunk, lds + ((threadIdx.x & ~63) + i * NT) * CHUNK);
            else r[i] = load_chunk<T>(p[i], at, kbytes);
        }
    }
    __device__ __forceinline__ void commit(char* lds) {
        if constexpr (!DMA)
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4*>(lds + (threadIdx.x + i * NT) * CHUNK) = r[i];
    }
};

// FC operand: 128 / sizeof(T) rows of the reduction, W columns each, from column byte `col0` of rows of `width` bytes.
template <typename T, int W, int NT, bool DMA>
struct FcStage {
    static constexpr int CW = W * (int)sizeof(T) / CHUNK, N = W * 8 / NT, KR = stage_k<T>();
    static_assert(W * 8 % NT == 0 && NT % CW == 0, "whole chunks per thread");
    const char* base;
    const int32_t* order;   // row k of the reduction is row order[first + k] / div of the matrix (div == 0: row first + k)
    int64_t ld;
    int64_t width, col0;
    int first, limit, P, div;   // rows [first, limit); P = bound of order's values
    int nxt[N];
    u32x4 r[DMA ? 1 : N];
    __device__ __forceinline__ static int k_of(int i) { return (threadIdx.x + i * NT) / CW; }
    __device__ __forceinline__ int64_t col_of(int i) const { return col0 + (((int)threadIdx.x % CW) ^ fc_swz<T, W>(k_of(i))) * CHUNK; }
    __device__ __forceinline__ void fetch(int kt) {   // the rows' places for stage kt
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = first + kt * KR + k_of(i);
            int src = row < limit ? row : -1;
            if (div > 0 && src >= 0) {
                src = order[row];
                src = src >= 0 && src < P ? src : -1;
            }
            nxt[i] = src;
        }
    }
    __device__ __forceinline__ void issue(char* lds, int kt) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t at = col_of(i);
            const int src = div > 1 && nxt[i] >= 0 ? nxt[i] / div : nxt[i];
            const char* row = base + (int64_t)src * ld;
            if constexpr (DMA) load_to_lds(src < 0 ? (const char*)zero_chunk : row + (at < width ? at : 0), lds + ((threadIdx.x & ~63) + i * NT) * CHUNK);
            else {
                r[i] = u32x4{0, 0, 0, 0};
                if (src >= 0) r[i] = load_chunk<T>(row, at, width);
            }
        }
        fetch(kt + 1);
    }
    __device__ __forceinline__ void commit(char* lds) {
        if constexpr (!DMA)
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<u32x4*>(lds + (threadIdx.x + i * NT) * CHUNK) = r[i];
    }
};

template <bool DMA>
__device__ __forceinline__ void stage_barrier() {   // this wave's loads have landed in LDS, then everybody's
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
}

// ---- stores -------------------------------------------------------------------------------------------------------------------------------
template <typename O>
__device__ __forceinline__ void store4(char* row, int n, int N, const float v[4], bool vec) {
    O* d = reinterpret_cast<O*>(row) + n;
    if (vec && n + 4 <= N) {
        typedef O O4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<O4*>(d) = O4{(O)v[0], (O)v[1], (O)v[2], (O)v[3]};   // (one rounding, to nearest even, from the fp32 accumulator)
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < N) d[i] = (O)v[i];
    }
}

// ---- forward / dX --------------------------------------------------------------------------------------------------------------------------
// BM rows x BN outputs per workgroup, WM x WN waves.  WFC: the matrix is used the other way round (element (k, n) at k * w_row + n): dX.
template <typename T, typename O, int BM, int BN, int WM, int WN, bool WFC, bool DMA>
__global__ __launch_bounds__(WM * WN * 64) void bnn_grouped_kernel(RowsParams p) {
    constexpr int NT = WM * WN * 64, FM = BM / WM / 16, FN = BN / WN / 16, BUF = (BM + BN) * STAGE_BYTES;
    using M = Mma<T>;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    int tm, tn;
    tile_of_block(p.nblk, p.tiles_n, p.band, tm, tn);
    const RowTile rt = find_rows<BM>(p.offsets, p.G, p.P, tm);
    if (rt.g < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave / WN, wn = wave % WN;
    const int n0 = tn * BN;
    const bool vec = p.N % 4 == 0 && p.ldy % (4 * sizeof(O)) == 0 && ((uintptr_t)p.y % (4 * sizeof(O))) == 0;
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
            for (int j = 0; j < FN; ++j) store4<O>(row, n0 + wn * (BN / WN) + j * 16 + (lane >> 4) * 4, p.N, z, vec);
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
    KcStage<T, BN, NT, DMA> sb;
    FcStage<T, BN, NT, DMA> sf;
    if constexpr (WFC) {
        sf.base = wg; sf.order = nullptr; sf.ld = p.w_row; sf.width = (int64_t)p.N * sizeof(T); sf.col0 = (int64_t)n0 * sizeof(T);
        sf.first = 0; sf.limit = p.K; sf.P = p.K; sf.div = 0;
        sf.fetch(0);
    } else {
        sb.init();
#pragma unroll
        for (int i = 0; i < sb.N; ++i) sb.p[i] = wg + (int64_t)min(n0 + sb.row_of(i), p.N - 1) * p.w_row;
    }
    auto issue = [&](int kt) {
        char* buf = smem + (kt & 1) * BUF;
        sa.issue(buf, (int64_t)kt * STAGE_BYTES, kbytes);
        if constexpr (WFC) sf.issue(buf + BM * STAGE_BYTES, kt);
        else sb.issue(buf + BM * STAGE_BYTES, (int64_t)kt * STAGE_BYTES, kbytes);
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
    issue(0);
    commit(0);
    for (int kt = 0; kt < KT; ++kt) {
        stage_barrier<DMA>();
        if (kt + 1 < KT) issue(kt + 1);
        const char* a = smem + (kt & 1) * BUF;
        const char* b = a + BM * STAGE_BYTES;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            if (s == 1 && (int64_t)kt * STAGE_BYTES + 64 >= kbytes) break;   // nothing of the reduction in the second half
            u32x4 fa[FM], fb[FN];
#pragma unroll
            for (int f = 0; f < FM; ++f) fa[f] = frag_kc<T>(a, wm * (BM / WM) + f * 16, s, lane);
#pragma unroll
            for (int j = 0; j < FN; ++j) {
                if constexpr (WFC) fb[j] = frag_fc<T, BN>(b, wn * (BN / WN) + j * 16, s, lane);
                else fb[j] = frag_kc<T>(b, wn * (BN / WN) + j * 16, s, lane);
            }
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int f = 0; f < FM; ++f) acc[j][f] = M::mul(fb[j], fa[f], acc[j][f]);
        }
        if (kt + 1 < KT) commit(kt + 1);
    }
#pragma unroll
    for (int f = 0; f < FM; ++f) {
        const int m = rt.r0 + wm * (BM / WM) + f * 16 + (lane & 15);
        char* row = out_row(m);
        if (!row) continue;
        float xs = 1.0f;
        if constexpr (sizeof(T) == 1) {
            int64_t src = m;
            if (p.gather_div) {
                const int o = p.order[m];
                src = o >= 0 && o < p.P ? o / p.gather_div : 0;
            }
            xs = p.xs[src];
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int n = n0 + wn * (BN / WN) + j * 16 + (lane >> 4) * 4;
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t col = (int64_t)rt.g * p.N + min(n + i, p.N - 1);
                if constexpr (sizeof(T) == 1) v[i] = (float)acc[j][f][i] * (xs * p.ws[col]);
                else v[i] = acc[j][f][i];
                if (p.bias) v[i] += (float)reinterpret_cast<const O*>(p.bias)[col];
                if (p.relu) v[i] = v[i] < 0.0f ? 0.0f : v[i];   // (NaN stays NaN, as in nn.ReLU)
            }
            store4<O>(row, n, p.N, v, vec);
        }
    }
}

// ---- dW, db --------------------------------------------------------------------------------------------------------------------------------
// BN outputs x BK inputs of one member per workgroup (blockIdx.y), over split blockIdx.z of the member's rows.  The bias gradient is the same
// product with a column of ones and falls out of the workgroups of the first input tile.
template <typename T, typename O, int BN, int BK, int WN, int WK, bool DMA>
__global__ __launch_bounds__(WN * WK * 64) void bnn_grouped_dw_kernel(ReduceParams p) {
    constexpr int NT = WN * WK * 64, FN = BN / WN / 16, FK = BK / WK / 16, BUF = (BN + BK) * STAGE_BYTES, KR = stage_k<T>();
    using M = Mma<T>;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wn = wave / WK, wk = wave % WK;
    const int g = blockIdx.y, n0 = ((int)blockIdx.x / p.tiles_k) * BN, k0 = ((int)blockIdx.x % p.tiles_k) * BK;
    int r0 = min(max(p.offsets[g], 0), p.P), r1 = min(max(p.offsets[g + 1], r0), p.P);
    if (p.splits > 1) {   // whole stages per split
        const int64_t len = (((int64_t)(r1 - r0) + p.splits - 1) / p.splits + KR - 1) / KR * KR;
        const int64_t lo = r0 + len * blockIdx.z;
        r0 = (int)(lo < r1 ? lo : r1);
        r1 = (int)(lo + len < r1 ? lo + len : r1);
        r1 = max(r1, r0);
    }
    FcStage<T, BN, NT, DMA> sy;
    FcStage<T, BK, NT, DMA> sx;
    sy.base = p.dy; sy.order = p.order; sy.ld = p.lddy; sy.width = (int64_t)p.N * sizeof(T); sy.col0 = (int64_t)n0 * sizeof(T);
    sy.first = r0; sy.limit = r1; sy.P = p.P; sy.div = p.dy_div;
    sx.base = p.x; sx.order = p.order; sx.ld = p.ldx; sx.width = (int64_t)p.K * sizeof(T); sx.col0 = (int64_t)k0 * sizeof(T);
    sx.first = r0; sx.limit = r1; sx.P = p.P; sx.div = p.x_div;
    typename M::Acc acc[FK][FN], sum[FN];
#pragma unroll
    for (int f = 0; f < FN; ++f) {
        sum[f] = typename M::Acc{};
#pragma unroll
        for (int j = 0; j < FK; ++j) acc[j][f] = typename M::Acc{};
    }
    const bool bias = p.db && k0 == 0 && wk == 0;
    const int KT = (r1 - r0 + KR - 1) / KR;
    auto issue = [&](int kt) {
        char* buf = smem + (kt & 1) * BUF;
        sy.issue(buf, kt);
        sx.issue(buf + BN * STAGE_BYTES, kt);
    };
    auto commit = [&](int kt) {
        char* buf = smem + (kt & 1) * BUF;
        sy.commit(buf);
        sx.commit(buf + BN * STAGE_BYTES);
    };
    if (KT > 0) {
        sy.fetch(0);
        sx.fetch(0);
        issue(0);
        commit(0);
    }
    for (int kt = 0; kt < KT; ++kt) {
        stage_barrier<DMA>();
        if (kt + 1 < KT) issue(kt + 1);
        const char* a = smem + (kt & 1) * BUF;
        const char* b = a + BN * STAGE_BYTES;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 fa[FN], fb[FK];
#pragma unroll
            for (int f = 0; f < FN; ++f) fa[f] = frag_fc<T, BN>(a, wn * (BN / WN) + f * 16, s, lane);
#pragma unroll
            for (int j = 0; j < FK; ++j) fb[j] = frag_fc<T, BK>(b, wk * (BK / WK) + j * 16, s, lane);
#pragma unroll
            for (int j = 0; j < FK; ++j)
#pragma unroll
                for (int f = 0; f < FN; ++f) acc[j][f] = M::mul(fb[j], fa[f], acc[j][f]);
            if (bias)
#pragma unroll
                for (int f = 0; f < FN; ++f) sum[f] = M::mul(M::ones(), fa[f], sum[f]);
        }
        if (kt + 1 < KT) commit(kt + 1);
    }
    const bool whole = p.splits == 1;
    const int64_t nk = (int64_t)p.N * p.K, gnk = p.G * nk;
    char* dst = whole ? p.dw + g * nk * (int64_t)sizeof(O) : reinterpret_cast<char*>(p.part + blockIdx.z * gnk + g * nk);
    const bool vec = p.K % 4 == 0 && ((uintptr_t)p.dw % (4 * sizeof(O))) == 0;   // (the workspace is 16-byte aligned: checked by the host)
#pragma unroll
    for (int f = 0; f < FN; ++f) {
        const int n = n0 + wn * (BN / WN) + f * 16 + (lane & 15);
        if (n >= p.N) continue;
#pragma unroll
        for (int j = 0; j < FK; ++j) {
            const int k = k0 + wk * (BK / WK) + j * 16 + (lane >> 4) * 4;
            const float v[4] = {acc[j][f][0], acc[j][f][1], acc[j][f][2], acc[j][f][3]};
            if (whole) store4<O>(dst + (int64_t)n * p.K * sizeof(O), k, p.K, v, vec);
            else store4<float>(dst + (int64_t)n * p.K * sizeof(float), k, p.K, v, p.K % 4 == 0);
        }
        if (bias && lane < 16) {   // (the product with ones has the same sum in every first index)
            const float v = sum[f][0];
            if (whole) reinterpret_cast<O*>(p.db)[(int64_t)g * p.N + n] = (O)v;
            else p.part[p.splits * gnk + ((int64_t)blockIdx.z * p.G + g) * p.N + n] = v;
        }
    }
}

}  // namespace bnn
