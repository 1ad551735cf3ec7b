// bnn_grouped_host.h -- choice of the tile and launch of the grouped layer's kernels (bnn_grouped.hip.h).
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "bnn_abi_common.h"
#include "bnn_grouped.hip.h"

namespace bnn {

template <typename T> struct Tag { using type = T; };

inline int type_size(int dtype) { return dtype == BNN_TYPE_F32 ? 4 : 2; }
inline bool aligned(int64_t v, int to) { return v % to == 0; }
inline bool aligned(const void* v, int to) { return (uintptr_t)v % to == 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// row tiles of BM that P grouped rows of G members (and nobody's) can need at most
inline int64_t row_tiles(const RowsParams& p, int BM) {
    return p.offsets ? p.P / BM + std::min<int64_t>((int64_t)p.G + 1, p.P) : ceil_div(p.P, BM);
}
// ... and about how many they will need: every member's last tile is half empty
inline int64_t likely_tiles(const RowsParams& p, int BM) {
    const int64_t used = std::min(p.G, p.P);
    return p.offsets ? std::max<int64_t>(used, p.P / BM + used / 2) : ceil_div(p.P, BM);
}

// a grid has fewer than 2^32 threads along x
inline int set_grid(RowsParams& p, int BM, int BN, int band, int threads) {
    p.tiles_n = (int32_t)ceil_div(p.N, BN);
    const int64_t nblk = row_tiles(p, BM) * p.tiles_n;
    if (nblk * threads > 0xffffffffLL) return fail(BNN_ERR_RANGE, "too many tiles for one launch");
    p.nblk = (int32_t)nblk;
    p.band = band;
    return 0;
}

template <typename T, typename O, int BM, int BN, int WM, int WN, bool WFC, bool DMA>
int launch_rows_tile(RowsParams p, hipStream_t st) {
    if (int rc = set_grid(p, BM, BN, 8, WM * WN * 64)) return rc;
    constexpr auto* kern = &bnn_grouped_kernel<T, O, BM, BN, WM, WN, WFC, DMA>;
    allow_big_lds<kern>();
    hipLaunchKernelGGL(*kern, dim3((unsigned)p.nblk), dim3(WM * WN * 64), (size_t)2 * (BM + BN) * STAGE_BYTES, st, p);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <typename T, typename O, int FM, int FN, int U, bool VEC>
int launch_rows_few(RowsParams p, hipStream_t st) {
    if (int rc = set_grid(p, 16 * FM, 16 * FN, 1, 512)) return rc;
    constexpr auto* kern = &bnn_grouped_few_kernel<T, O, FM, FN, U, VEC>;
    allow_big_lds<kern>();
    hipLaunchKernelGGL(*kern, dim3((unsigned)p.nblk), dim3(512), (size_t)8 * FM * FN * 64 * 16, st, p);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <typename T, typename O, int FN, int ST>
int launch_rows_short(RowsParams p, int rows, hipStream_t st) {
    constexpr int WN = 4;
    p.block_rows = rows;
    if (int rc = set_grid(p, rows, 16 * FN * WN, 1, 256)) return rc;
    hipLaunchKernelGGL((bnn_grouped_short_kernel<T, O, FN, ST, WN>), dim3((unsigned)p.nblk), dim3(256), 0, st, p);
    HIP_TRY(hipGetLastError());
    return 0;
}

// whole, aligned 16-byte chunks along every staged row (and four aligned outputs per store: p.vec)
template <typename T>
bool whole_chunks(const RowsParams& p, bool wfc) {
    return p.vec && aligned(p.x, CHUNK) && aligned(p.ldx, CHUNK) && aligned((int64_t)p.K * sizeof(T), CHUNK) && aligned(p.w, CHUNK) && aligned(p.w_member, CHUNK) &&
           aligned(p.w_row, CHUNK) && (!wfc || aligned((int64_t)p.N * sizeof(T), CHUNK));
}

// Which kernel.  The tiles' costs are rounds of the chip times the measured cost of a round, in units of a 256 x 256 tile (one workgroup per CU;
// two of 128 x 128, four of 64 x 64): the larger tile reads LDS and L2 less per product, the smaller ones leave fewer CUs and rows idle.
// (what is chosen, in numbers, is also what bnn_grouped_linear_form returns)
struct RowsForm {
    int32_t kind;            // bnn_grouped_kind
    int32_t rows, outputs;   // of a workgroup
    int32_t direct;          // 1: whole aligned chunks; 0: rows of any alignment
    int32_t steps;           // short rows: of 64 bytes
};
template <typename T, typename O, bool WFC>
RowsForm rows_form(const RowsParams& p) {
    const bool dma = whole_chunks<T>(p, WFC);
    const auto tiles = [&](int BM, int BN) { return likely_tiles(p, BM) * ceil_div(p.N, BN); };
    const int64_t steps = ceil_div((int64_t)p.K * sizeof(T), 64), used = std::min(p.G, p.P);
    if constexpr (!WFC) {
        // few rows a member and not enough 64 x 64 tiles to fill the chip: split the reduction over a workgroup's waves instead
        // (one row x 4 096 x 4 096 in 8 bits: 5.6 us against 13.2; 480 rows of 30 members, 480 tiles: 26 against 16)
        if (p.P <= 64 * used && tiles(64, 64) <= 320) {
            if (likely_tiles(p, 16) > used) return {BNN_GROUPED_FEW, 32, 32, dma};          // more than 16 rows a member
            return {BNN_GROUPED_FEW, 16, tiles(16, 16) <= 512 ? 16 : 32, dma};              // two workgroups per CU
        }
        // rows of up to 256 bytes that cannot be loaded straight into LDS (150 000 x 41 -> 128: 44 us against 61)
        if (!dma && steps <= 4 && p.P >= 64 * used) {
            const int outputs = p.N <= 64 ? 64 : 128;
            // 128 rows per workgroup where that still makes four workgroups per CU (150 000 rows x 41 -> 128: 44 us; 64 rows 47, 256 rows 51), else 64
            return {BNN_GROUPED_SHORT, tiles(128, outputs) >= 1024 ? 128 : 64, outputs, 0, (int32_t)steps};
        }
    }
    // (exact fp32 products: the matrix pipe is the bound in every tile, the small ones lose less)
    const double r128 = sizeof(T) == 4 ? 0.52 : 0.64, r64 = sizeof(T) == 4 ? 0.27 : 0.5;
    const double t256 = (double)ceil_div(tiles(256, 256), 256), t128 = ceil_div(tiles(128, 128), 512) * r128, t64 = ceil_div(tiles(64, 64), 1024) * r64;
    if (dma && t256 <= t128 && t256 <= t64) return {BNN_GROUPED_TILE, 256, 256, 1};
    // 16 384 x 4 095 -> 4 096 in 8 bits: 542 us against 842 in 128 x 128 tiles (bf16 loses with it: 32 768 x 4 095 -> 4 096 2 250 against 2 000)
    if (!dma && sizeof(T) == 1 && ceil_div(tiles(256, 128), 256) * 0.41 <= std::min(t128, t64)) return {BNN_GROUPED_TILE, 256, 128, 0};
    return t128 <= t64 ? RowsForm{BNN_GROUPED_TILE, 128, 128, dma} : RowsForm{BNN_GROUPED_TILE, 64, 64, dma};
}

// four aligned outputs per store
template <typename O>
void set_vec(RowsParams& p) { p.vec = p.N % 4 == 0 && aligned(p.ldy, 4 * sizeof(O)) && aligned(p.y, 4 * sizeof(O)); }

template <typename T, typename O, bool VEC>
int launch_few(const RowsParams& p, const RowsForm& f, hipStream_t st) {
    if (f.rows == 32) return launch_rows_few<T, O, 2, 2, 4, VEC>(p, st);
    return f.outputs == 16 ? launch_rows_few<T, O, 1, 1, 8, VEC>(p, st) : launch_rows_few<T, O, 1, 2, 4, VEC>(p, st);
}

template <typename T, typename O, int ST>
int launch_short(const RowsParams& p, const RowsForm& f, hipStream_t st) {
    return f.outputs == 64 ? launch_rows_short<T, O, 1, ST>(p, f.rows, st) : launch_rows_short<T, O, 2, ST>(p, f.rows, st);
}

template <typename T, typename O, bool WFC>
int launch_rows_typed(RowsParams p, hipStream_t st) {
    set_vec<O>(p);
    const RowsForm f = rows_form<T, O, WFC>(p);
    if constexpr (!WFC) {
        if (f.kind == BNN_GROUPED_FEW) return f.direct ? launch_few<T, O, true>(p, f, st) : launch_few<T, O, false>(p, f, st);
        if (f.kind == BNN_GROUPED_SHORT) {
            if (f.steps <= 1) return launch_short<T, O, 1>(p, f, st);
            if (f.steps == 2) return launch_short<T, O, 2>(p, f, st);
            return f.steps == 3 ? launch_short<T, O, 3>(p, f, st) : launch_short<T, O, 4>(p, f, st);
        }
    }
    if (f.direct) {
        if (f.rows == 256) return launch_rows_tile<T, O, 256, 256, 2, 4, WFC, true>(p, st);
        return f.rows == 128 ? launch_rows_tile<T, O, 128, 128, 2, 2, WFC, true>(p, st) : launch_rows_tile<T, O, 64, 64, 2, 2, WFC, true>(p, st);
    }
    if constexpr (sizeof(T) == 1)
        if (f.rows == 256) return launch_rows_tile<T, O, 256, 128, 4, 2, WFC, false>(p, st);
    return f.rows == 128 ? launch_rows_tile<T, O, 128, 128, 2, 2, WFC, false>(p, st) : launch_rows_tile<T, O, 64, 64, 2, 2, WFC, false>(p, st);
}

int launch_rows(int dtype, int out, bool wfc, const RowsParams& p, hipStream_t st);
RowsForm form_of_rows(int dtype, int out, bool wfc, RowsParams p);

// dW: the tile, and into how many parts the rows of a member are cut (by the sizes alone: the workspace is asked for before the pointers are known)
struct ReducePlan { int tile, splits; };
inline ReducePlan reduce_plan(int64_t P, int64_t G, int64_t N, int64_t K, bool f32) {
    const auto tiles = [&](int b) { return G * ceil_div(N, b) * ceil_div(K, b); };
    if (!f32 && tiles(256) >= 192) return {256, 1};
    if (tiles(128) >= 192) return {128, 1};
    // about two rounds of four workgroups per CU, at least 128 rows each
    return {64, (int)std::max<int64_t>(1, std::min<int64_t>({2048 / tiles(64), P / G / 128, 16}))};
}

template <typename T, int BT, int WN, int WK, bool DMA, bool LISTED>
int launch_reduce_form(ReduceParams p, hipStream_t st) {
    p.tiles_k = (int32_t)ceil_div(p.K, BT);
    p.tiles_n = (int32_t)ceil_div(p.N, BT);
    const int64_t nbias = p.db ? p.G * ceil_div((int64_t)p.N * sizeof(T), STAGE_BYTES) : 0;
    const int64_t each = (int64_t)p.tiles_n * p.tiles_k, nblk = ceil_div(nbias, 8) * 8 + p.G * (each < 8 ? each : ceil_div(each, 8) * 8);
    if (nblk >= (1LL << 32) / (WN * WK * 64)) return fail(BNN_ERR_RANGE, "too many tiles for one launch");
    // members of uneven size, 32 768 rows of 16, 2 048 x 2 048, with bias: 400 us in their own order, 310 largest first; short splits do not pay for the sort
    p.by_size = p.G <= 64 && p.splits == 1 && nblk > 256;
    constexpr auto* kern = &bnn_grouped_dw_kernel<T, T, BT, WN, WK, DMA, LISTED>;
    allow_big_lds<kern>();
    hipLaunchKernelGGL(*kern, dim3((unsigned)nblk, (unsigned)p.splits), dim3(WN * WK * 64), (size_t)4 * BT * STAGE_BYTES, st, p);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <typename T, int BT, int WN, int WK, bool DMA>
int launch_reduce_tile(const ReduceParams& p, hipStream_t st) {
    return p.list ? launch_reduce_form<T, BT, WN, WK, DMA, true>(p, st) : launch_reduce_form<T, BT, WN, WK, DMA, false>(p, st);
}

// tile: the plan's; rows that cannot be loaded straight into LDS have no tile of 256
template <typename T>
RowsForm reduce_form(const ReduceParams& p, int tile) {
    const bool dma = p.vec && aligned(p.x, CHUNK) && aligned(p.dy, CHUNK) && aligned(p.ldx, CHUNK) && aligned(p.lddy, CHUNK) && aligned((int64_t)p.K * sizeof(T), CHUNK) &&
                     aligned((int64_t)p.N * sizeof(T), CHUNK);
    const int32_t b = dma ? tile : std::min(tile, 128);
    return {p.list ? BNN_GROUPED_DW_LISTED : BNN_GROUPED_DW, b, b, dma};
}
template <typename T>
void set_vec(ReduceParams& p) { p.vec = p.K % 4 == 0 && aligned(p.dw, 4 * sizeof(T)); }

template <typename T>
int launch_reduce_typed(ReduceParams p, int tile, hipStream_t st) {
    set_vec<T>(p);
    const RowsForm f = reduce_form<T>(p, tile);
    if (f.direct) {
        if constexpr (sizeof(T) == 2)
            if (f.rows == 256) return launch_reduce_tile<T, 256, 2, 4, true>(p, st);
        return f.rows == 128 ? launch_reduce_tile<T, 128, 2, 4, true>(p, st) : launch_reduce_tile<T, 64, 2, 2, true>(p, st);
    }
    return f.rows == 128 ? launch_reduce_tile<T, 128, 2, 4, false>(p, st) : launch_reduce_tile<T, 64, 2, 2, false>(p, st);
}

int launch_reduce(int dtype, const ReduceParams& p, int tile, hipStream_t st);
RowsForm form_of_reduce(int dtype, ReduceParams p, int tile);

}  // namespace bnn
