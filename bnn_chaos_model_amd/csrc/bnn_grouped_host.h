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

// row tiles of BM that P grouped rows of G members (and nobody's) can need
inline int64_t row_tiles(const RowsParams& p, int BM) {
    return p.offsets ? p.P / BM + std::min<int64_t>((int64_t)p.G + 1, p.P) : ((int64_t)p.P + BM - 1) / BM;
}

template <typename T, typename O, int BM, int BN, int WM, int WN, bool WFC, bool DMA>
int launch_rows_tile(RowsParams p, hipStream_t st) {
    p.tiles_n = (p.N + BN - 1) / BN;
    const int64_t tm = row_tiles(p, BM), nblk = tm * p.tiles_n;
    if (nblk > 0x7fffffffLL) return fail(BNN_ERR_RANGE, "too many tiles for one launch");
    p.nblk = (int32_t)nblk;
    p.band = 8;
    constexpr auto* kern = &bnn_grouped_kernel<T, O, BM, BN, WM, WN, WFC, DMA>;
    allow_big_lds<kern>();
    hipLaunchKernelGGL(*kern, dim3((unsigned)nblk), dim3(WM * WN * 64), (size_t)2 * (BM + BN) * STAGE_BYTES, st, p);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <typename T, typename O, bool WFC>
int launch_rows_typed(const RowsParams& p, hipStream_t st) {
    return launch_rows_tile<T, O, 64, 64, 2, 2, WFC, false>(p, st);
}

int launch_rows(int dtype, int out, bool wfc, const RowsParams& p, hipStream_t st);

inline int reduce_splits(const bnn_grouped* q) { return 1; }

template <typename T, int BN, int BK, int WN, int WK, bool DMA>
int launch_reduce_tile(ReduceParams p, hipStream_t st) {
    p.tiles_k = (p.K + BK - 1) / BK;
    const int64_t tiles = (int64_t)((p.N + BN - 1) / BN) * p.tiles_k;
    if (tiles > 0x7fffffffLL || p.G > 65535) return fail(BNN_ERR_RANGE, "dW takes up to 65535 members");
    constexpr auto* kern = &bnn_grouped_dw_kernel<T, T, BN, BK, WN, WK, DMA>;
    allow_big_lds<kern>();
    hipLaunchKernelGGL(*kern, dim3((unsigned)tiles, (unsigned)p.G, (unsigned)p.splits), dim3(WN * WK * 64), (size_t)2 * (BN + BK) * STAGE_BYTES, st, p);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <typename T>
int launch_reduce_typed(const ReduceParams& p, hipStream_t st) {
    return launch_reduce_tile<T, 64, 64, 2, 2, false>(p, st);
}

int launch_reduce(int dtype, const ReduceParams& p, hipStream_t st);

}  // namespace bnn
