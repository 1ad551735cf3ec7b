// bnn_gmm.hip -- the grouped layer's product kernels (bnn_grouped.hip.h) for the float types: forward, dX and dW.
#include "bnn_grouped_host.h"

namespace bnn {

int launch_rows(int dtype, int out, bool wfc, const RowsParams& p, hipStream_t st) {
    const bool f32 = out == BNN_TYPE_F32;
    if (dtype == BNN_TYPE_F32) return wfc ? launch_rows_typed<float, float, true>(p, st) : launch_rows_typed<float, float, false>(p, st);
    if (dtype == BNN_TYPE_BF16) {
        if (!wfc) return launch_rows_typed<__bf16, __bf16, false>(p, st);
        return f32 ? launch_rows_typed<__bf16, float, true>(p, st) : launch_rows_typed<__bf16, __bf16, true>(p, st);
    }
    if (!wfc) return launch_rows_typed<_Float16, _Float16, false>(p, st);
    return f32 ? launch_rows_typed<_Float16, float, true>(p, st) : launch_rows_typed<_Float16, _Float16, true>(p, st);
}

int launch_reduce(int dtype, const ReduceParams& p, int tile, hipStream_t st) {
    if (dtype == BNN_TYPE_F32) return launch_reduce_typed<float>(p, tile, st);
    return dtype == BNN_TYPE_BF16 ? launch_reduce_typed<__bf16>(p, tile, st) : launch_reduce_typed<_Float16>(p, tile, st);
}

}  // namespace bnn
