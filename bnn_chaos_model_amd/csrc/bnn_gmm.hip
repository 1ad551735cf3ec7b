// bnn_gmm.hip -- the grouped layer's product kernels (bnn_grouped.hip.h) for the float types: forward, dX and dW.
#include "bnn_grouped_host.h"

namespace bnn {

// call(operand type, output type, backwards) for a layer's types
template <class F>
static auto with_types(int dtype, int out, bool wfc, F call) {
    const bool f32 = out == BNN_TYPE_F32;
    using Fw = std::false_type;
    using Bw = std::true_type;
    if (dtype == BNN_TYPE_F32) return wfc ? call(Tag<float>{}, Tag<float>{}, Bw{}) : call(Tag<float>{}, Tag<float>{}, Fw{});
    if (dtype == BNN_TYPE_BF16) {
        if (!wfc) return call(Tag<__bf16>{}, Tag<__bf16>{}, Fw{});
        return f32 ? call(Tag<__bf16>{}, Tag<float>{}, Bw{}) : call(Tag<__bf16>{}, Tag<__bf16>{}, Bw{});
    }
    if (!wfc) return call(Tag<_Float16>{}, Tag<_Float16>{}, Fw{});
    return f32 ? call(Tag<_Float16>{}, Tag<float>{}, Bw{}) : call(Tag<_Float16>{}, Tag<_Float16>{}, Bw{});
}

int launch_rows(int dtype, int out, bool wfc, const RowsParams& p, hipStream_t st) {
    return with_types(dtype, out, wfc, [&](auto t, auto o, auto w) { return launch_rows_typed<typename decltype(t)::type, typename decltype(o)::type, decltype(w)::value>(p, st); });
}
RowsForm form_of_rows(int dtype, int out, bool wfc, RowsParams p) {
    return with_types(dtype, out, wfc, [&](auto t, auto o, auto w) {
        using O = typename decltype(o)::type;
        set_vec<O>(p);
        return rows_form<typename decltype(t)::type, O, decltype(w)::value>(p);
    });
}

int launch_reduce(int dtype, const ReduceParams& p, int tile, hipStream_t st) {
    if (dtype == BNN_TYPE_F32) return launch_reduce_typed<float>(p, tile, st);
    return dtype == BNN_TYPE_BF16 ? launch_reduce_typed<__bf16>(p, tile, st) : launch_reduce_typed<_Float16>(p, tile, st);
}
RowsForm form_of_reduce(int dtype, ReduceParams p, int tile) {
    const auto of = [&](auto tag) {
        using T = typename decltype(tag)::type;
        set_vec<T>(p);
        return reduce_form<T>(p, tile);
    };
    if (dtype == BNN_TYPE_F32) return of(Tag<float>{});
    return dtype == BNN_TYPE_BF16 ? of(Tag<__bf16>{}) : of(Tag<_Float16>{});
}

}  // namespace bnn
