// bnn_ops_int8.hip -- rows to 8-bit integers with a scale each, and the linear layer on 8-bit operands (dense or over row groups).
// One of the translation units of libbnn_chaos_hip.so (bnn_internal.h lists them); entry points declared in include/bnn_chaos_hip.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "bnn_abi_common.h"
#include "bnn_grouped_host.h"

using namespace bnn;

// q = 127 v / amax rounded half to even, exactly.  fp32 decides except next to the middle between two integers: there (about 1 value in 5000)
// the two sides 254 v and (2 floor + 1) amax are compared in fp64, where both products are exact.  |v| <= amax; amax in the normal range.
__device__ __forceinline__ int quantize_one(float v, float amax, float inv) {
    const float t = v * inv;
    float q = rintf(t);
    if (fabsf(t - q) > 0.4999f) {
        const float lo = floorf(t);
        const double a = 254.0 * (double)v, m = (2.0 * (double)lo + 1.0) * (double)amax;
        q = a > m ? lo + 1.0f : a < m ? lo : 2.0f * floorf((lo + 1.0f) * 0.5f);
    }
    return (int)q;
}

// One row per workgroup: largest magnitude, then the codes.  A row with NaN or +-inf gets scale NaN (its products are NaN) and codes 0.
template <typename T>
__global__ __launch_bounds__(256) void bnn_quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int K, int8_t* __restrict__ q, int64_t ldq,
                                                                float* __restrict__ scale) {
    __shared__ float part[4];
    const T* row = x + (int64_t)blockIdx.x * ldx;
    int8_t* out = q + (int64_t)blockIdx.x * ldq;
    float amax = 0.0f;
    bool bad = false;
    for (int k = threadIdx.x; k < K; k += 256) {
        const float v = (float)row[k];
        bad |= !(fabsf(v) < INFINITY);
        amax = fmaxf(amax, fabsf(v));
    }
    if (bad) amax = INFINITY;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
    __syncthreads();
    amax = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const bool none = amax == 0.0f || amax == INFINITY;
    const float up = amax < 0x1p-100f ? 0x1p100f : 1.0f;   // (exact: 127 / amax must not overflow)
    const float am = amax * up, inv = none ? 0.0f : 127.0f / am;
    for (int k = threadIdx.x; k < ldq; k += 256) out[k] = k < K && !none ? (int8_t)quantize_one((float)row[k] * up, am, inv) : (int8_t)0;
    if (threadIdx.x == 0) scale[blockIdx.x] = amax == INFINITY ? NAN : amax / 127.0f;
}

extern "C" {

int bnn_quantize_rows(const void* x, int32_t dtype, int64_t rows, int32_t K, int64_t x_row, int8_t* q, int64_t q_row, float* scale, void* stream) {
    if (rows < 0 || K < 1 || dtype < BNN_TYPE_F32 || dtype > BNN_TYPE_F16 || q_row < K) return fail(BNN_ERR_INVALID, "bad argument");
    if (rows == 0) return 0;
    if (!x || !q || !scale) return fail(BNN_ERR_INVALID, "NULL argument");
    if (rows > 0x7fffffffLL || K > (1 << 24)) return fail(BNN_ERR_RANGE, "rows must stay below 2^31, their length below 2^24");
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == BNN_TYPE_F32) hipLaunchKernelGGL(bnn_quantize_rows_kernel<float>, dim3((unsigned)rows), dim3(256), 0, st, (const float*)x, x_row, K, q, q_row, scale);
    else if (dtype == BNN_TYPE_BF16) hipLaunchKernelGGL(bnn_quantize_rows_kernel<__bf16>, dim3((unsigned)rows), dim3(256), 0, st, (const __bf16*)x, x_row, K, q, q_row, scale);
    else hipLaunchKernelGGL(bnn_quantize_rows_kernel<_Float16>, dim3((unsigned)rows), dim3(256), 0, st, (const _Float16*)x, x_row, K, q, q_row, scale);
    HIP_TRY(hipGetLastError());
    return 0;
}

int bnn_int8_linear(const bnn_grouped* q, const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale, const void* bias, void* y,
                    void* stream) {
    if (!q) return fail(BNN_ERR_INVALID, "grouped descriptor is NULL");
    if (q->dtype < BNN_TYPE_F32 || q->dtype > BNN_TYPE_F16) return fail(BNN_ERR_INVALID, "dtype must be one of bnn_dtype");
    if (q->rows < 0 || q->copies < 1 || q->members < 1 || q->inputs < 1 || q->outputs < 1) return fail(BNN_ERR_INVALID, "bad rows / copies / members / inputs / outputs");
    if (q->rows > 0x7fffffffLL / q->copies) return fail(BNN_ERR_RANGE, "rows x copies must stay below 2^31");
    if (q->outputs > (1 << 24) || q->members > (1 << 24)) return fail(BNN_ERR_RANGE, "members and outputs must stay below 2^24");
    if (q->inputs > 131072) return fail(BNN_ERR_RANGE, "the 32-bit sums hold up to 131072 products of 8-bit integers");   // 2^17 * 127^2 < 2^31
    if (q->rows == 0) return 0;
    if (!x || !x_scale || !w || !w_scale || !y) return fail(BNN_ERR_INVALID, "NULL argument");
    if ((q->gather || q->scatter) && !q->order) return fail(BNN_ERR_INVALID, "gather / scatter need order");
    if (!q->offsets && (q->members != 1 || q->copies != 1 || q->gather || q->scatter)) return fail(BNN_ERR_INVALID, "without offsets there is one member and no order");
    const int os = type_size(q->dtype);
    RowsParams p{};
    p.x = (const char*)x; p.w = (const char*)w; p.bias = bias; p.y = (char*)y; p.xs = x_scale; p.ws = w_scale;
    p.order = q->order; p.offsets = q->offsets;
    p.ldx = q->x_row; p.w_member = q->w_member; p.w_row = q->w_row; p.ldy = q->y_row * os;
    p.P = (int32_t)(q->rows * q->copies); p.G = q->members; p.N = q->outputs; p.K = q->inputs;
    p.gather_div = q->gather ? q->copies : 0; p.scatter = q->scatter ? 1 : 0; p.relu = q->relu ? 1 : 0;
    if (q->dtype == BNN_TYPE_F32) return launch_rows_typed<int8_t, float, false>(p, (hipStream_t)stream);
    if (q->dtype == BNN_TYPE_BF16) return launch_rows_typed<int8_t, __bf16, false>(p, (hipStream_t)stream);
    return launch_rows_typed<int8_t, _Float16, false>(p, (hipStream_t)stream);
}

}  // extern "C"
