// bnn_ops_int8.hip -- rows to 8-bit integers with a scale each, and the linear layer on 8-bit operands (dense or over row groups).
// One of the translation units of libbnn_chaos_hip.so (bnn_internal.h lists them); entry points declared in include/bnn_chaos_hip.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "bnn_abi_common.h"
#include "bnn_grouped_host.h"

using namespace bnn;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// A row's scaling: amax in the normal range and not so large that 255 amax overflows (a power of two takes values there, exactly where it matters).
struct Scaling {
    float up, amax, inv, scale;   // code = round(127 (v up) / amax);  scale = what a code of 1 stands for
    __device__ __forceinline__ explicit Scaling(uint32_t top) {   // bit pattern of the row's largest magnitude
        const float m = __uint_as_float(top);
        const bool bad = top >= 0x7f800000u;   // NaN or +-inf in the row: scale NaN, codes 0
        up = m < 0x1p-100f ? 0x1p100f : m > 0x1p100f ? 0x1p-100f : 1.0f;
        amax = m * up;
        inv = bad || top == 0 ? 0.0f : 127.0f / amax;
        scale = bad ? NAN : m / 127.0f;
    }
};

// The code of v next to the middle between lo and lo + 1, exactly: the sign of 254 v - (2 lo + 1) amax.  p is the second product rounded and e what
// the rounding left; 254 v - p is exact, the two agree in their leading bits.
__device__ __forceinline__ float quantize_middle(float v, float t, float amax) {
    const float lo = floorf(t), m = 2.0f * lo + 1.0f, p = m * amax, e = fmaf(m, amax, -p), d = fmaf(254.0f, v, -p);
    return d > e ? lo + 1.0f : d < e ? lo : 2.0f * floorf((lo + 1.0f) * 0.5f);
}

// E neighbours of a row -> their codes, four to a word: 127 v / amax rounded half to even, as the exact quotient rounds.  Adding 1.5 * 2^23 rounds
// |t| <= 127 to an integer and leaves it (modulo 256) in the sum's low byte; t is off by at most 2^-15, so only values within 1e-4 of a middle
// (1 in 5000) are looked at again.
template <typename T, int E>
__device__ __forceinline__ void quantize_chunk(u32x4 raw, const Scaling& sc, uint32_t (&word)[E / 4]) {
    constexpr float MAGIC = 12582912.0f;
    T t[E];
    __builtin_memcpy(t, &raw, CHUNK);
    uint32_t s[E];
    float off = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float v = (float)t[e] * sc.up * sc.inv, r = v + MAGIC;
        s[e] = __float_as_uint(r);
        off = fmaxf(off, fabsf(v - (r - MAGIC)));
    }
    if (off > 0.4999f)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = (float)t[e] * sc.up, x = v * sc.inv;
            if (fabsf(x - rintf(x)) > 0.4999f) s[e] = __float_as_uint(quantize_middle(v, x, sc.amax) + MAGIC);
        }
#pragma unroll
    for (int w = 0; w < E / 4; ++w)
        word[w] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(s[4 * w + 3], s[4 * w + 2], 0x0c0c0400), __builtin_amdgcn_perm(s[4 * w + 1], s[4 * w], 0x0c0c0400), 0x05040100);
}

template <int E> struct __attribute__((packed, aligned(1))) Codes { uint32_t w[E / 4]; };

// Largest magnitude of a row, then its codes.  TPR threads take a row, in chunks of 16 bytes; the first HELD chunks of a thread stay in registers
// between the two sweeps, longer rows are read again.  Rows are at least one chunk long.
// Bound by memory: 65 536 x 4 096 bf16 read once, 8-bit codes written once, 165 us (4.9 TB/s).
template <typename T, int TPR>
__global__ __launch_bounds__(256) void bnn_quantize_rows_kernel(const char* __restrict__ x, int64_t ldx, int64_t rows, int K, int8_t* __restrict__ q, int64_t ldq,
                                                                float* __restrict__ scale) {
    constexpr int E = CHUNK / (int)sizeof(T), HELD = 8;
    __shared__ uint32_t part[4];
    const int tid = threadIdx.x % TPR;
    const int64_t r = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    if (r >= rows) return;   // (whole groups of TPR threads; with 256 threads a row every workgroup has one)
    const char* row = x + r * ldx;
    const int64_t kbytes = (int64_t)K * sizeof(T);
    const int chunks = (K + E - 1) / E;
    const auto load = [&](int c) { return load_tail<T>(row, (int64_t)c * CHUNK, kbytes); };
    uint32_t top = 0;   // magnitudes compare like their bit patterns, and +-inf and NaN above them all
    const auto fold = [&](u32x4 raw) {
        if constexpr (sizeof(T) == 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, raw[e] & 0x7fffffffu);
        else   // the two halves of a word side by side
#pragma unroll
            for (int e = 0; e < 4; ++e)
                top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top), __builtin_bit_cast(u16x2, raw[e] & 0x7fff7fffu)));
    };
    u32x4 held[HELD];
#pragma unroll
    for (int h = 0; h < HELD; ++h)   // (uniform; a chunk twice does not change the largest)
        if (h * TPR < chunks) held[h] = load(min(h * TPR + tid, chunks - 1));
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (h * TPR < chunks) fold(held[h]);
    for (int c = HELD * TPR + tid; c < chunks; c += TPR) fold(load(c));
    if constexpr (sizeof(T) == 2) {   // as fp32 from here on
        T half;
        const uint16_t bits = (uint16_t)max(top & 0xffffu, top >> 16);
        __builtin_memcpy(&half, &bits, 2);
        top = __float_as_uint((float)half);
    }
#pragma unroll
    for (int d = TPR < 64 ? TPR / 2 : 32; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if constexpr (TPR == 256) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
        __syncthreads();
        top = max(max(part[0], part[1]), max(part[2], part[3]));
    }
    const Scaling sc(top);
    const bool none = sc.inv == 0.0f;
    int8_t* out = q + r * ldq;
    uint32_t last[E / 4] = {};   // codes of a chunk that does not fit the row of q
    bool partial = false;
    const auto store = [&](int c, u32x4 raw) {
        uint32_t word[E / 4];
        if (none) raw = u32x4{0, 0, 0, 0};
        quantize_chunk<T, E>(raw, sc, word);
        Codes<E> codes;
#pragma unroll
        for (int w = 0; w < E / 4; ++w) codes.w[w] = word[w];
        if ((int64_t)(c + 1) * E <= ldq) *reinterpret_cast<Codes<E>*>(out + (int64_t)c * E) = codes;   // (codes behind K are zero: so is what was loaded there)
        else {
            partial = true;
#pragma unroll
            for (int w = 0; w < E / 4; ++w) last[w] = word[w];
        }
    };
#pragma unroll
    for (int h = 0; h < HELD; ++h)
        if (h * TPR < chunks) {
            const int c = h * TPR + tid;
            asm volatile("" : "+v"(held[h]));   // (a chunk after the other: the compiler starts on all of them at once, in 230 registers and at half the speed)
            if (c < chunks) store(c, held[h]);
        }
    for (int c = HELD * TPR + tid; c < chunks; c += TPR) store(c, load(c));
    if (partial) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if ((int64_t)(chunks - 1) * E + e < ldq) out[(int64_t)(chunks - 1) * E + e] = (int8_t)(last[e >> 2] >> ((e & 3) * 8));
    }
    for (int64_t k = (int64_t)chunks * E + tid; k < ldq; k += TPR) out[k] = 0;
    if (tid == 0) scale[r] = sc.scale;
}

// rows shorter than a chunk: a thread a row
template <typename T>
__global__ __launch_bounds__(256) void bnn_quantize_short_rows_kernel(const char* __restrict__ x, int64_t ldx, int64_t rows, int K, int8_t* __restrict__ q, int64_t ldq,
                                                                      float* __restrict__ scale) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r >= rows) return;
    const T* row = reinterpret_cast<const T*>(x + r * ldx);
    uint32_t top = 0;
    for (int k = 0; k < K; ++k) top = max(top, __float_as_uint((float)row[k]) & 0x7fffffffu);
    const Scaling sc(top);
    for (int64_t k = 0; k < ldq; ++k) {
        float v = k < K && sc.inv != 0.0f ? (float)row[k] * sc.up : 0.0f;
        const float t = v * sc.inv, c = rintf(t);
        q[r * ldq + k] = (int8_t)(fabsf(t - c) > 0.4999f ? quantize_middle(v, t, sc.amax) : c);
    }
    scale[r] = sc.scale;
}

// The layer for a handful of rows in one launch: a workgroup of eight waves quantises the (up to 16) rows of its tile into LDS -- every workgroup
// again: that is a few kilobytes from L2 against a launch -- while its first fragments of the matrix are on their way, then goes on like
// bnn_grouped_few_kernel: an eighth of the reduction per wave, partial sums joined in LDS.  Bound by latency: one row of 4 096 -> 4 096, 8.2 us (its matrix
// alone: 3.5).
template <typename XT, typename O>
__global__ __launch_bounds__(512) void bnn_int8_handful_kernel(RowsParams p, int ldq) {
    constexpr int WAVES = 8, BM = 16, STEP = 64, U = 8, E = CHUNK / (int)sizeof(XT);
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    i32x4* part = reinterpret_cast<i32x4*>(smem);                            // [WAVES][64]
    float* sx = reinterpret_cast<float*>(smem + WAVES * 64 * 16);            // [BM] scales
    uint32_t* tops = reinterpret_cast<uint32_t*>(sx + BM);                   // [WAVES]
    char* codes = reinterpret_cast<char*>(tops + 16);                        // [rows of the tile][ldq]
    int tm, tn;
    tile_of_block(p.nblk, p.tiles_n, p.band, tm, tn);
    const RowTile rt = find_rows(p.offsets, p.G, p.P, tm, BM);
    if (rt.g < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n0 = tn * 16, i16 = lane & 15, q16 = (lane >> 4) * CHUNK;
    const bool nobody = rt.g == p.G && p.offsets;
    const int nrows = rt.r1 - rt.r0;
    i32x4 acc = {0, 0, 0, 0};
    if (!nobody) {
        const char* pw = p.w + rt.g * p.w_member + (int64_t)min(n0 + i16, p.N - 1) * p.w_row;
        const int steps = (p.K + STEP - 1) / STEP, per = (steps + WAVES - 1) / WAVES, end = min(steps, (wave + 1) * per);
        const auto load_w = [&](int step) -> u32x4 {
            const int64_t at = (int64_t)step * STEP + q16;
            if (p.K < CHUNK) return load_short<int8_t>(pw, at, step < end ? p.K : 0);
            const u32x4 v = load_tail<int8_t>(pw, at, p.K);
            return step < end ? v : u32x4{0, 0, 0, 0};
        };
        u32x4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) w[u] = load_w(wave * per + u);
        // threads of a row: all of them for one row, down to a wave a row
        const int waves = nrows == 1 ? WAVES : nrows == 2 ? 4 : nrows <= 4 ? 2 : 1, tpr = waves * 64;
        const int64_t kbytes = (int64_t)p.K * sizeof(XT);
        const int chunks = (p.K + E - 1) / E;
        for (int first = 0; first < nrows; first += WAVES / waves) {   // (one round up to eight rows, two up to sixteen)
            const int r = first + tid / tpr, t = tid % tpr;
            const char* row = nullptr;
            if (r < nrows) {
                int64_t src = rt.r0 + r;
                if (p.gather_div) {
                    const int o = p.order[src];
                    src = o >= 0 && o < p.P ? o / p.gather_div : 0;
                }
                row = p.x + src * p.ldx;
            }
            const auto load_x = [&](int c) { return kbytes >= CHUNK ? load_tail<XT>(row, (int64_t)c * CHUNK, kbytes) : load_short<XT>(row, (int64_t)c * CHUNK, kbytes); };
            uint32_t top = 0;
            u32x4 held = {0, 0, 0, 0};
            if (row)
                for (int c = t; c < chunks; c += tpr) {
                    const u32x4 raw = load_x(c);
                    if (c == t) held = raw;
                    XT v[E];
                    __builtin_memcpy(v, &raw, CHUNK);
#pragma unroll
                    for (int e = 0; e < E; ++e) top = max(top, __float_as_uint((float)v[e]) & 0x7fffffffu);
                }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
            if (lane == 0) tops[wave] = top;
            __syncthreads();
            for (int i = 0; i < waves; ++i) top = max(top, tops[wave / waves * waves + i]);
            __syncthreads();
            const Scaling sc(top);
            if (row) {
                for (int c = t; c * E < ldq; c += tpr) {   // (zero up to the stage's end)
                    uint32_t word[E / 4] = {};
                    if (c < chunks && sc.inv != 0.0f) quantize_chunk<XT, E>(c == t ? held : load_x(c), sc, word);
                    *reinterpret_cast<Codes<E>*>(codes + r * ldq + c * E) = *reinterpret_cast<Codes<E>*>(word);
                }
                if (t == 0) sx[r] = sc.scale;
            }
        }
        __syncthreads();
        const char* row = codes + min(i16, nrows - 1) * ldq;
        for (int s0 = wave * per; s0 < end; s0 += U) {
            if (s0 > wave * per)
#pragma unroll
                for (int u = 0; u < U; ++u) w[u] = load_w(s0 + u);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s0 + u < end) acc = Mma<int8_t>::mul(w[u], *reinterpret_cast<const u32x4*>(row + (s0 + u) * STEP + q16), acc);
        }
    }
    part[wave * 64 + lane] = acc;
    __syncthreads();
    if (tid >= 64) return;
    i32x4 a = part[lane];
    for (int w = 1; w < WAVES; ++w) a = join(a, part[w * 64 + lane]);
    const int m = rt.r0 + i16, n = n0 + (lane >> 4) * 4;
    if (m >= rt.r1) return;
    int64_t o = m;
    if (p.scatter) {
        o = p.order[m];
        if (o < 0 || o >= p.P) return;
    }
    float v[4] = {0, 0, 0, 0};
    if (!nobody) {
        float ws[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ws[i] = p.ws[(int64_t)rt.g * p.N + min(n + i, p.N - 1)];
        values_of(a, sx[i16], ws, false, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (p.bias) v[i] += (float)reinterpret_cast<const O*>(p.bias)[(int64_t)rt.g * p.N + min(n + i, p.N - 1)];
            if (p.relu) v[i] = v[i] < 0.0f ? 0.0f : v[i];
        }
    }
    store4<O>(p.y + o * p.ldy, n, p.N, v, p.vec);
}

namespace {

int64_t code_row(int64_t K) { return (K + CHUNK - 1) / CHUNK * CHUNK; }   // codes in whole chunks

int check_int8(const bnn_grouped* q) {
    if (!q) return fail(BNN_ERR_INVALID, "grouped descriptor is NULL");
    if (q->dtype < BNN_TYPE_F32 || q->dtype > BNN_TYPE_F16) return fail(BNN_ERR_INVALID, "dtype must be one of bnn_dtype");
    if (q->rows < 0 || q->copies < 1 || q->members < 1 || q->inputs < 1 || q->outputs < 1) return fail(BNN_ERR_INVALID, "bad rows / copies / members / inputs / outputs");
    if (q->rows >= (1LL << 30) / q->copies + ((1LL << 30) % q->copies != 0)) return fail(BNN_ERR_RANGE, "rows x copies must stay below 2^30");
    if (q->outputs > (1 << 24) || q->members > (1 << 24)) return fail(BNN_ERR_RANGE, "members and outputs must stay below 2^24");
    if (q->inputs > 131072) return fail(BNN_ERR_RANGE, "the 32-bit sums hold up to 131072 products of 8-bit integers");   // 2^17 * 128^2 = 2^31: sum_f32
    if (q->rows == 0) return 0;
    if ((q->gather || q->scatter) && !q->order) return fail(BNN_ERR_INVALID, "gather / scatter need order");
    if (!q->offsets && (q->members != 1 || q->copies != 1 || q->gather || q->scatter)) return fail(BNN_ERR_INVALID, "without offsets there is one member and no order");
    return 0;
}

RowsParams int8_params(const bnn_grouped* q, const int8_t* w, const float* w_scale, const void* bias, void* y) {
    RowsParams p{};
    p.w = (const char*)w; p.bias = bias; p.y = (char*)y; p.ws = w_scale;
    p.order = q->order; p.offsets = q->offsets;
    p.w_member = q->w_member; p.w_row = q->w_row; p.ldy = q->y_row * type_size(q->dtype);
    p.P = (int32_t)(q->rows * q->copies); p.G = q->members; p.N = q->outputs; p.K = q->inputs;
    p.gather_div = q->gather ? q->copies : 0; p.scatter = q->scatter ? 1 : 0; p.relu = q->relu ? 1 : 0;
    return p;
}

}  // namespace

extern "C" {

int bnn_quantize_rows(const void* x, int32_t dtype, int64_t rows, int32_t K, int64_t x_row, int8_t* q, int64_t q_row, float* scale, void* stream) {
    if (rows < 0 || K < 1 || dtype < BNN_TYPE_F32 || dtype > BNN_TYPE_F16 || q_row < K) return fail(BNN_ERR_INVALID, "bad argument");
    if (rows == 0) return 0;
    if (!x || !q || !scale) return fail(BNN_ERR_INVALID, "NULL argument");
    if (rows > 0x7fffffffLL || K > (1 << 24)) return fail(BNN_ERR_RANGE, "rows must stay below 2^31, their length below 2^24");
    const hipStream_t st = (hipStream_t)stream;
    const auto launch = [&](auto tag) -> int {
        using T = typename decltype(tag)::type;
        const char* xb = (const char*)x;
        const int64_t ldx = x_row * (int64_t)sizeof(T);
        // a wave a row once the rows fill the chip with waves (a quarter of one for rows of up to 1 KB); a workgroup a row below that, and for rows
        // that a wave would not hold
        const int64_t kbytes = (int64_t)K * sizeof(T);
        const int tpr = rows < 2048 || kbytes > 64 * 8 * CHUNK ? 256 : kbytes <= 1024 ? 16 : 64;
        for (int64_t r0 = 0; r0 < rows; r0 += 1 << 22) {   // (a grid has fewer than 2^32 threads)
            const int64_t n = std::min<int64_t>(rows - r0, 1 << 22);
            const unsigned nblk = (unsigned)((n + 256 / tpr - 1) / (256 / tpr));
            const char* xr = xb + r0 * ldx;
            int8_t* qr = q + r0 * q_row;
            if (kbytes < CHUNK) hipLaunchKernelGGL(bnn_quantize_short_rows_kernel<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, xr, ldx, n, K, qr, q_row, scale + r0);
            else if (tpr == 16) hipLaunchKernelGGL((bnn_quantize_rows_kernel<T, 16>), dim3(nblk), dim3(256), 0, st, xr, ldx, n, K, qr, q_row, scale + r0);
            else if (tpr == 64) hipLaunchKernelGGL((bnn_quantize_rows_kernel<T, 64>), dim3(nblk), dim3(256), 0, st, xr, ldx, n, K, qr, q_row, scale + r0);
            else hipLaunchKernelGGL((bnn_quantize_rows_kernel<T, 256>), dim3(nblk), dim3(256), 0, st, xr, ldx, n, K, qr, q_row, scale + r0);
            HIP_TRY(hipGetLastError());
        }
        return 0;
    };
    if (dtype == BNN_TYPE_F32) return launch(Tag<float>{});
    return dtype == BNN_TYPE_BF16 ? launch(Tag<__bf16>{}) : launch(Tag<_Float16>{});
}

int bnn_int8_linear_form(const bnn_grouped* q, const int8_t* x, const int8_t* w, const void* y, int32_t* form) {
    if (!form) return fail(BNN_ERR_INVALID, "bad argument");
    if (int rc = check_int8(q)) return rc;
    RowsParams p = int8_params(q, w, nullptr, nullptr, (void*)y);
    p.x = (const char*)x; p.ldx = q->x_row;
    const auto of = [&](auto tag) {
        using O = typename decltype(tag)::type;
        set_vec<O>(p);
        return rows_form<int8_t, O, false>(p);
    };
    const RowsForm f = q->dtype == BNN_TYPE_F32 ? of(Tag<float>{}) : q->dtype == BNN_TYPE_BF16 ? of(Tag<__bf16>{}) : of(Tag<_Float16>{});
    const int32_t values[6] = {f.kind, f.rows, f.outputs, f.direct, f.steps, 1};
    std::copy(values, values + 6, form);
    return 0;
}

int bnn_int8_linear(const bnn_grouped* q, const int8_t* x, const float* x_scale, const int8_t* w, const float* w_scale, const void* bias, void* y,
                    void* stream) {
    if (int rc = check_int8(q)) return rc;
    if (q->rows == 0) return 0;
    if (!x || !x_scale || !w || !w_scale || !y) return fail(BNN_ERR_INVALID, "NULL argument");
    RowsParams p = int8_params(q, w, w_scale, bias, y);
    p.x = (const char*)x; p.xs = x_scale; p.ldx = q->x_row;
    if (q->dtype == BNN_TYPE_F32) return launch_rows_typed<int8_t, float, false>(p, (hipStream_t)stream);
    if (q->dtype == BNN_TYPE_BF16) return launch_rows_typed<int8_t, __bf16, false>(p, (hipStream_t)stream);
    return launch_rows_typed<int8_t, _Float16, false>(p, (hipStream_t)stream);
}

size_t bnn_int8_linear_rows_workspace_bytes(const bnn_grouped* q) {
    if (!q || q->rows <= 0 || q->copies < 1 || q->inputs < 1) return 0;
    const size_t rows = (size_t)q->rows * (q->gather ? 1 : q->copies);
    return rows * (code_row(q->inputs) + sizeof(float));
}

int bnn_int8_linear_rows(const bnn_grouped* q, const void* x, int32_t x_dtype, void* workspace, const int8_t* w, const float* w_scale, const void* bias, void* y,
                         void* stream) {
    if (int rc = check_int8(q)) return rc;
    if (x_dtype < BNN_TYPE_F32 || x_dtype > BNN_TYPE_F16) return fail(BNN_ERR_INVALID, "x_dtype must be one of bnn_dtype");
    if (q->rows == 0) return 0;
    if (!x || !workspace || !w || !w_scale || !y) return fail(BNN_ERR_INVALID, "NULL argument");
    const int64_t P = q->rows * q->copies, ld = code_row(q->inputs);
    // a handful of rows: one launch (one row x 4 096 x 4 096: see the kernel) as long as their codes fit LDS
    const size_t lds = 8 * 64 * 16 + 16 * 4 + 16 * 4 + (size_t)std::min<int64_t>(P, 16) * ((ld + 63) / 64 * 64 + 16);
    if (P <= 32 && lds <= 160 * 1024) {
        RowsParams p = int8_params(q, w, w_scale, bias, y);
        p.x = (const char*)x;
        p.ldx = q->x_row * type_size(x_dtype);
        const auto launch = [&](auto xt, auto ot) -> int {
            using XT = typename decltype(xt)::type;
            using O = typename decltype(ot)::type;
            set_vec<O>(p);
            if (int rc = set_grid(p, 16, 16, 1, 512)) return rc;
            constexpr auto* kern = &bnn_int8_handful_kernel<XT, O>;
            allow_big_lds<kern>();
            hipLaunchKernelGGL(*kern, dim3((unsigned)p.nblk), dim3(512), lds, (hipStream_t)stream, p, (int)((ld + 63) / 64 * 64 + 16));
            HIP_TRY(hipGetLastError());
            return 0;
        };
        const auto with_out = [&](auto xt) -> int {
            if (q->dtype == BNN_TYPE_F32) return launch(xt, Tag<float>{});
            return q->dtype == BNN_TYPE_BF16 ? launch(xt, Tag<__bf16>{}) : launch(xt, Tag<_Float16>{});
        };
        if (x_dtype == BNN_TYPE_F32) return with_out(Tag<float>{});
        return x_dtype == BNN_TYPE_BF16 ? with_out(Tag<__bf16>{}) : with_out(Tag<_Float16>{});
    }
    const int64_t rows = q->gather ? q->rows : P;
    int8_t* codes = (int8_t*)workspace;
    float* scale = (float*)(codes + rows * ld);
    if (int rc = bnn_quantize_rows(x, x_dtype, rows, q->inputs, q->x_row, codes, ld, scale, stream)) return rc;
    bnn_grouped quant = *q;
    quant.x_row = ld;
    return bnn_int8_linear(&quant, codes, scale, w, w_scale, bias, y, stream);
}

}  // extern "C"
