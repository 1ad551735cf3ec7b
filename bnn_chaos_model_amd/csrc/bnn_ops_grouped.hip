// bnn_ops_grouped.hip -- rows sorted by the ensemble member that evaluates them, and the linear layer over such groups with its gradients.
// One of the translation units of libbnn_chaos_hip.so (bnn_internal.h lists them); entry points declared in include/bnn_chaos_hip.h, kernels of
// the products in bnn_grouped.hip.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "bnn_abi_common.h"
#include "bnn_grouped_host.h"

using namespace bnn;

// ---- group_rows: a stable counting sort -----------------------------------------------------------------------------------------------------
// One wave takes 64 consecutive pairs at a time, in order: the lanes that hold the same member are found with one ballot per bit of the key, a
// lane's place is the number of such lanes before it, and the wave's running count per member lives in LDS.  Pairs of nobody (member outside
// [0, G)) take key G and come last.  Counts per (member, block), their prefix sums, then places; up to GROUP_CHUNK pairs one workgroup does it
// all.  A thread's keys are loaded at once and stay in registers.  Measured: 3 000 pairs of 30 members 4.5 us, 4 M pairs 5.7 + 3.0 + 17.3 (32 MB read and
// 16 MB written would take 10): bound by the chain of count, prefix and place in every workgroup.
constexpr int GROUP_CHUNK = 4096;      // pairs per workgroup
constexpr int GROUP_MAX_MEMBERS = 4096;

template <int WAVES>
struct Keys {
    static constexpr int PER = GROUP_CHUNK / WAVES, N = PER / 64;
    int key[N];   // of pairs lo + wave * PER + i * 64 + lane; -1 behind the end
    __device__ __forceinline__ void load(const int32_t* __restrict__ member, int64_t lo, int64_t P, int G) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t at = pair(lo, i);
            const int m = member[at < P ? at : P - 1];
            key[i] = at >= P ? -1 : m >= 0 && m < G ? m : G;
        }
    }
    __device__ __forceinline__ int64_t pair(int64_t lo, int i) const { return lo + (int64_t)(threadIdx.x >> 6) * PER + i * 64 + (threadIdx.x & 63); }
    // this workgroup's counts: wc[wave][G + 1]
    __device__ __forceinline__ void count(int G, int32_t* wc) const {
        for (int i = threadIdx.x; i < WAVES * (G + 1); i += WAVES * 64) wc[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (key[i] >= 0) atomicAdd(&wc[(threadIdx.x >> 6) * (G + 1) + key[i]], 1);   // (whole numbers: any order gives the same counts)
        __syncthreads();
    }
};

template <int WAVES>
__global__ __launch_bounds__(WAVES * 64) void bnn_group_count_kernel(const int32_t* __restrict__ member, int64_t P, int G, int32_t* __restrict__ cnt) {
    extern __shared__ int32_t wc[];
    Keys<WAVES> keys;
    keys.load(member, (int64_t)blockIdx.x * GROUP_CHUNK, P, G);
    keys.count(G, wc);
    for (int g = threadIdx.x; g <= G; g += WAVES * 64) {
        int32_t s = 0;
        for (int w = 0; w < WAVES; ++w) s += wc[w * (G + 1) + g];
        cnt[(int64_t)g * gridDim.x + blockIdx.x] = s;
    }
}

// sums along a row of 64 lanes, lane by lane
__device__ __forceinline__ int32_t wave_scan(int32_t v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int32_t o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// member g's counts over the blocks -> exclusive prefix in place, total behind the table; 1 024 counts a sweep, four to a thread
__global__ __launch_bounds__(256) void bnn_group_scan_kernel(int32_t* __restrict__ cnt, int nb, int32_t* __restrict__ total) {
    __shared__ int32_t wsum[4];
    int32_t* row = cnt + (int64_t)blockIdx.x * nb;
    const int wave = threadIdx.x >> 6;
    int32_t carry = 0;
    for (int b0 = 0; b0 < nb; b0 += 1024) {
        int32_t v[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = b0 + threadIdx.x * 4 + i;
            v[i] = b < nb ? row[b] : 0;
            sum += v[i];
        }
        const int32_t inc = wave_scan(sum);
        if ((threadIdx.x & 63) == 63) wsum[wave] = inc;
        __syncthreads();
        int32_t at = carry + inc - sum;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) at += wsum[w];
            carry += wsum[w];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = b0 + threadIdx.x * 4 + i;
            if (b < nb) row[b] = at;
            at += v[i];
        }
    }
    if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

// Between lanes of one wave that hand values to each other through LDS: what is read and written before comes before what follows.  A wave's LDS accesses
// are carried out in order, so this costs nothing; it holds the compiler to that order.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// SINGLE: one workgroup holds every pair (no count and scan launches in front)
template <int WAVES, bool SINGLE>
__global__ __launch_bounds__(WAVES * 64) void bnn_group_place_kernel(const int32_t* __restrict__ member, int64_t P, int G, const int32_t* __restrict__ cnt,
                                                                     const int32_t* __restrict__ total, int nbits, int32_t* __restrict__ order,
                                                                     int32_t* __restrict__ offsets) {
    extern __shared__ int32_t wc[];   // [WAVES][G + 1] counts -> places, then [G + 1] member starts
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, G1 = G + 1;
    int32_t* start = wc + WAVES * G1;
    const int64_t lo = (int64_t)blockIdx.x * GROUP_CHUNK;
    Keys<WAVES> keys;
    if (!SINGLE || P > 0) keys.load(member, lo, P, G);
    else
        for (int i = 0; i < keys.N; ++i) keys.key[i] = -1;
    if constexpr (!SINGLE)
        for (int g = threadIdx.x; g < G1; g += WAVES * 64) start[g] = total[g];
    keys.count(G, wc);
    if constexpr (SINGLE) {
        for (int g = threadIdx.x; g < G1; g += WAVES * 64) {
            int32_t s = 0;
            for (int w = 0; w < WAVES; ++w) s += wc[w * G1 + g];
            start[g] = s;
        }
        __syncthreads();
    }
    if (wave == 0) {
        int32_t carry = 0;
        for (int g0 = 0; g0 < G1; g0 += 64) {
            const int g = g0 + lane;
            const int32_t v = g < G1 ? start[g] : 0, inc = wave_scan(v);
            if (g < G1) {
                start[g] = carry + inc - v;
                if (blockIdx.x == 0) offsets[g] = carry + inc - v;
            }
            carry += __shfl(inc, 63);
        }
    }
    __syncthreads();
    for (int g = threadIdx.x; g < G1; g += WAVES * 64) {
        int32_t at = start[g];
        if constexpr (!SINGLE) at += cnt[(int64_t)g * gridDim.x + blockIdx.x];
        for (int w = 0; w < WAVES; ++w) {
            const int32_t c = wc[w * G1 + g];
            wc[w * G1 + g] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < keys.N; ++i) {
        const int key = keys.key[i];
        const bool in = key >= 0;
        uint64_t same = __ballot(in);
        for (int b = 0; b < nbits; ++b) {
            const uint64_t set = __ballot(in && ((key >> b) & 1));
            same &= ((key >> b) & 1) ? set : ~set;
        }
        if (in) {
            const int before = __popcll(same & ((1ull << lane) - 1));
            const int32_t at = wc[wave * G1 + key];
            order[at + before] = (int32_t)keys.pair(lo, i);
            wave_sync();   // every lane of the wave has read `at` ...
            if (before == 0) wc[wave * G1 + key] = at + __popcll(same);
        }
        wave_sync();       // ... and reads what its first one has written
    }
}

// ---- small kernels of the gradients --------------------------------------------------------------------------------------------------------
// Both sweeps below go over rows of `nc` chunks of V elements and are bound by memory.  A thread finds its row once by division and then steps by the
// grid's width.  V: 16 bytes of the narrowest operand where every row starts on a 16-byte border, else one element.  Against one element and one
// 64-bit division at a time: the mask of 65 536 x 4 096 bf16 648 -> 321 us (5.0 TB/s), dX of 32 768 x 2 copies x 4 096 with its product 645 -> 567.
struct Sweep {
    int64_t r, dr;
    int32_t c, dc, nc;
    __device__ __forceinline__ Sweep(int32_t chunks) : nc(chunks) {
        const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
        r = first / nc; c = (int32_t)(first - r * nc);
        dr = step / nc; dc = (int32_t)(step - dr * nc);
    }
    __device__ __forceinline__ void next() {
        r += dr; c += dc;
        if (c >= nc) { c -= nc; ++r; }
    }
};
template <typename T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Chunk {
    T v[V];
};

// dx of a row that fed several (row, copy) pairs: their sum, in the copies' order
template <typename O, int V>
__global__ __launch_bounds__(256) void bnn_sum_copies_kernel(const float* __restrict__ pair, int64_t rows, int copies, int K, O* __restrict__ dx) {
    for (Sweep at(K / V); at.r < rows; at.next()) {
        const float* from = pair + at.r * copies * K + at.c * V;
        float s[V] = {};
        for (int c = 0; c < copies; ++c, from += K) {
            const Chunk<float, V> f = *(const Chunk<float, V>*)from;
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] += f.v[i];
        }
        Chunk<O, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) out.v[i] = (O)s[i];
        *(Chunk<O, V>*)(dx + at.r * K + at.c * V) = out;
    }
}

// the splits' sums added in order: dW (n values), then db (nb) behind all the splits of dW
template <typename O>
__global__ __launch_bounds__(256) void bnn_sum_splits_kernel(const float* __restrict__ part, int splits, int64_t n, O* __restrict__ dw, int64_t nb, O* __restrict__ db) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n + nb; i += (int64_t)gridDim.x * 256) {
        const bool w = i < n;
        const int64_t at = w ? i : splits * n + (i - n), step = w ? n : nb;
        float s = 0.0f;
        for (int c = 0; c < splits; ++c) s += part[at + c * step];
        if (w) dw[i] = (O)s;
        else db[i - n] = (O)s;
    }
}

// nn.ReLU's gradient: zero where the layer's output is <= 0, dy elsewhere (a NaN output passes it, so that a NaN is not lost on the way back)
template <typename T, int V>
__global__ __launch_bounds__(256) void bnn_relu_grad_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ y, int64_t ldy, int64_t rows, int N,
                                                            T* __restrict__ out) {
    for (Sweep at(N / V); at.r < rows; at.next()) {
        const Chunk<T, V> d = *(const Chunk<T, V>*)(dy + at.r * lddy + at.c * V), v = *(const Chunk<T, V>*)(y + at.r * ldy + at.c * V);
        Chunk<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = (float)v.v[i] <= 0.0f ? (T)0 : d.v[i];
        *(Chunk<T, V>*)(out + at.r * N + at.c * V) = o;
    }
}

namespace {

unsigned sweep_blocks(int64_t n) { return (unsigned)std::min<int64_t>(std::max<int64_t>((n + 255) / 256, 1), 256 * 16); }

ReducePlan plan_of(const bnn_grouped* q) { return reduce_plan(q->rows * q->copies, q->members, q->outputs, q->inputs, q->dtype == BNN_TYPE_F32); }

int check_grouped(const bnn_grouped* q) {
    if (!q) return fail(BNN_ERR_INVALID, "grouped descriptor is NULL");
    if (q->dtype < BNN_TYPE_F32 || q->dtype > BNN_TYPE_F16) return fail(BNN_ERR_INVALID, "dtype must be one of bnn_dtype");
    if (q->rows < 0 || q->copies < 1 || q->members < 1 || q->inputs < 1 || q->outputs < 1) return fail(BNN_ERR_INVALID, "bad rows / copies / members / inputs / outputs");
    if (q->rows >= (1LL << 30) / q->copies + ((1LL << 30) % q->copies != 0)) return fail(BNN_ERR_RANGE, "rows x copies must stay below 2^30");
    if (q->inputs > (1 << 24) || q->outputs > (1 << 24) || q->members > (1 << 24)) return fail(BNN_ERR_RANGE, "members, inputs and outputs must stay below 2^24");
    if (q->x_row < 0 || q->y_row < 0 || q->x_row > (1 << 28) || q->y_row > (1 << 28)) return fail(BNN_ERR_RANGE, "rows must be less than 2^28 elements apart");
    if ((q->gather || q->scatter) && q->rows && !q->order) return fail(BNN_ERR_INVALID, "gather / scatter need order");
    return 0;
}

RowsParams forward_params(const bnn_grouped* q, const void* x, const void* w, const void* bias, void* y) {
    const int es = type_size(q->dtype);
    RowsParams p{};
    p.x = (const char*)x; p.w = (const char*)w; p.bias = bias; p.y = (char*)y;
    p.order = q->order; p.offsets = q->offsets;
    p.ldx = q->x_row * es; p.w_member = q->w_member * es; p.w_row = q->w_row * es; p.ldy = q->y_row * es;
    p.P = (int32_t)(q->rows * q->copies); p.G = q->members; p.N = q->outputs; p.K = q->inputs;
    p.gather_div = q->gather ? q->copies : 0; p.scatter = q->scatter ? 1 : 0; p.relu = q->relu ? 1 : 0;
    return p;
}

// a row of x fed several pairs: their gradients meet in fp32, one rounding at the end
bool dx_by_pairs(const bnn_grouped* q) { return q->gather && q->copies > 1; }

RowsParams dx_params(const bnn_grouped* q, const void* dy, const void* w, void* out) {   // out: dx, or the pairs' gradients
    const int es = type_size(q->dtype);
    RowsParams p{};
    p.x = (const char*)dy; p.w = (const char*)w; p.y = (char*)out;
    p.order = q->order; p.offsets = q->offsets;
    p.ldx = q->y_row * es; p.w_member = q->w_member * es; p.w_row = q->w_row * es;
    p.ldy = dx_by_pairs(q) ? (int64_t)q->inputs * sizeof(float) : q->x_row * es;
    p.P = (int32_t)(q->rows * q->copies); p.G = q->members; p.N = q->inputs; p.K = q->outputs;
    p.gather_div = q->scatter ? 1 : 0; p.scatter = q->gather ? 1 : 0;
    return p;
}

ReduceParams dw_params(const bnn_grouped* q, const void* dy, const void* x, void* dw) {
    const int es = type_size(q->dtype);
    ReduceParams p{};
    p.x = (const char*)x; p.dy = (const char*)dy; p.dw = (char*)dw;
    p.offsets = q->offsets;
    p.ldx = (uint32_t)(q->x_row * es); p.lddy = (uint32_t)(q->y_row * es);
    p.P = (int32_t)(q->rows * q->copies); p.G = q->members; p.N = q->outputs; p.K = q->inputs;
    p.m_x = q->gather ? -1 : 0; p.m_dy = q->scatter ? -1 : 0;
    p.list = p.m_x | p.m_dy ? q->order : nullptr;
    while ((1LL << p.shift) < q->copies) ++p.shift;   // pair / copies = (2 pair * magic >> 32) >> shift, exact below 2^31: magic = ceil(2^(31 + shift) / copies)
    p.magic = (uint32_t)(((1ULL << (31 + p.shift)) + q->copies - 1) / q->copies);
    return p;
}

}  // namespace

extern "C" {

int bnn_grouped_linear_form(const bnn_grouped* q, int32_t pass, const void* a, const void* b, const void* out, int32_t* form) {
    if (!form || pass < BNN_PASS_FORWARD || pass > BNN_PASS_DW) return fail(BNN_ERR_INVALID, "bad argument");
    if (int rc = check_grouped(q)) return rc;
    RowsForm f;
    int splits = 1;
    if (pass == BNN_PASS_FORWARD) f = form_of_rows(q->dtype, q->dtype, false, forward_params(q, a, b, nullptr, (void*)out));
    else if (pass == BNN_PASS_DX) f = form_of_rows(q->dtype, dx_by_pairs(q) ? BNN_TYPE_F32 : q->dtype, true, dx_params(q, a, b, (void*)out));
    else {
        const ReducePlan plan = plan_of(q);
        f = form_of_reduce(q->dtype, dw_params(q, a, b, (void*)out), plan.tile);
        splits = plan.splits;
    }
    const int32_t values[6] = {f.kind, f.rows, f.outputs, f.direct, f.steps, splits};
    std::copy(values, values + 6, form);
    return 0;
}

size_t bnn_group_rows_workspace_bytes(int64_t pairs, int32_t members) {
    if (pairs <= GROUP_CHUNK || members < 1 || members > GROUP_MAX_MEMBERS) return 0;
    const int64_t nb = (pairs + GROUP_CHUNK - 1) / GROUP_CHUNK;
    return (size_t)(nb + 1) * (members + 1) * sizeof(int32_t);
}

int bnn_group_rows_i32(const int32_t* member, int64_t pairs, int32_t members, int32_t* order, int32_t* offsets, void* workspace, void* stream) {
    if (pairs < 0 || members < 1) return fail(BNN_ERR_INVALID, "bad pairs / members");
    if (members > GROUP_MAX_MEMBERS) return fail(BNN_ERR_UNSUPPORTED, "group_rows sorts by up to 4096 members");
    if (pairs >= (1LL << 30)) return fail(BNN_ERR_RANGE, "pairs must stay below 2^30");
    if (!offsets || (pairs && (!member || !order))) return fail(BNN_ERR_INVALID, "NULL argument");
    const int64_t nb = (pairs + GROUP_CHUNK - 1) / GROUP_CHUNK;
    if (nb > 1 && !workspace) return fail(BNN_ERR_INVALID, "workspace is NULL");
    int nbits = 1;
    while ((members >> nbits) != 0) ++nbits;   // keys 0 .. members
    const hipStream_t st = (hipStream_t)stream;
    // sixteen waves while their counts fit the 160 KB of LDS, four beyond that
    const auto launch = [&](auto waves_tag) -> int {
        constexpr int WAVES = decltype(waves_tag)::value;
        const size_t lds_count = (size_t)WAVES * (members + 1) * sizeof(int32_t), lds = lds_count + (size_t)(members + 1) * sizeof(int32_t);
        if (nb <= 1) {
            allow_big_lds<bnn_group_place_kernel<WAVES, true>>();
            hipLaunchKernelGGL((bnn_group_place_kernel<WAVES, true>), dim3(1), dim3(WAVES * 64), lds, st, member, pairs, members, (const int32_t*)nullptr,
                               (const int32_t*)nullptr, nbits, order, offsets);
            HIP_TRY(hipGetLastError());
            return 0;
        }
        int32_t* cnt = (int32_t*)workspace;
        int32_t* total = cnt + nb * (members + 1);
        allow_big_lds<bnn_group_count_kernel<WAVES>>();
        allow_big_lds<bnn_group_place_kernel<WAVES, false>>();
        hipLaunchKernelGGL(bnn_group_count_kernel<WAVES>, dim3((unsigned)nb), dim3(WAVES * 64), lds_count, st, member, pairs, members, cnt);
        HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL(bnn_group_scan_kernel, dim3((unsigned)members + 1), dim3(256), 0, st, cnt, (int)nb, total);
        HIP_TRY(hipGetLastError());
        hipLaunchKernelGGL((bnn_group_place_kernel<WAVES, false>), dim3((unsigned)nb), dim3(WAVES * 64), lds, st, member, pairs, members, (const int32_t*)cnt,
                           (const int32_t*)total, nbits, order, offsets);
        HIP_TRY(hipGetLastError());
        return 0;
    };
    return members < 1024 ? launch(std::integral_constant<int, 16>{}) : launch(std::integral_constant<int, 4>{});
}

int bnn_grouped_linear(const bnn_grouped* q, const void* x, const void* w, const void* bias, void* y, void* stream) {
    if (int rc = check_grouped(q)) return rc;
    if (q->rows == 0) return 0;
    if (!x || !w || !y || !q->offsets) return fail(BNN_ERR_INVALID, "NULL argument");
    return launch_rows(q->dtype, q->dtype, false, forward_params(q, x, w, bias, y), (hipStream_t)stream);
}

size_t bnn_grouped_linear_dx_workspace_bytes(const bnn_grouped* q) {
    if (!q || q->rows <= 0 || q->inputs < 1 || q->copies < 2 || !q->gather) return 0;
    return (size_t)q->rows * q->copies * q->inputs * sizeof(float);
}

int bnn_grouped_linear_dx(const bnn_grouped* q, const void* dy, const void* w, void* dx, void* workspace, void* stream) {
    if (int rc = check_grouped(q)) return rc;
    if (q->rows == 0) return 0;
    if (!dy || !w || !dx || !q->offsets) return fail(BNN_ERR_INVALID, "NULL argument");
    const bool pairs = dx_by_pairs(q);
    if (pairs && !workspace) return fail(BNN_ERR_INVALID, "workspace is NULL");
    if (pairs && q->x_row != q->inputs) return fail(BNN_ERR_INVALID, "dx of several copies must be dense");
    if (int rc = launch_rows(q->dtype, pairs ? BNN_TYPE_F32 : q->dtype, true, dx_params(q, dy, w, pairs ? workspace : dx), (hipStream_t)stream)) return rc;
    if (!pairs) return 0;
    const auto join = [&](auto tag) -> int {
        using O = typename decltype(tag)::type;
        constexpr int V = 16 / sizeof(O);
        const float* part = (const float*)workspace;
        const int64_t n = q->rows * (int64_t)q->inputs;
        if (q->inputs % V == 0 && ((uintptr_t)workspace | (uintptr_t)dx) % 16 == 0)
            hipLaunchKernelGGL((bnn_sum_copies_kernel<O, V>), dim3(sweep_blocks(n / V)), dim3(256), 0, (hipStream_t)stream, part, q->rows, q->copies, q->inputs, (O*)dx);
        else
            hipLaunchKernelGGL((bnn_sum_copies_kernel<O, 1>), dim3(sweep_blocks(n)), dim3(256), 0, (hipStream_t)stream, part, q->rows, q->copies, q->inputs, (O*)dx);
        HIP_TRY(hipGetLastError());
        return 0;
    };
    if (q->dtype == BNN_TYPE_F32) return join(Tag<float>{});
    if (q->dtype == BNN_TYPE_BF16) return join(Tag<__bf16>{});
    return join(Tag<_Float16>{});
}

size_t bnn_grouped_linear_dw_workspace_bytes(const bnn_grouped* q) {
    if (!q || q->rows <= 0 || q->members < 1 || q->inputs < 1 || q->outputs < 1) return 0;
    const int s = plan_of(q).splits;
    return s > 1 ? (size_t)s * q->members * q->outputs * ((size_t)q->inputs + 1) * sizeof(float) : 0;
}

int bnn_grouped_linear_dw(const bnn_grouped* q, const void* dy, const void* x, void* dw, void* db, void* workspace, void* stream) {
    if (int rc = check_grouped(q)) return rc;
    if (!dw || !q->offsets || (q->rows && (!dy || !x))) return fail(BNN_ERR_INVALID, "NULL argument");
    ReduceParams p = dw_params(q, dy, x, dw);
    p.db = db; p.part = (float*)workspace;
    const ReducePlan plan = plan_of(q);
    p.splits = q->rows ? plan.splits : 1;
    if (p.splits > 1 && (!workspace || (uintptr_t)workspace % 16)) return fail(BNN_ERR_INVALID, "workspace is NULL or not 16-byte aligned");
    if (int rc = launch_reduce(q->dtype, p, plan.tile, (hipStream_t)stream)) return rc;
    if (p.splits == 1) return 0;
    const int64_t n = (int64_t)p.G * p.N * p.K, nb = (int64_t)p.G * p.N;
    const float* part = (const float*)workspace;
    const hipStream_t st = (hipStream_t)stream;
    const auto join = [&](auto tag) -> int {
        using O = typename decltype(tag)::type;
        hipLaunchKernelGGL(bnn_sum_splits_kernel<O>, dim3(sweep_blocks(n + (db ? nb : 0))), dim3(256), 0, st, part, p.splits, n, (O*)dw, db ? nb : 0, (O*)db);
        HIP_TRY(hipGetLastError());
        return 0;
    };
    if (q->dtype == BNN_TYPE_F32) return join(Tag<float>{});
    if (q->dtype == BNN_TYPE_BF16) return join(Tag<__bf16>{});
    return join(Tag<_Float16>{});
}

int bnn_relu_grad(const void* dy, int64_t dy_row, const void* y, int64_t y_row, int64_t rows, int32_t N, int32_t dtype, void* out, void* stream) {
    if (rows < 0 || N < 1 || dtype < BNN_TYPE_F32 || dtype > BNN_TYPE_F16) return fail(BNN_ERR_INVALID, "bad argument");
    if (rows == 0) return 0;
    if (!dy || !y || !out) return fail(BNN_ERR_INVALID, "NULL argument");
    const auto launch = [&](auto tag) -> int {
        using T = typename decltype(tag)::type;
        constexpr int V = 16 / sizeof(T);
        const bool wide = N % V == 0 && dy_row % V == 0 && y_row % V == 0 && ((uintptr_t)dy | (uintptr_t)y | (uintptr_t)out) % 16 == 0;
        const int64_t n = rows * (int64_t)N;
        if (wide)
            hipLaunchKernelGGL((bnn_relu_grad_kernel<T, V>), dim3(sweep_blocks(n / V)), dim3(256), 0, (hipStream_t)stream, (const T*)dy, dy_row, (const T*)y, y_row, rows, N, (T*)out);
        else
            hipLaunchKernelGGL((bnn_relu_grad_kernel<T, 1>), dim3(sweep_blocks(n)), dim3(256), 0, (hipStream_t)stream, (const T*)dy, dy_row, (const T*)y, y_row, rows, N, (T*)out);
        HIP_TRY(hipGetLastError());
        return 0;
    };
    if (dtype == BNN_TYPE_F32) return launch(Tag<float>{});
    if (dtype == BNN_TYPE_BF16) return launch(Tag<__bf16>{});
    return launch(Tag<_Float16>{});
}

}  // extern "C"
