// bnn_tile.hip.h -- the matrix-product tiles under the grouped and 8-bit linear layers (bnn_ops_grouped.hip, bnn_ops_int8.hip).
//
// A tile product is C[m][n] += sum_k A(m, k) B(n, k).  Both operands are staged through LDS 128 bytes of the reduction at a time (64 16-bit
// values, 32 floats or 128 8-bit integers) in one of two layouts:
//   KC  the reduction is contiguous in memory: [row][128 bytes]; the eight 16-byte chunks of a row are permuted by its index, so that the
//       16 rows one matrix instruction reads at a time lie in different banks;
//   FC  the other ("free") index is contiguous: [k][width]; a fragment is read through the transposing LDS read (16-bit types) or float by
//       float.  Used where the reduction runs over the rows of a row-major matrix: dX = dY W, dW = dY^T X.
// The matrix instructions take 64 bytes of the reduction per fragment: lane l holds row l & 15, bytes 16 (l >> 4) .. + 15.  Their result has
// four consecutive FIRST-operand indices in one lane, so the operand whose index is contiguous in the output goes first and a lane stores
// 8 or 16 bytes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace bnn {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float tf32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

#define BNN_LDS __attribute__((address_space(3)))
#define BNN_GLOBAL __attribute__((address_space(1)))

constexpr int STAGE_BYTES = 128;   // of the reduction per LDS stage
constexpr int CHUNK = 16;          // bytes of one load

// ---- one fragment product: 64 bytes of the reduction of 16 x 16 outputs --------------------------------------------------------------
template <typename T> struct Mma;
template <> struct Mma<__bf16> {
    using Acc = tf32x4;
    static __device__ __forceinline__ Acc mul(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<_Float16> {
    using Acc = tf32x4;
    static __device__ __forceinline__ Acc mul(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<float> {   // k = 4 q + j goes into instruction j from lane group q: the same order for both operands
    using Acc = tf32x4;
    static __device__ __forceinline__ Acc mul(u32x4 a, u32x4 b, Acc c) {
        const tf32x4 x = __builtin_bit_cast(tf32x4, a), y = __builtin_bit_cast(tf32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
};
template <> struct Mma<int8_t> {
    using Acc = i32x4;
    static __device__ __forceinline__ Acc mul(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    }
};

// Partial sums joined.  Whole numbers as unsigned ones: 2^17 products of -128 and -128 are 2^31, the one sum beyond 32 signed bits (the least is
// -2^17 x 128 x 127), and it stands as the lowest value until it becomes a float.
__device__ __forceinline__ tf32x4 join(tf32x4 a, tf32x4 b) { return a + b; }
__device__ __forceinline__ i32x4 join(i32x4 a, i32x4 b) { return __builtin_bit_cast(i32x4, __builtin_bit_cast(u32x4, a) + __builtin_bit_cast(u32x4, b)); }
__device__ __forceinline__ float sum_f32(int32_t s) { return s == INT32_MIN ? 0x1p31f : (float)s; }

// What a product's sum stands for.  Of 8-bit operands: sum * (xs * ws), the scales taken apart into mantissa and exponent, so that their product may be
// far smaller or larger than a float (1e-30 and 1e-20; 1e30 and 1e30 where the sum is zero).  Where every
// factor and product is a normal float the bits are those of the plain product.
struct Scale {
    float m;   // in [0.5, 1); zero, NaN and infinity stay as they are
    int e;
    __device__ __forceinline__ Scale() : m(1.0f), e(0) {}
    __device__ __forceinline__ explicit Scale(float s) : m(__builtin_amdgcn_frexp_mantf(s)), e(__builtin_amdgcn_frexp_expf(s)) {}
};
__device__ __forceinline__ float value_of(int32_t sum, Scale xs, Scale ws) { return __builtin_amdgcn_ldexpf(sum_f32(sum) * (xs.m * ws.m), xs.e + ws.e); }
__device__ __forceinline__ float value_of(float sum, Scale, Scale) { return sum; }
// The same of four neighbours where a wave's few instructions in a row are what counts: plain products first, looked at again if one of the scales' is
// not an ordinary float (3 000 rows x 40 -> 40 in 8 bits: 6.20 us, taken apart every time 6.45).  nobody: rows whose sums are zero and have no scales (zero
// times another member's NaN scale is not zero).
__device__ __forceinline__ void values_of(i32x4 sum, float xs, const float (&ws)[4], bool nobody, float (&v)[4]) {
    bool ordinary = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float s = xs * ws[i];
        v[i] = sum_f32(sum[i]) * s;
        ordinary &= __builtin_isnormal(s);
    }
    if (!ordinary)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = nobody ? 0.0f : value_of(sum[i], Scale(xs), Scale(ws[i]));
}
__device__ __forceinline__ void values_of(tf32x4 sum, float, const float (&)[4], bool, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = sum[i];
}

// ---- 16-byte loads of rows with any alignment and any length -------------------------------------------------------------------------
struct __attribute__((packed, aligned(1))) Bytes16 { u32x4 v; };
__device__ __forceinline__ u32x4 load_any(const char* at) { return reinterpret_cast<const Bytes16*>(at)->v; }

// Bytes [byte, byte + 16) of a row of nbytes >= 16, zero behind it: the row's last 16 bytes at most, shifted down (no branch: the loads of a
// thread stay in flight together)
template <typename T>
__device__ __forceinline__ u32x4 load_tail(const char* row, int64_t byte, int64_t nbytes) {
    const int64_t at = byte < nbytes - CHUNK ? byte : nbytes - CHUNK;
    const int d = byte - at < CHUNK ? (int)(byte - at) : CHUNK;
    u32x4 v = load_any(row + at);
    if (d & 4) v = u32x4{v.y, v.z, v.w, 0};
    if (d & 8) v = u32x4{v.z, v.w, 0, 0};
    if (d & 16) v = u32x4{0, 0, 0, 0};
    if constexpr (sizeof(T) < 4) {
        const unsigned s = d & 3;
        v = u32x4{__builtin_amdgcn_alignbyte(v.y, v.x, s), __builtin_amdgcn_alignbyte(v.z, v.y, s), __builtin_amdgcn_alignbyte(v.w, v.z, s),
                  __builtin_amdgcn_alignbyte(0, v.w, s)};
    }
    return v;
}
// the same for rows shorter than that
template <typename T>
__device__ __forceinline__ u32x4 load_short(const char* row, int64_t byte, int64_t nbytes) {
    u32x4 r;
    T tmp[CHUNK / sizeof(T)];
#pragma unroll
    for (int i = 0; i < (int)(CHUNK / sizeof(T)); ++i)
        tmp[i] = byte + (int64_t)((i + 1) * sizeof(T)) <= nbytes ? reinterpret_cast<const T*>(row + byte)[i] : (T)0;
    __builtin_memcpy(&r, tmp, CHUNK);
    return r;
}
// inside: the caller knows (for all lanes) that the chunk ends within the row
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const char* row, int64_t byte, int64_t nbytes, bool inside) {
    if (inside) return load_any(row + byte);
    if (nbytes >= CHUNK) return load_tail<T>(row, byte, nbytes);
    return load_short<T>(row, byte, nbytes);
}

static __device__ __attribute__((aligned(16))) const uint32_t zero_chunk[4] = {0, 0, 0, 0};   // where a lane outside the reduction reads

// 64 lanes x 16 bytes from their own addresses to 1 024 contiguous bytes of LDS, without a register in between
__device__ __forceinline__ void load_to_lds(const char* src, char* lds) {
    __builtin_amdgcn_global_load_lds((const BNN_GLOBAL void*)src, (BNN_LDS void*)lds, CHUNK, 0, 0);
}

// ---- LDS layouts ----------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int kc_swz(int row) { return (row >> 1) & 7; }

template <typename T, int W>
__device__ __forceinline__ int fc_swz(int k) {   // in chunks; the rows one fragment read touches go to different 32 (64) byte blocks
    constexpr int blocks = W * (int)sizeof(T) / 32;
    if constexpr (sizeof(T) == 4) return (((k >> 2) & 3) << 2) & (W / 4 - 1);
    else if constexpr (blocks >= 8) return ((k & 3) | ((k >> 1) & 4)) << 1;
    else return (((k >> 1) & 1) | ((k >> 2) & 2)) << 1 & (2 * blocks - 1);
}

template <typename T>
constexpr int stage_k() { return STAGE_BYTES / (int)sizeof(T); }

// a 16-row fragment, 64-byte step s of the stage
template <typename T>
__device__ __forceinline__ u32x4 frag_kc(const char* tile, int row0, int s, int lane) {
    const int row = row0 + (lane & 15);
    return *reinterpret_cast<const u32x4*>(tile + row * STAGE_BYTES + (((s * 4 + (lane >> 4)) ^ kc_swz(row)) << 4));
}
// The transposing read of four rows: lanes 4 j .. 4 j + 3 of a group of 16 give row j, lane i receives column i.  (The pointer is restrict: it never
// meets a load into LDS that is still under way -- the waits are written in the loop -- and without the word the compiler waits for all of them.)
__device__ __forceinline__ u32x2 read_transposed(const BNN_LDS s16x4* __restrict__ a) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((BNN_LDS s16x4*)a));
}
template <typename T, int W>
__device__ __forceinline__ u32x4 frag_fc(const char* tile, int col0, int s, int lane) {
    const int q = lane >> 4, i = lane & 15;
    if constexpr (sizeof(T) == 4) {
        u32x4 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int k = s * 16 + 4 * q + j, col = col0 + i;
            r[j] = *reinterpret_cast<const uint32_t*>(tile + k * W * 4 + (((col >> 2) ^ fc_swz<T, W>(k)) << 4) + (col & 3) * 4);
        }
        return r;
    } else {
        u32x4 r;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = s * 32 + 8 * q + 4 * h + (i >> 2);
            const int chunk = (col0 >> 3) + ((i & 3) >> 1);
            const char* a = tile + k * W * 2 + ((chunk ^ fc_swz<T, W>(k)) << 4) + (i & 1) * 8;
            const u32x2 v = read_transposed((const BNN_LDS s16x4*)a);
            r[2 * h] = v.x;
            r[2 * h + 1] = v.y;
        }
        return r;
    }
}

// ---- the tile of a workgroup --------------------------------------------------------------------------------------------------------------
struct RowTile { int g, r0, r1; };   // member, first row and end of the tile's rows (g == G: rows of nobody; g < 0: no such tile)

// Tile `t` of the grouped rows cut into pieces of BM per member.  Every wave finds it by itself: a lane takes the member(s) of its index, the
// tile counts are summed along the wave.  Offsets out of order or out of range are clamped to [0, P]: rows may then be wrong, accesses not.
__device__ __forceinline__ RowTile find_rows(const int32_t* __restrict__ off, int G, int P, int t, int BM) {
    const int lane = threadIdx.x & 63;
    if (off == nullptr) {
        const int64_t r0 = (int64_t)t * BM;
        return r0 < P ? RowTile{0, (int)r0, (int)(r0 + BM < P ? r0 + BM : P)} : RowTile{-1, 0, 0};
    }
    auto range = [&](int g, int& s, int& e) {
        s = min(max(off[g], 0), P);
        e = g < G ? min(max(off[g + 1], s), P) : P;
    };
    const int per = (G + 64) / 64;   // members per lane: G + 1 entries, the last one the rows of nobody
    int s = 0, e = 0, mine = 0;
    for (int j = 0; j < per; ++j) {
        const int g = lane * per + j;
        if (g > G) break;
        range(g, s, e);
        mine += (e - s + BM - 1) / BM;
    }
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(incl, d);
        if (lane >= d) incl += v;
    }
    const uint64_t hit = __ballot(incl > t);
    if (hit == 0) return RowTile{-1, 0, 0};
    const int src = __ffsll((unsigned long long)hit) - 1;
    int left = t - (__shfl(incl, src) - __shfl(mine, src));
    RowTile rt{-1, 0, 0};
    for (int j = 0; j < per; ++j) {
        const int g = __builtin_amdgcn_readfirstlane(src * per + j);
        if (g > G) break;
        range(g, s, e);
        const int n = (e - s + BM - 1) / BM;
        if (left < n) {
            rt.g = g;
            rt.r0 = s + left * BM;
            rt.r1 = min(rt.r0 + BM, e);
            break;
        }
        left -= n;
    }
    rt.g = __builtin_amdgcn_readfirstlane(rt.g);
    rt.r0 = __builtin_amdgcn_readfirstlane(rt.r0);
    rt.r1 = __builtin_amdgcn_readfirstlane(rt.r1);
    return rt;
}

// Workgroup -> (row tile, column tile): XCD x takes the x-th contiguous eighth of the order (workgroups go round the XCDs one by one), and the
// order walks bands of `band` row tiles by all column tiles, so that what runs together on an XCD shares its L2.
__device__ __forceinline__ void tile_of_block(int nblk, int tiles_n, int band, int& tm, int& tn) {
    int b = blockIdx.x;
    const int per = nblk / 8, rem = nblk % 8, x = b % 8, i = b / 8;
    b = x * per + min(x, rem) + i;
    const int width = band * tiles_n, bnd = b / width, in = b - bnd * width;
    const int rows_total = nblk / tiles_n, rows = min(band, rows_total - bnd * band);
    tn = in / rows;
    tm = bnd * band + in - tn * rows;
}

}  // namespace bnn
