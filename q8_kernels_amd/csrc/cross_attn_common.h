// Shared pieces of the 16-bit cross attention kernels (forward and backward): operand layouts, tile staging, row addressing.
//
// Matrix products run on v_mfma_f32_32x32x16 (bf16 or fp16 operands, fp32 sums): A is 32 x 16 with lane l holding row l % 32,
// elements 8 (l / 32) .. + 7 of the 16; B the same with columns; the result has column l % 32 in every lane and rows
// 8 (i / 4) + 4 (l / 32) + i % 4 for i = 0 .. 15. Scores are formed with the long side as rows, so the 16 results of a lane
// belong to ONE column, and after rounding to 16 bits they are, eight by eight, the B operand of the next product without
// leaving the lane: result i = 8 s + j is element j of step s. The other operand of that product has to enumerate its 16
// long-side rows the same way (8 (j / 4) + 4 (l / 32) + j % 4), which is what two transposing LDS reads
// (ds_read_b64_tr_b16: lane i of 16 supplies the address of 4 elements of row i / 4 and receives column i of the 4 x 16
// block) give: rows 4 (l / 32) .. + 3 and the same 8 rows further.
//
// Query rows: the G query heads that share a key head are one sequence of R = G M rows (row r = query r % M of head r / M of
// the group). K and V are read once for all of them, and dK, dV are sums over all R rows, which is the gradient of a shared
// head. A unit is one (batch, key head).
//
// Tiles in LDS are row-major with rows of DP + 16 elements (DP: the head size D padded to 32, 64, 96 or 128): the 8 lanes of
// one LDS cycle of a 16-byte read, and the 4 rows of a transposing read, then fall on different banks.
#pragma once
#include "q8_common.h"
#include "q8_host.h"

namespace q8 {

constexpr int kXThreads = 256, kXWaves = 4, kXTile = 64;  // a workgroup; rows of a staged tile
constexpr float kLog2e = 1.4426950408889634f;

typedef short v4s16 __attribute__((ext_vector_type(4)));

struct XTensor {  // [B, heads, tokens, D] with unit last stride
    const uint16_t* p;
    int64_t sb, sh, st;
};
struct XOut {
    uint16_t* p;
    int64_t sb, sh, st;
};

template <int DT>
__device__ __forceinline__ v16f mfma16(v4u a, v4u b, v16f c) {
    if constexpr (DT == Q8_BF16) {
        typedef __bf16 v8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    } else {
        typedef _Float16 v8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
}

// two values rounded to nearest even
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (DT == Q8_BF16) return pack2_bf16(lo, hi);
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, f16x2));
}
template <int DT>
__device__ __forceinline__ float unpack(uint32_t h) { return DT == Q8_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h); }

__device__ __forceinline__ v16f splat16(float v) {
    v16f r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = v;
    return r;
}

// A operand: rows row0 + l % 32 of a row-major LDS tile, elements e0 + 8 (l / 32) .. + 7
template <int LD>
__device__ __forceinline__ v4u lds_rows(const uint16_t* tile, int row0, int e0, int lane) {
    return *reinterpret_cast<const v4u*>(tile + (row0 + (lane & 31)) * LD + e0 + ((lane >> 5) << 3));
}
// A operand of the transposed tile: column e0 + l % 32 over the 16 rows from row0, in the order of a score column's results
template <int LD>
__device__ __forceinline__ v4u lds_cols(const uint16_t* tile, int row0, int e0, int lane) {
    const uint16_t* p = tile + (row0 + ((lane >> 5) << 2) + ((lane & 15) >> 2)) * LD + e0 + (lane & 16) + ((lane & 3) << 2);
    const v4s16 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s16*)(p));
    const v4s16 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s16*)(p + 8 * LD));
    const v2i x = __builtin_bit_cast(v2i, a), y = __builtin_bit_cast(v2i, b);
    return v4u{(unsigned)x[0], (unsigned)x[1], (unsigned)y[0], (unsigned)y[1]};
}

// The B operand that results 8 s .. 8 s + 7 of a score column make
template <int DT>
__device__ __forceinline__ v4u pack_step(const v16f& v, int s) {
    return v4u{pack2<DT>(v[8 * s], v[8 * s + 1]), pack2<DT>(v[8 * s + 2], v[8 * s + 3]), pack2<DT>(v[8 * s + 4], v[8 * s + 5]),
               pack2<DT>(v[8 * s + 6], v[8 * s + 7])};
}

// 64 rows of a tensor on their way to LDS: requested early, written later. Rows or elements outside are zeros.
template <int DP>
struct Stage {
    static constexpr int LD = DP + 16, CPR = DP / 8, N = kXTile * CPR / kXThreads;
    v4u r[N];
    template <typename At>  // at(row): pointer to the row's first element, or NULL for a row of zeros
    __device__ __forceinline__ void load(At at, int D) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const int i = threadIdx.x + c * kXThreads, row = i / CPR, e = (i - row * CPR) * 8;
            const uint16_t* p = at(row);
            r[c] = (p != nullptr && e < D) ? *reinterpret_cast<const v4u*>(p + e) : v4u{0u, 0u, 0u, 0u};
        }
    }
    __device__ __forceinline__ void store(uint16_t* tile) const {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const int i = threadIdx.x + c * kXThreads, row = i / CPR, e = (i - row * CPR) * 8;
            *reinterpret_cast<v4u*>(tile + row * LD + e) = r[c];
        }
    }
};

// Which keys of a batch element count: those below its length whose mask byte is not zero.
struct XKeys {
    const int32_t* lens;   // [B] or NULL
    const uint8_t* mask;   // [B, N] or NULL
    int64_t mask_stride;
    int N;
    __device__ __forceinline__ int length(int b) const {
        if (lens == nullptr) return N;
        const int n = lens[b];
        return n < 0 ? 0 : n < N ? n : N;
    }
    __device__ __forceinline__ const uint8_t* row(int b) const { return mask == nullptr ? nullptr : mask + b * mask_stride; }
};

// Work item of a workgroup such that consecutive items run on the same XCD (workgroups go to the 8 XCDs in turn): the row
// blocks of a unit then share its K and V in one L2. The grid is 8 * ceil(items / 8); false: nothing to do.
__device__ __forceinline__ bool xcd_item(unsigned items, unsigned& item) {
    const unsigned per = (items + 7) / 8;
    item = (blockIdx.x & 7u) * per + (blockIdx.x >> 3);
    return (blockIdx.x >> 3) < per && item < items;
}
inline unsigned xcd_grid(unsigned items) { return 8u * ((items + 7) / 8); }

// One 32 x D result of a wave (columns = rows of the output, results = its elements) to memory in whole 16-byte chunks,
// through `buf` (32 rows of DP + 8 elements, the wave's own). at(row): pointer to the output row or NULL.
template <int DT, int DP, typename At>
__device__ __forceinline__ void store_tile(const v16f (&acc)[DP / 32], float scale, uint16_t* buf, int D, int lane, At at) {
    constexpr int LB = DP + 8, CPR = DP / 8;
    uint16_t* mine = buf + (lane & 31) * LB + ((lane >> 5) << 2);
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<v2i*>(mine + t * 32 + i * 8) = v2i{(int)pack2<DT>(acc[t][4 * i] * scale, acc[t][4 * i + 1] * scale),
                                                                 (int)pack2<DT>(acc[t][4 * i + 2] * scale, acc[t][4 * i + 3] * scale)};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = 0; c < 32 * CPR / 64; ++c) {
        const int i = lane + c * 64, row = i / CPR, e = (i - row * CPR) * 8;
        uint16_t* p = at(row);
        if (p != nullptr && e < D) *reinterpret_cast<v4u*>(p + e) = *reinterpret_cast<const v4u*>(buf + row * LB + e);
    }
}

// ---- host side ---------------------------------------------------------------------------------------------

// strides of a [B, heads, tokens, D] tensor: 0 or more (outputs: as given by the caller, not checked for overlap), multiples
// of 8 elements where there is more than one index, offsets that fit; base 16-byte aligned
inline int x_tensor(const char* who, const char* name, const void* p, const int64_t* s, int64_t b, int64_t h, int64_t t, int D) {
    if (p == nullptr || s == nullptr) return fail(Q8_ERR_NULL, "%s: %s is NULL", who, name);
    const int64_t n[3] = {b, h, t};
    __int128 e = D;
    for (int i = 0; i < 3; ++i) {
        if (n[i] <= 1) continue;
        if (s[i] < 0) return fail(Q8_ERR_SHAPE, "%s: negative stride of %s", who, name);
        if (s[i] % 8) return fail(Q8_ERR_ALIGN, "%s: strides of %s must be multiples of 8 elements", who, name);
        e += (__int128)(n[i] - 1) * s[i];
    }
    if (e > (INT64_MAX >> 4)) return fail(Q8_ERR_SHAPE, "%s: strides of %s", who, name);
    if (!aligned16(p)) return fail(Q8_ERR_ALIGN, "%s: %s must be 16-byte aligned", who, name);
    return Q8_OK;
}

inline int x_sizes(const char* who, int dt, int64_t B, int H, int Hkv, int M, int N, int D, float scale) {
    if (dt != Q8_BF16 && dt != Q8_F16) return fail(Q8_ERR_DTYPE, "%s: element type %d (bf16 or fp16)", who, dt);
    if (B < 0 || H < 1 || Hkv < 1 || M < 0 || N < 0) return fail(Q8_ERR_SHAPE, "%s: B %lld, heads %d and %d, M %d, N %d", who, (long long)B, H, Hkv, M, N);
    if (H % Hkv) return fail(Q8_ERR_SHAPE, "%s: %d query heads on %d key heads (a multiple is needed)", who, H, Hkv);
    if (D < 8 || D > 128 || D % 8) return fail(Q8_ERR_SHAPE, "%s: head dim %d (a multiple of 8 up to 128)", who, D);
    if (!(scale > 0.f) || scale > 3e38f) return fail(Q8_ERR_SHAPE, "%s: softmax scale %g (positive and finite)", who, (double)scale);
    // rows, units and the fp32 scratch stay in 32-bit counts
    if ((int64_t)(H / Hkv) * M > 0x3fffffff || N > 0x3fffffff || (B && (int64_t)Hkv > 0x3fffffff / B) ||
        (B && M && (int64_t)H > ((int64_t)1 << 40) / B / M))
        return fail(Q8_ERR_SHAPE, "%s: sizes out of range", who);
    return Q8_OK;
}

inline int padded_head(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

}  // namespace q8
