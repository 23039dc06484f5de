// Rotary positions from the positions and the frequencies themselves, for queries and keys in one launch.
//
// Pair i of a head at position p turns by the angle a = p f_i: (u, v) -> factor (u cos a - v sin a, v cos a + u sin a); the
// backward is the transposed rotation, the same with -sin. u, v are elements (i, i + R/2) of the head (half layout) or
// (2 i, 2 i + 1) (interleaved); elements from the rotary dimension R on are copied.
//
// HBM-bound: every head is read and written once. The angles are formed here instead of being read from a table: p * f_i
// in fp64, whose whole turns are dropped there before the fp32 sine and cosine of the rest, so a far position is as exact as
// its fp64 angle, and no table limits the positions. A workgroup forms the R / 2 angles of
// its tokens once, in LDS, and all heads of those tokens use them.
#include "q8_common.h"
#include "q8_host.h"

namespace q8 {

constexpr int kRotThreads = 256;
constexpr int kRotMaxDim = 512;        // elements of a head
constexpr int kRotAngles = 1024;       // angles of a workgroup's tokens (8 KiB of LDS)

struct RotTensor {
    const void* in;
    void* out;
    int64_t ib, ih, it, ob, oh, ot;  // element strides of batch, head, token
};

struct RotArgs {
    RotTensor q, k;
    const void* positions;    // int32 or int64, or NULL: 0 .. tokens - 1
    int64_t pos_stride;       // elements between batch rows (0: one row for all)
    const double* inv_freq;   // [R / 2], radians per position
    float factor, sign;
    int pos64, q_heads, heads, dim, pairs;
    int64_t tokens, all_tokens;
    int per_block;            // tokens of a workgroup
};

template <int DT>
__device__ __forceinline__ float rot_get(const void* p, int64_t e) {
    if constexpr (DT == Q8_F32) return static_cast<const float*>(p)[e];
    const uint32_t h = static_cast<const uint16_t*>(p)[e];
    return DT == Q8_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}
template <int DT>
__device__ __forceinline__ void rot_put(void* p, int64_t e, float v) {
    if constexpr (DT == Q8_F32) static_cast<float*>(p)[e] = v;
    else static_cast<uint16_t*>(p)[e] = DT == Q8_BF16 ? (uint16_t)(pack2_bf16(v, 0.f) & 0xffffu) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <int DT>
__device__ __forceinline__ void rot_store8(void* p, int64_t e, const float (&v)[8]) {
    if constexpr (DT == Q8_F32) {
        v4f* s = reinterpret_cast<v4f*>(static_cast<float*>(p) + e);
        s[0] = v4f{v[0], v[1], v[2], v[3]};
        s[1] = v4f{v[4], v[5], v[6], v[7]};
    } else {
        v4u w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = DT == Q8_BF16 ? pack2_bf16(v[2 * i], v[2 * i + 1])
                                 : __builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16);
        *reinterpret_cast<v4u*>(static_cast<uint16_t*>(p) + e) = w;
    }
}

// One work item of a head: VEC = 8: 8 pairs (half) / 4 pairs (interleaved) or 8 copied elements, in 16-byte accesses;
// VEC = 1: one pair or one copied element. Threads with the same threadIdx / items share a head.
template <int DT, bool HALF, int VEC>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs a) {
    __shared__ float2 cs[kRotAngles];
    const int64_t token0 = (int64_t)blockIdx.x * a.per_block;
    const int here = (int)(a.all_tokens - token0 < a.per_block ? a.all_tokens - token0 : a.per_block);
    for (int i = threadIdx.x; i < here * a.pairs; i += kRotThreads) {
        const int tok = i / a.pairs, pr = i - tok * a.pairs;
        const int64_t g = token0 + tok, b = g / a.tokens, t = g - b * a.tokens;
        int64_t p = t;
        if (a.positions != nullptr) {
            const int64_t at = b * a.pos_stride + t;
            p = a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
        }
        // whole turns leave the angle by two fused steps, 2 pi = hi + lo: exact to the fp64 rounding of the angle itself
        const double angle = (double)p * a.inv_freq[pr], whole = __builtin_rint(angle * 0.15915494309189533577);
        const double left = __builtin_fma(-whole, 2.4492935982947064e-16, __builtin_fma(-whole, 6.2831853071795865, angle));
        const float rest = (float)(left * 0.15915494309189533577);
        float s, c;
        sincospif(2.0f * rest, &s, &c);
        cs[i] = make_float2(c * a.factor, s * a.factor * a.sign);
    }
    __syncthreads();
    constexpr int PAIRS = VEC == 1 ? 1 : (HALF ? 8 : 4);  // pairs of an item
    const int rot_items = a.pairs / PAIRS, items = rot_items + (a.dim - 2 * a.pairs) / VEC;
    const int lanes = kRotThreads / items > 0 ? kRotThreads / items : 1;  // heads in flight
    const int item0 = items <= kRotThreads ? (int)threadIdx.x % items : (int)threadIdx.x;
    const int lane = items <= kRotThreads ? (int)threadIdx.x / items : 0;
    if (lane >= lanes) return;
    for (int item = item0; item < items; item += kRotThreads) {  // (one turn unless a head has more items than there are threads)
        int tok = lane / a.heads, head = lane - tok * a.heads;
        const int dtok = lanes / a.heads, dhead = lanes - dtok * a.heads;
        while (tok < here) {
            const int64_t g = token0 + tok, b = g / a.tokens, t = g - b * a.tokens;
            const bool is_q = head < a.q_heads;
            const int h = is_q ? head : head - a.q_heads;
            const RotTensor& x = is_q ? a.q : a.k;
            const int64_t in = b * x.ib + h * x.ih + t * x.it, out = b * x.ob + h * x.oh + t * x.ot;
            if (item < rot_items) {
                const float2* w = cs + tok * a.pairs + item * PAIRS;
                if constexpr (VEC == 1) {
                    const int eu = HALF ? item : 2 * item, ev = HALF ? item + a.pairs : 2 * item + 1;
                    const float u = rot_get<DT>(x.in, in + eu), v = rot_get<DT>(x.in, in + ev);
                    rot_put<DT>(x.out, out + eu, u * w[0].x - v * w[0].y);
                    rot_put<DT>(x.out, out + ev, v * w[0].x + u * w[0].y);
                } else if constexpr (HALF) {
                    float u[8], v[8], ou[8], ov[8];
                    load8<DT>(x.in, in + item * 8, u);
                    load8<DT>(x.in, in + a.pairs + item * 8, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        ou[i] = u[i] * w[i].x - v[i] * w[i].y;
                        ov[i] = v[i] * w[i].x + u[i] * w[i].y;
                    }
                    rot_store8<DT>(x.out, out + item * 8, ou);
                    rot_store8<DT>(x.out, out + a.pairs + item * 8, ov);
                } else {
                    float u[8], o[8];
                    load8<DT>(x.in, in + item * 8, u);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[2 * i] = u[2 * i] * w[i].x - u[2 * i + 1] * w[i].y;
                        o[2 * i + 1] = u[2 * i + 1] * w[i].x + u[2 * i] * w[i].y;
                    }
                    rot_store8<DT>(x.out, out + item * 8, o);
                }
            } else {
                const int e = 2 * a.pairs + (item - rot_items) * VEC;
                if constexpr (VEC == 1) {
                    rot_put<DT>(x.out, out + e, rot_get<DT>(x.in, in + e));
                } else {
                    float u[8];
                    load8<DT>(x.in, in + e, u);
                    rot_store8<DT>(x.out, out + e, u);
                }
            }
            tok += dtok;
            head += dhead;
            if (head >= a.heads) { head -= a.heads; ++tok; }
        }
    }
}

// largest element offset of a [B, heads, tokens, dim] tensor with these strides; negative: not representable or a negative stride
static int64_t rot_extent(int64_t b, int64_t h, int64_t t, int dim, const int64_t* s) {
    const int64_t n[3] = {b, h, t};
    __int128 e = dim;
    for (int i = 0; i < 3; ++i) {
        if (s[i] < 0) return -1;
        e += (__int128)(n[i] - 1) * s[i];
    }
    return e > (INT64_MAX >> 4) ? -1 : (int64_t)e;
}

}  // namespace q8

using namespace q8;

extern "C" int q8_rotary(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int q_heads, const void* k,
                         const int64_t* k_strides, void* k_out, const int64_t* k_out_strides, int k_heads, int dt, const void* positions, int pos_bits,
                         int64_t pos_row_stride, const double* inv_freq, int rotary_dim, int half_layout, float factor, int backward, int64_t batch,
                         int64_t tokens, int dim, q8_stream_t stream) {
    if (dt != Q8_BF16 && dt != Q8_F16 && dt != Q8_F32) return fail(Q8_ERR_DTYPE, "q8_rotary: element type %d (bf16, fp16 or fp32)", dt);
    if (batch < 0 || tokens < 0 || q_heads < 0 || k_heads < 0 || q_heads > 65536 || k_heads > 65536 || dim < 1 || dim > kRotMaxDim)
        return fail(Q8_ERR_SHAPE, "q8_rotary: batch %lld, tokens %lld, heads %d and %d, head size %d (1 .. %d)", (long long)batch, (long long)tokens, q_heads,
                    k_heads, dim, kRotMaxDim);
    if (rotary_dim < 2 || rotary_dim > dim || rotary_dim % 2) return fail(Q8_ERR_SHAPE, "q8_rotary: rotary size %d of a head of %d (even, 2 or more)", rotary_dim, dim);
    if (tokens && batch > ((int64_t)1 << 40) / tokens) return fail(Q8_ERR_SHAPE, "q8_rotary: too many tokens");
    const int64_t all = batch * tokens;
    if (all == 0 || q_heads + k_heads == 0) return Q8_OK;
    if ((q_heads && (!q || !q_out || !q_strides || !q_out_strides)) || (k_heads && (!k || !k_out || !k_strides || !k_out_strides)) || !inv_freq)
        return fail(Q8_ERR_NULL, "q8_rotary: null pointer");
    if (positions && pos_bits != 32 && pos_bits != 64) return fail(Q8_ERR_DTYPE, "q8_rotary: positions of %d bits (32 or 64)", pos_bits);
    if (positions && (pos_row_stride < 0 || (pos_row_stride && pos_row_stride < tokens) || (batch > 1 && pos_row_stride > INT64_MAX / 16 / batch)))
        return fail(Q8_ERR_SHAPE, "q8_rotary: row stride %lld of the positions", (long long)pos_row_stride);
    RotArgs a{};
    const int size = elem_size(dt), half = half_layout != 0;
    const int need = 8;  // elements of a 16- or 32-byte access
    bool vec = dim % 8 == 0 && rotary_dim % (half ? 16 : 8) == 0;
    const struct { const void* in; void* out; const int64_t *is, *os; int heads; RotTensor* to; } side[2] = {
        {q, q_out, q_strides, q_out_strides, q_heads, &a.q}, {k, k_out, k_strides, k_out_strides, k_heads, &a.k}};
    for (const auto& s : side) {
        if (!s.heads) continue;
        if (rot_extent(batch, s.heads, tokens, dim, s.is) < 0 || rot_extent(batch, s.heads, tokens, dim, s.os) < 0)
            return fail(Q8_ERR_SHAPE, "q8_rotary: strides (0 or more, offsets below 2^59)");
        if ((reinterpret_cast<uintptr_t>(s.in) | reinterpret_cast<uintptr_t>(s.out)) & (uintptr_t)(size - 1)) return fail(Q8_ERR_ALIGN, "q8_rotary: tensor not aligned to its element type");
        *s.to = RotTensor{s.in, s.out, s.is[0], s.is[1], s.is[2], s.os[0], s.os[1], s.os[2]};
        vec = vec && aligned16(s.in) && aligned16(s.out);
        for (int i = 0; i < 3; ++i) vec = vec && s.is[i] % need == 0 && s.os[i] % need == 0;
    }
    if ((reinterpret_cast<uintptr_t>(inv_freq) & 7) || (positions && (reinterpret_cast<uintptr_t>(positions) & (uintptr_t)(pos_bits / 8 - 1))))
        return fail(Q8_ERR_ALIGN, "q8_rotary: positions or frequencies not aligned");
    a.positions = positions;
    a.pos64 = pos_bits == 64;
    a.pos_stride = pos_row_stride;
    a.inv_freq = inv_freq;
    a.factor = factor;
    a.sign = backward ? -1.f : 1.f;
    a.q_heads = q_heads;
    a.heads = q_heads + k_heads;
    a.dim = dim;
    a.pairs = rotary_dim / 2;
    a.tokens = tokens;
    a.all_tokens = all;
    // tokens of a workgroup: about 2048 items of 8 elements, while 1024 workgroups remain and the angles fit
    const int64_t per_token = (int64_t)a.heads * ((dim + 7) / 8);
    int64_t per = 2048 / per_token;
    if (per > all / 1024) per = all / 1024;
    if (per > kRotAngles / a.pairs) per = kRotAngles / a.pairs;
    a.per_block = per < 1 ? 1 : (int)per;
    const int64_t blocks = (all + a.per_block - 1) / a.per_block;
    if (blocks > 0x7fffffff) return fail(Q8_ERR_SHAPE, "q8_rotary: too many tokens");
    hipStream_t s = static_cast<hipStream_t>(stream);
#define ROT(DT)                                                                                             \
    do {                                                                                                    \
        if (vec && half) rotary_kernel<DT, true, 8><<<(unsigned)blocks, kRotThreads, 0, s>>>(a);            \
        else if (vec) rotary_kernel<DT, false, 8><<<(unsigned)blocks, kRotThreads, 0, s>>>(a);              \
        else if (half) rotary_kernel<DT, true, 1><<<(unsigned)blocks, kRotThreads, 0, s>>>(a);              \
        else rotary_kernel<DT, false, 1><<<(unsigned)blocks, kRotThreads, 0, s>>>(a);                       \
    } while (0)
    if (dt == Q8_BF16) ROT(Q8_BF16);
    else if (dt == Q8_F16) ROT(Q8_F16);
    else ROT(Q8_F32);
#undef ROT
    return launch_status("q8_rotary");
}
