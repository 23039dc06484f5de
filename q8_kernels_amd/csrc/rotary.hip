// Rotary positions from the positions and the frequencies themselves, for queries and keys in one launch.
//
// Pair i of a head at position p turns by the angle a = p f_i: (u, v) -> factor (u cos a - v sin a, v cos a + u sin a); the
// backward is the transposed rotation, the same with -sin. u, v are elements (i, i + R/2) of the head (half layout) or
// (2 i, 2 i + 1) (interleaved); elements from the rotary dimension R on are copied.
//
// HBM-bound: every head is read and written once. The angles are formed here instead of being read from a table: p * f_i
// in fp64, whose whole turns are dropped there; the rest goes to the fp32 sine and cosine as two fp32 numbers, the second to first
// order, so a far position's are as exact as a near one's, and no table limits the positions. fp32 results are 1.6 roundings off in
// the square mean, as with tables from fp64 (of one fp32 number of turns: 2.1). A workgroup forms the R / 2 angles of
// its tokens once, in LDS, and all heads of those tokens use them. bf16, 2 x 6144 tokens, 32 + 32 heads of 64: 38 to 39 us for
// 201 MB (5.2 TB/s; a large copy 5.1), 16 single tokens of 32 + 8 heads of 128 4.5 us, which is the launch.
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

// A work item's elements as they are in memory: VEC of them from one place, or from two for the pairs of the half layout, in
// accesses of 16 bytes (8 bytes for 4 16-bit elements, an element for VEC = 1).
template <int DT, int VEC>
struct RotPart {
    static constexpr int N = VEC == 1 ? 1 : DT == Q8_F32 ? VEC : VEC / 2, CHUNK = N < 4 ? N : 4;
    typedef uint32_t Words __attribute__((ext_vector_type(CHUNK > 1 ? CHUNK : 2)));
    uint32_t r[N];
    __device__ __forceinline__ void load(const void* p, int64_t e) {
        if constexpr (VEC == 1) {
            r[0] = DT == Q8_F32 ? static_cast<const uint32_t*>(p)[e] : static_cast<const uint16_t*>(p)[e];
        } else {
            const Words* s = reinterpret_cast<const Words*>(static_cast<const char*>(p) + e * (DT == Q8_F32 ? 4 : 2));
#pragma unroll
            for (int q = 0; q < N / CHUNK; ++q) {
                const Words w = s[q];
#pragma unroll
                for (int i = 0; i < CHUNK; ++i) r[q * CHUNK + i] = w[i];
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (DT == Q8_F32) return __uint_as_float(r[i]);
        const uint32_t h = VEC == 1 ? r[0] : i & 1 ? r[i >> 1] >> 16 : r[i >> 1] & 0xffffu;
        return DT == Q8_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
    }
    __device__ __forceinline__ void set(const float (&v)[VEC]) {
        if constexpr (VEC == 1) {
            r[0] = DT == Q8_F32 ? __float_as_uint(v[0]) : DT == Q8_BF16 ? pack2_bf16(v[0], 0.f) & 0xffffu : __builtin_bit_cast(uint16_t, (_Float16)v[0]);
        } else if constexpr (DT == Q8_F32) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) r[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                r[i] = DT == Q8_BF16 ? pack2_bf16(v[2 * i], v[2 * i + 1])
                                     : __builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16);
        }
    }
    __device__ __forceinline__ void store(void* p, int64_t e) const {
        if constexpr (VEC == 1) {
            if constexpr (DT == Q8_F32) static_cast<uint32_t*>(p)[e] = r[0];
            else static_cast<uint16_t*>(p)[e] = (uint16_t)r[0];
        } else {
            Words* s = reinterpret_cast<Words*>(static_cast<char*>(p) + e * (DT == Q8_F32 ? 4 : 2));
#pragma unroll
            for (int q = 0; q < N / CHUNK; ++q) {
                Words w;
#pragma unroll
                for (int i = 0; i < CHUNK; ++i) w[i] = r[q * CHUNK + i];
                s[q] = w;
            }
        }
    }
};

// One work item of a head: VEC pairs (half) / VEC / 2 pairs (interleaved) or VEC copied elements; VEC = 1: one pair or one copied
// element. Threads with the same threadIdx / items share a head; a thread has BATCH items
// under way at once, the first of them requested before the angles are formed.
template <int DT, bool HALF, int VEC>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotArgs a) {
    constexpr int BATCH = 4, PAIRS = VEC == 1 ? 1 : (HALF ? VEC : VEC / 2);  // pairs of an item
    constexpr bool TWO = HALF || VEC == 1;                          // a pair's elements come from two places
    __shared__ float2 cs[kRotAngles];
    const int64_t token0 = (int64_t)blockIdx.x * a.per_block;
    const int here = (int)(a.all_tokens - token0 < a.per_block ? a.all_tokens - token0 : a.per_block);
    const int64_t b0 = token0 / a.tokens, t0 = token0 - b0 * a.tokens;
    // batch element and token of the workgroup's token tok (of fewer than 64)
    auto place = [&](int tok, int64_t& b, int64_t& t) {
        b = b0;
        t = t0 + tok;
        if (a.tokens >= 64) {
            if (t >= a.tokens) { t -= a.tokens; ++b; }
        } else {
            const unsigned n = (unsigned)t / (unsigned)a.tokens;
            b += n;
            t -= (int64_t)n * a.tokens;
        }
    };
    const int rot_items = a.pairs / PAIRS, items = rot_items + (a.dim - 2 * a.pairs) / VEC;
    const int lanes = kRotThreads / items > 0 ? kRotThreads / items : 1;  // heads in flight
    const int dtok = lanes / a.heads, dhead = lanes - dtok * a.heads;

    struct Item {
        RotPart<DT, VEC> u, v;
        void* out;
        int64_t to;
        int tok;
    } x[BATCH];
    int item = items <= kRotThreads ? (int)threadIdx.x % items : (int)threadIdx.x;
    const int lane = items <= kRotThreads ? (int)threadIdx.x / items : 0;
    int tok = here, head = 0;  // a thread without a head, or with no item, has no token
    auto begin = [&] {
        if (lane < lanes && item < items) {
            tok = lane / a.heads;
            head = lane - tok * a.heads;
        } else {
            tok = here;
        }
    };
    // element offsets of the item's first and second place in a head
    auto places = [&](int& eu, int& ev) {
        if (item >= rot_items) eu = ev = 2 * a.pairs + (item - rot_items) * VEC;
        else if (VEC == 1) { eu = HALF ? item : 2 * item; ev = HALF ? item + a.pairs : 2 * item + 1; }
        else { eu = item * VEC; ev = HALF ? a.pairs + item * VEC : eu; }
    };
    auto request = [&] {
        int eu, ev;
        places(eu, ev);
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            x[k].tok = tok;
            if (tok < here) {
                int64_t b, t;
                place(tok, b, t);
                const bool is_q = head < a.q_heads;
                const int h = is_q ? head : head - a.q_heads;
                const RotTensor& y = is_q ? a.q : a.k;
                const int64_t in = b * y.ib + h * y.ih + t * y.it;
                x[k].out = y.out;
                x[k].to = b * y.ob + h * y.oh + t * y.ot;
                x[k].u.load(y.in, in + eu);
                if (TWO && item < rot_items) x[k].v.load(y.in, in + ev);
            }
            tok += dtok;
            head += dhead;
            if (head >= a.heads) { head -= a.heads; ++tok; }
        }
    };
    auto finish = [&] {
        int eu, ev;
        places(eu, ev);
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            if (x[k].tok >= here) continue;
            if (item < rot_items) {
                const float2* w = cs + x[k].tok * a.pairs + item * PAIRS;
                if constexpr (TWO) {
                    float ou[VEC], ov[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float u = x[k].u.get(i), v = x[k].v.get(i);
                        ou[i] = u * w[i].x - v * w[i].y;
                        ov[i] = v * w[i].x + u * w[i].y;
                    }
                    x[k].u.set(ou);
                    x[k].v.set(ov);
                    x[k].v.store(x[k].out, x[k].to + ev);
                } else {
                    float o[VEC];
#pragma unroll
                    for (int i = 0; i < VEC / 2; ++i) {
                        const float u = x[k].u.get(2 * i), v = x[k].u.get(2 * i + 1);
                        o[2 * i] = u * w[i].x - v * w[i].y;
                        o[2 * i + 1] = v * w[i].x + u * w[i].y;
                    }
                    x[k].u.set(o);
                }
            }
            x[k].u.store(x[k].out, x[k].to + eu);
        }
    };

    begin();
    request();
    for (int i = threadIdx.x; i < here * a.pairs; i += kRotThreads) {
        const int n = i / a.pairs, pr = i - n * a.pairs;
        int64_t b, t;
        place(n, b, t);
        int64_t p = t;
        if (a.positions != nullptr) {
            const int64_t at = b * a.pos_stride + t;
            p = a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
        }
        // whole turns leave the angle by two fused steps, 2 pi = hi + lo: exact to the fp64 rounding of the angle itself
        const double angle = (double)p * a.inv_freq[pr], whole = __builtin_rint(angle * 0.15915494309189533577);
        const double left = __builtin_fma(-whole, 2.4492935982947064e-16, __builtin_fma(-whole, 6.2831853071795865, angle));
        // the rest in half turns, in fp32, and by how much that is off (in radians, below 2^-23): turned on by it to first order
        const double half_turns = left * 0.31830988618379067154;
        const float rest = (float)half_turns, more = (float)((half_turns - (double)rest) * 3.1415926535897932385);
        float s0, c0;
        sincospif(rest, &s0, &c0);
        const float s = __builtin_fmaf(more, c0, s0), c = __builtin_fmaf(-more, s0, c0);
        cs[i] = make_float2(c * a.factor, s * a.factor * a.sign);
    }
    __syncthreads();
    for (;;) {
        finish();
        if (tok >= here) {  // the next item, where a head has more of them than there are threads
            item += kRotThreads;
            if (item >= items) break;
            begin();
        }
        request();
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
    // The elements of an item: 8, or 4 where the pairs' second halves or the strides are not multiples of 8 (fp16, 10183 tokens of
    // 10 heads of 48, 24 elements of them turned in the half layout: 10.0 us, by single elements 20.6), else one.
    auto fits = [&](int n) { return dim % n == 0 && rotary_dim % (half ? 2 * n : n) == 0; };
    int vec = fits(8) ? 8 : fits(4) ? 4 : 1;
    const struct { const void* in; void* out; const int64_t *is, *os; int heads; RotTensor* to; } side[2] = {
        {q, q_out, q_strides, q_out_strides, q_heads, &a.q}, {k, k_out, k_strides, k_out_strides, k_heads, &a.k}};
    for (const auto& s : side) {
        if (!s.heads) continue;
        if (rot_extent(batch, s.heads, tokens, dim, s.is) < 0 || rot_extent(batch, s.heads, tokens, dim, s.os) < 0)
            return fail(Q8_ERR_SHAPE, "q8_rotary: strides (0 or more, offsets below 2^59)");
        if ((reinterpret_cast<uintptr_t>(s.in) | reinterpret_cast<uintptr_t>(s.out)) & (uintptr_t)(size - 1)) return fail(Q8_ERR_ALIGN, "q8_rotary: tensor not aligned to its element type");
        *s.to = RotTensor{s.in, s.out, s.is[0], s.is[1], s.is[2], s.os[0], s.os[1], s.os[2]};
        const auto goes = [&](int n) {
            const uintptr_t bytes = n * size < 16 ? n * size : 16;
            bool ok = ((reinterpret_cast<uintptr_t>(s.in) | reinterpret_cast<uintptr_t>(s.out)) & (bytes - 1)) == 0;
            for (int i = 0; i < 3; ++i) ok = ok && s.is[i] % n == 0 && s.os[i] % n == 0;
            return ok;
        };
        if (vec == 8 && !goes(8)) vec = fits(4) ? 4 : 1;
        if (vec == 4 && !goes(4)) vec = 1;
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
    // tokens of a workgroup (63 at most): about 2048 items of 8 elements (2 x 4099 tokens of 40 heads of 128: 38.1 us; 1024 items
    // 42.0, 4096 38.0; of 2 x 6144 and 64 heads of 64 38.2, 38.5, 39.6), while 1024 workgroups remain (10183 tokens of 10 heads of 48:
    // 10.0 us; 256 workgroups 14.4) and the angles fit
    const int64_t per_token = (int64_t)a.heads * ((dim + 7) / 8);
    int64_t per = 2048 / per_token;
    if (per > all / 1024) per = all / 1024;
    if (per > 63) per = 63;
    if (per > kRotAngles / a.pairs) per = kRotAngles / a.pairs;
    a.per_block = per < 1 ? 1 : (int)per;
    const int64_t blocks = (all + a.per_block - 1) / a.per_block;
    if (blocks > most_blocks(kRotThreads)) return fail(Q8_ERR_SHAPE, "q8_rotary: too many tokens");
    hipStream_t s = static_cast<hipStream_t>(stream);
#define ROT_VEC(DT, HALF)                                                                                   \
    do {                                                                                                    \
        if (vec == 8) rotary_kernel<DT, HALF, 8><<<(unsigned)blocks, kRotThreads, 0, s>>>(a);               \
        else if (vec == 4) rotary_kernel<DT, HALF, 4><<<(unsigned)blocks, kRotThreads, 0, s>>>(a);          \
        else rotary_kernel<DT, HALF, 1><<<(unsigned)blocks, kRotThreads, 0, s>>>(a);                        \
    } while (0)
#define ROT(DT)                                                                                             \
    do {                                                                                                    \
        if (half) ROT_VEC(DT, true);                                                                        \
        else ROT_VEC(DT, false);                                                                            \
    } while (0)
    if (dt == Q8_BF16) ROT(Q8_BF16);
    else if (dt == Q8_F16) ROT(Q8_F16);
    else ROT(Q8_F32);
#undef ROT
#undef ROT_VEC
    return launch_status("q8_rotary");
}
