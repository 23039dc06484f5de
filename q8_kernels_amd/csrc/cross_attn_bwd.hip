// 16-bit cross attention, backward. With P = exp2(c S - lse) formed again from Q, K and the forward's log-sums:
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),  delta = rowsum(dO O),  dQ = scale dS K,  dK = scale dS^T Q
//
// Up to 128 keys (or 256, with many rows) a kernel of its own holds all of them, see there. Otherwise:
//
// Two kernels, so that every sum has one owner and a fixed order (no atomics), at the price of forming S and dP twice (seven
// products instead of five; partial sums of dQ per key tile would move more time's worth of bytes than the two products
// cost). The first owns 128 query rows and walks over the keys: it forms delta, writes it for the second, and dQ. The second
// owns 128 keys and walks over the rows of all query heads of the group, so dK and dV of a shared head come out summed. P and
// dS are rounded to 16 bits for the products they enter (P in fp16 times 2^14, which is taken off dV); scores, dP, sums and delta
// are fp32.
//
// fp16 holds neither the dS of small gradients (of 1e-3 with 2048 keys they are below 2^-14) nor those of scaled ones (above
// 65504). There dS enters its products times a power of two, which is taken off the fp32 sums. In the two kernels every
// column of a block has its own, a row of dQ or a key of dK: the largest |dS| of a block is looked at, and where it goes above
// 2^15 the power is lowered so that it comes to 2^9, with the sums so far (as the forward does with its maximum). The kernel for
// few keys has one for a tile, from a bound: |dS| <= |dO_i| max_j |V_j| / 2, for p (1 - p) is 1/4 at most.
//
// A key that does not count: in the first kernel its score is -infinity (P = 0 exactly, whatever lse is) and its rows of K
// and V are zeros; in the second a key is a column of every product, whose garbage stays in its column, and its gradient is
// written as zeros. A row without keys has lse = +infinity, which makes its P zero everywhere.
//
// delta's error is that of every score's gradient in the row. It is formed from the forward's O with 8 bits
// more than its result has, normalised by the sum of the rounded P: what is left of the error is sum_j r_j dS_j with the
// roundings r_j of the forward's P. To the 1.4 roundings that dS and the result cost it adds nothing with many keys and at most
// 0.2 with few (from the rounded O alone dQ is 2.0 off with 512 keys and scores of deviation 4, 6.1 with a mean of 3 in V as well,
// 2.3 with 2 keys). Up to kXExact keys, which one wave or one score tile holds, that goes too: the dS of a row are summed before they
// are rounded; the true ones add up to zero, so the sum is the error, and it is taken off.
//
// Few workgroups: the walk is divided over several of them, their fp32 sums are added by a third kernel in order.
#include "cross_attn_common.h"

#include <type_traits>

namespace q8 {

constexpr int kXExact = 32;
template <int DT>
constexpr float kUnshiftP = 1.0f / (1 << kShiftP<DT>);
constexpr int kMostShift = 60;  // log2 of the largest factor of dS: P |dP| below 2^39 stays finite beside it

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 .. 127

// One column of a block of dS times a power of two, in 16 results of the lanes l and l + 32: the power's change (0 or less) where
// the largest of them has grown beyond fp16's reach. NaN and infinity change nothing: their column is lost.
__device__ __forceinline__ int shift_change(const v16f& ds) {
    float top = max_ieee(__builtin_fabsf(ds[0]), __builtin_fabsf(ds[1]));
#pragma unroll
    for (int i = 2; i < 16; ++i) top = max_ieee(top, __builtin_fabsf(ds[i]));
    top = half_pair_max(top);
    const int to = 9 - __builtin_amdgcn_frexp_expf(top);
    return top > 32768.f && to < 0 ? to : 0;
}
template <int N>
__device__ __forceinline__ void scale_all(v16f (&x)[N], float f) {
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[t][i] *= f;
}

// d + sum of g o over 8 elements, o with its rest
template <int DT>
__device__ __forceinline__ float dot_sum(v4u g, v4u o, v2i low, float d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        d += unpack<DT>(g[i] & 0xffffu) * with_rest<DT>(o[i] & 0xffffu, (uint32_t)low[i / 2], i % 2 * 2);
        d += unpack<DT>(g[i] >> 16) * with_rest<DT>(o[i] >> 16, (uint32_t)low[i / 2], i % 2 * 2 + 1);
    }
    return d;
}

struct XBwd {
    XTensor q, k, v, o, g;
    const uint8_t* o_low;   // [units, R, D]: what the rounding of O left off
    XOut dq, dk, dv;
    const float* lse;    // [units, R]
    float* delta;        // [units, R], workspace
    XKeys keys;
    float c, scale;
    int Hkv, G, M, N, D, R;
    int blocks;          // of 128 rows (second kernel: keys) in a unit
    XSchedule plan;
    float* part;         // divided blocks: [splits, tail, 128, D], or [splits, tail, 128, 2 D] (dK, dV)
};

// 2 x 16 heads of 128 on 4, 4096 x 4096: bf16 380 to 393 us (three products, 1050 to 1090 TFLOP/s), fp16 415; operands in groups of 2:
// with groups of 4, as in the forward, 27 registers are spilled and it takes 432 to 440. Heads up to 64 fit three waves on a SIMD.
template <int DT, int DP>
__global__ __launch_bounds__(kXThreads, DP <= 64 ? 3 : 2) void cross_attn_dq_kernel(XBwd a) {
    constexpr int KS = DP / 16, DTL = DP / 32, ELEMS = kXTile * DP;
    __shared__ __align__(16) uint16_t k0[ELEMS], k1[ELEMS], v0[ELEMS], v1[ELEMS];
    __shared__ __align__(16) float bias0[kXTile], bias1[kXTile];
    unsigned block;
    int split, of;
    if (!a.plan.item(block, split, of)) return;
    const int unit = block / a.blocks, rb = block - unit * a.blocks;
    const int b = unit / a.Hkv, hk = unit - b * a.Hkv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int row0 = (rb * kXWaves + wave) * 32, row = row0 + (lane & 31);

    KVTiles<DP> kv;
    kv.len = a.keys.length(b);
    kv.mask = a.keys.row(b);
    kv.copies.D = a.D;
    kv.kp = a.k.p + b * a.k.sb + hk * a.k.sh;
    kv.vp = a.v.p + b * a.v.sb + hk * a.v.sh;
    kv.kst = a.k.st;
    kv.vst = a.v.st;
    kv.copies.wave = wave;
    const int tiles = (kv.len + kXTile - 1) / kXTile, per = (tiles + of - 1) / of;
    const int t0 = split * per, t1 = t0 + per < tiles ? t0 + per : tiles;
    const bool few = kv.len > 0 && kv.len <= kXExact;

    v4u qf[KS], gf[KS];
    float delta = 0.f, lse = __builtin_inff();  // lse: less the power of two of the row's dS
    {
        const bool ok = row < a.R;
        const int g = ok ? row / a.M : 0, m = row - g * a.M;
        const uint16_t* qp = a.q.p + b * a.q.sb + (int64_t)(hk * a.G + g) * a.q.sh + m * a.q.st + half * 8;
        const uint16_t* gp = a.g.p + b * a.g.sb + (int64_t)(hk * a.G + g) * a.g.sh + m * a.g.st + half * 8;
        const uint16_t* op = a.o.p + b * a.o.sb + (int64_t)(hk * a.G + g) * a.o.sh + m * a.o.st + half * 8;
        const uint8_t* lp = a.o_low + ((int64_t)unit * a.R + row) * a.D + half * 8;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const bool in = ok && s * 16 + half * 8 < a.D;
            qf[s] = in ? *reinterpret_cast<const v4u*>(qp + s * 16) : v4u{0u, 0u, 0u, 0u};
            gf[s] = in ? *reinterpret_cast<const v4u*>(gp + s * 16) : v4u{0u, 0u, 0u, 0u};
            const v4u of = in ? *reinterpret_cast<const v4u*>(op + s * 16) : v4u{0u, 0u, 0u, 0u};
            const v2i lf = in ? *reinterpret_cast<const v2i*>(lp + s * 16) : v2i{0, 0};
            delta = dot_sum<DT>(gf[s], of, lf, delta);
        }
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(delta), __float_as_uint(delta), false, false);
        delta = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        if (ok) {
            const int64_t at = (int64_t)unit * a.R + row;
            lse = a.lse[at];
            if constexpr (DT == Q8_F16) lse -= kMostShift;
            if (split == 0 && half == 0 && !few) a.delta[at] = delta;
        }
    }
    if (t0 < t1) kv.first(t0, k0, v0, bias0);

    v16f acc[DTL];
#pragma unroll
    for (int t = 0; t < DTL; ++t) acc[t] = splat16(0.f);
    wait_loads();
    __syncthreads();

    LaneOffsets<DP> at(lane);
    Operands<DP, 2> ops;
    auto step = [&](int t, auto buffer) {
        constexpr int BUF = decltype(buffer)::value;
        at.fresh();
        const uint16_t *kl = BUF ? k1 : k0, *vl = BUF ? v1 : v0;
        uint16_t *kn = BUF ? k0 : k1, *vn = BUF ? v0 : v1;
        // (past the last tile of this workgroup the copies are of a tile that nobody reads, or empty)
        kv.bias_of(kv.live[1], BUF ? bias0 : bias1);
        kv.ask(t + 2);
        const XTile knext = kv.k_tile(t + 1), vnext = kv.v_tile(t + 1);
        constexpr int PARTS = 4 * ops.RN;  // groups that form scores and dP in a tile: the next tile's copies go with them
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            v16f s, dp = splat16(-delta);
            auto scores = [&](auto masked) {
                if constexpr (masked) s = bias16(BUF ? bias1 : bias0, u, half);
                else s = splat16(0.f);
                if (u == 0) ops.rows(0, kl, 0, 0, at);
#pragma unroll
                for (int g = 0; g < ops.RN; ++g) {
                    if (g + 1 < ops.RN) ops.rows((g + 1) & 1, kl, u * 32, g + 1, at);
                    else ops.rows((g + 1) & 1, vl, u * 32, 0, at);
                    kv.copies.group(u * 2 * ops.RN + g, PARTS, knext, vnext, ~kv.live[1], kn, vn);
                    fence();
#pragma unroll
                    for (int j = 0; j < ops.RG; ++j) s = mfma16<DT>(ops.f[g & 1][j], qf[g * ops.RG + j], s);
                    fence();
                }
            };
            if (kv.live[0] == ~(uint64_t)0) scores(std::false_type{});
            else scores(std::true_type{});
#pragma unroll
            for (int g = 0; g < ops.RN; ++g) {
                const int now = (ops.RN + g) & 1;
                if (g + 1 < ops.RN) ops.rows(now ^ 1, vl, u * 32, g + 1, at);
                else ops.cols(now ^ 1, kl, u * 32, 0, at);
                kv.copies.group((u * 2 + 1) * ops.RN + g, PARTS, knext, vnext, ~kv.live[1], kn, vn);
                fence();
#pragma unroll
                for (int j = 0; j < ops.RG; ++j) dp = mfma16<DT>(ops.f[now][j], gf[g * ops.RG + j], dp);
                fence();
            }
            // (2 RN groups so far: the columns are in place 0)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.c, -lse));
            if constexpr (BUF == 0) {
                if (u == 0 && few) {  // all keys are here: what their dS adds up to is the error of delta
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum += dp[i] * s[i];
                    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
                    sum = __uint_as_float(r[0]) + __uint_as_float(r[1]);
                    if constexpr (DT == Q8_F16) sum = __builtin_ldexpf(sum, -kMostShift);  // (the first block: no change so far)
#pragma unroll
                    for (int i = 0; i < 16; ++i) dp[i] -= sum;
                    if (const XBwd& z = arguments_again<XBwd>(); row < z.R && half == 0) z.delta[(int64_t)unit * z.R + row] = delta + sum;
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) dp[i] *= s[i];
            if constexpr (DT == Q8_F16) {
                const int change = shift_change(dp);
                if (__builtin_amdgcn_ballot_w64(change != 0) != 0) {
                    const float f = __builtin_ldexpf(1.0f, change);
#pragma unroll
                    for (int i = 0; i < 16; ++i) dp[i] *= f;
                    scale_all(acc, f);
                    lse -= (float)change;
                }
            }
            int w = 0;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const v4u p = pack_step<DT>(dp, k);
#pragma unroll
                for (int c = 0; c < ops.CN; ++c, w ^= 1) {
                    if (c + 1 < ops.CN) ops.cols(w ^ 1, kl, u * 32 + k * 16, c + 1, at);
                    else if (k == 0) ops.cols(w ^ 1, kl, u * 32 + 16, 0, at);
                    else if (u == 0) ops.rows(w ^ 1, kl, 32, 0, at);
                    fence();
#pragma unroll
                    for (int d = 0; d < ops.CG; ++d) acc[c * ops.CG + d] = mfma16<DT>(ops.f[w][d], p, acc[c * ops.CG + d]);
                    fence();
                }
            }
            // (an even number of groups: the next rows are in place 0)
        }
        kv.end(t);
        __syncthreads();
    };
    for (int t = t0; t < t1; t += 2) {
        step(t, std::integral_constant<int, 0>{});
        if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{});
    }
    const XBwd& z = arguments_again<XBwd>();
    if constexpr (DT == Q8_F16) {  // (where no key counts there are zeros)
        const float whole = row < z.R ? z.lse[(int64_t)unit * z.R + row] : 0.f;
        scale_all(acc, row < z.R && whole < __builtin_inff() ? __builtin_amdgcn_exp2f(lse - whole) : 1.0f);
    }
    if (of > 1) {
        if (row < z.R) {
            float* p = z.part + (((int64_t)split * z.plan.tail + (block - z.plan.full)) * kXRows + wave * 32 + (lane & 31)) * z.D;
#pragma unroll
            for (int d = 0; d < DTL; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = d * 32 + i * 8 + half * 4;
                    if (e < z.D) *reinterpret_cast<v4f*>(p + e) = v4f{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
                }
        }
        return;
    }
    const int g = row < z.R ? row / z.M : 0;
    store_rows<DT, DP>(acc, z.scale, row < z.R ? z.dq.p + b * z.dq.sb + (int64_t)(hk * z.G + g) * z.dq.sh + (row - g * z.M) * z.dq.st : nullptr, z.D, lane);
}

// A head of more than 96 leaves no registers for V beside K and the two sums (two waves a SIMD have 256 each): V stays in
// LDS, the rows are walked in tiles of 32, and the order of the instructions is the compiler's (keeping the groups apart costs
// registers that have to be spilled). 2 x 16 heads of 128 on 4, 4096 x 4096: bf16 503 to 516 us (four products, 1065 to 1090 TFLOP/s;
// an earlier build with V in registers, staged through registers and spilled, 784), fp16 557.
template <int DT, int DP>
__global__ __launch_bounds__(kXThreads, 2) void cross_attn_dkdv_kernel(XBwd a) {
    constexpr int KS = DP / 16, DTL = DP / 32;
    constexpr bool V_IN_LDS = DP > 96;
    constexpr int TR = V_IN_LDS ? 32 : 64, ELEMS = TR * DP;
    __shared__ __align__(16) uint16_t q0[ELEMS], q1[ELEMS], g0[ELEMS], g1[ELEMS], vl[V_IN_LDS ? kXRows * DP : 8];
    __shared__ __align__(16) float lse0[TR], lse1[TR], delta0[TR], delta1[TR];  // -lse and -delta of the tile's rows
    unsigned block;
    int split, of;
    if (!a.plan.item(block, split, of)) return;
    const int unit = block / a.blocks, kb = block - unit * a.blocks;
    const int b = unit / a.Hkv, hk = unit - b * a.Hkv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int key0 = (kb * kXWaves + wave) * 32, key = key0 + (lane & 31);

    const int len = a.keys.length(b);
    const uint8_t* mask = a.keys.row(b);
    const bool counts = key < len && (mask == nullptr || mask[key]);
    // tiles of one head's rows each: the last of a head may be short
    const int head_tiles = (a.M + TR - 1) / TR, tiles = a.G * head_tiles, per = (tiles + of - 1) / of;
    const int t0 = split * per;
    int t1 = t0 + per < tiles ? t0 + per : tiles;
    if (kb * kXRows >= len) t1 = t0;  // no key of this workgroup counts: zeros

    // rows go to LDS by copies, their log-sums and deltas through a register each
    float row_lse = 0.f, row_delta = 0.f;
    int rows = 0;
    const uint16_t *qp = a.q.p + b * a.q.sb + (int64_t)hk * a.G * a.q.sh, *gp = a.g.p + b * a.g.sb + (int64_t)hk * a.G * a.g.sh;
    Copies<DP, TR> copies;
    copies.wave = wave;
    copies.D = a.D;
    // the tile that is next (t past the end: empty)
    auto aim = [&](int t) {
        const int g = t / head_tiles, m = (t - g * head_tiles) * TR;
        rows = t < t1 ? a.M - m : 0;
        const int n = (int)threadIdx.x & (TR - 1);
        const int64_t at = (int64_t)unit * a.R + (rows ? g * a.M + m + (n < rows ? n : rows - 1) : 0);
        row_lse = a.lse[at];
        row_delta = a.delta[at];
    };
    auto q_tile = [&](int t) {
        const int g = t / head_tiles, m = (t - g * head_tiles) * TR;
        return XTile(qp + g * a.q.sh + m * a.q.st, a.q.st, rows, a.D, TR);
    };
    auto g_tile = [&](int t) {
        const int g = t / head_tiles, m = (t - g * head_tiles) * TR;
        return XTile(gp + g * a.g.sh + m * a.g.st, a.g.st, rows, a.D, TR);
    };
    auto finish = [&](float* lt, float* dt) {
        wait_loads();
        if (threadIdx.x < TR) {
            lt[threadIdx.x] = (int)threadIdx.x < rows ? kShiftP<DT> - row_lse : -__builtin_inff();
            dt[threadIdx.x] = (int)threadIdx.x < rows ? -row_delta : 0.f;
        }
    };

    v4u kf[KS], vf[V_IN_LDS ? 1 : KS];
    {
        const uint16_t* kp = a.k.p + b * a.k.sb + hk * a.k.sh + key * a.k.st + half * 8;
        const uint16_t* vp = a.v.p + b * a.v.sb + hk * a.v.sh + key * a.v.st + half * 8;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const bool in = counts && s * 16 + half * 8 < a.D;
            kf[s] = in ? *reinterpret_cast<const v4u*>(kp + s * 16) : v4u{0u, 0u, 0u, 0u};
            const v4u v = in ? *reinterpret_cast<const v4u*>(vp + s * 16) : v4u{0u, 0u, 0u, 0u};
            if constexpr (V_IN_LDS) *reinterpret_cast<v4u*>(vl + wave * 32 * DP + tile_at<DP>(lane & 31, 2 * s + half)) = v;
            else vf[s] = v;
        }
    }
    if (t0 < t1) {
        aim(t0);
        copies.group(0, 1, q_tile(t0), g_tile(t0), 0, q0, g0);
        finish(lse0, delta0);
    }

    v16f dk[DTL], dv[DTL];
#pragma unroll
    for (int t = 0; t < DTL; ++t) { dk[t] = splat16(0.f); dv[t] = splat16(0.f); }
    wait_loads();
    __syncthreads();
    LaneOffsets<DP> at(lane);
    Operands<DP, V_IN_LDS ? 2 : 4> ops;
    float factor = __builtin_ldexpf(kUnshiftP<DT>, kMostShift);  // fp16: of dS beside the shifted P's
    auto step = [&](int t, auto buffer) {
        constexpr int BUF = decltype(buffer)::value;
        at.fresh();
        const uint16_t *ql = BUF ? q1 : q0, *gl = BUF ? g1 : g0;
        const float *lt = BUF ? lse1 : lse0, *dt = BUF ? delta1 : delta0;
        uint16_t *qnext = BUF ? q0 : q1, *gnext = BUF ? g0 : g1;
        aim(t + 1);
        const XTile qtile = q_tile(t + 1), gtile = g_tile(t + 1);
        constexpr int PARTS = TR / 16 * ops.RN;
        auto keep = [] { if constexpr (!V_IN_LDS) fence(); };
#pragma unroll
        for (int u = 0; u < TR / 32; ++u) {
            v16f s = splat16(0.f), dp = bias16(dt, u, half);
            int w = 0;  // the place of the operands that are next
            if (u == 0) ops.rows(0, ql, 0, 0, at);
#pragma unroll
            for (int g = 0; g < ops.RN; ++g, w ^= 1) {
                if (g + 1 < ops.RN) ops.rows(w ^ 1, ql, u * 32, g + 1, at);
                else ops.rows(w ^ 1, gl, u * 32, 0, at);
                copies.group(u * 2 * ops.RN + g, PARTS, qtile, gtile, 0, qnext, gnext);
                keep();
#pragma unroll
                for (int j = 0; j < ops.RG; ++j) s = mfma16<DT>(ops.f[w][j], kf[g * ops.RG + j], s);
                keep();
            }
#pragma unroll
            for (int g = 0; g < ops.RN; ++g, w ^= 1) {
                v4u v[ops.RG];
#pragma unroll
                for (int j = 0; j < ops.RG; ++j) {
                    if constexpr (V_IN_LDS) v[j] = lds_rows<DP>(vl, wave * 32, g * ops.RG + j, at);
                    else v[j] = vf[g * ops.RG + j];
                }
                if (g + 1 < ops.RN) ops.rows(w ^ 1, gl, u * 32, g + 1, at);
                else ops.cols(w ^ 1, gl, u * 32, 0, at);
                copies.group((u * 2 + 1) * ops.RN + g, PARTS, qtile, gtile, 0, qnext, gnext);
                keep();
#pragma unroll
                for (int j = 0; j < ops.RG; ++j) dp = mfma16<DT>(ops.f[w][j], v[j], dp);
                // P, a part of it beside each group
#pragma unroll
                for (int i = g * 4 / ops.RN; i < (g + 1) * 4 / ops.RN; ++i) {
                    const v4f x = *reinterpret_cast<const v4f*>(&lt[u * 32 + i * 8 + half * 4]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[i * 4 + j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i * 4 + j], a.c, x[j]));
                }
                keep();
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const v4u p = pack_step<DT>(s, k);
#pragma unroll
                for (int c = 0; c < ops.CN; ++c, w ^= 1) {
                    if (c + 1 < ops.CN) ops.cols(w ^ 1, gl, u * 32 + k * 16, c + 1, at);
                    else if (k == 0) ops.cols(w ^ 1, gl, u * 32 + 16, 0, at);
                    else ops.cols(w ^ 1, ql, u * 32, 0, at);
                    keep();
#pragma unroll
                    for (int d = 0; d < ops.CG; ++d) dv[c * ops.CG + d] = mfma16<DT>(ops.f[w][d], p, dv[c * ops.CG + d]);
                    if (k == 0 && c == 0) {  // dS, beside them (P's second half is still needed as it is)
#pragma unroll
                        for (int i = 0; i < 16; ++i) dp[i] *= DT == Q8_F16 ? s[i] * factor : s[i];
                    }
                    keep();
                }
            }
            if constexpr (DT == Q8_F16) {
                const int change = counts ? shift_change(dp) : 0;
                if (__builtin_amdgcn_ballot_w64(change != 0) != 0) {
                    const float f = __builtin_ldexpf(1.0f, change);
#pragma unroll
                    for (int i = 0; i < 16; ++i) dp[i] *= f;
                    scale_all(dk, f);
                    factor *= f;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const v4u p = pack_step<DT>(dp, k);
#pragma unroll
                for (int c = 0; c < ops.CN; ++c, w ^= 1) {
                    if (c + 1 < ops.CN) ops.cols(w ^ 1, ql, u * 32 + k * 16, c + 1, at);
                    else if (k == 0) ops.cols(w ^ 1, ql, u * 32 + 16, 0, at);
                    else if (u + 1 < TR / 32) ops.rows(w ^ 1, ql, 32, 0, at);
                    keep();
#pragma unroll
                    for (int d = 0; d < ops.CG; ++d) dk[c * ops.CG + d] = mfma16<DT>(ops.f[w][d], p, dk[c * ops.CG + d]);
                    keep();
                }
            }
        }
        finish(BUF ? lse0 : lse1, BUF ? delta0 : delta1);
        __syncthreads();
    };
    for (int t = t0; t < t1; t += 2) {
        step(t, std::integral_constant<int, 0>{});
        if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{});
    }
    if (!counts) {  // a key that does not count has no gradient, whatever its column holds
#pragma unroll
        for (int t = 0; t < DTL; ++t) { dk[t] = splat16(0.f); dv[t] = splat16(0.f); }
    }
    if constexpr (DT == Q8_F16) {
        scale_all(dv, kUnshiftP<DT>);
        scale_all(dk, kUnshiftP<DT> / factor);  // (a power of two)
    }
    const XBwd& z = arguments_again<XBwd>();
    if (of > 1) {
        if (key < z.N) {
            float* p = z.part + (((int64_t)split * z.plan.tail + (block - z.plan.full)) * kXRows + wave * 32 + (lane & 31)) * 2 * z.D;
#pragma unroll
            for (int d = 0; d < DTL; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = d * 32 + i * 8 + half * 4;
                    if (e < z.D) {
                        *reinterpret_cast<v4f*>(p + e) = v4f{dk[d][4 * i], dk[d][4 * i + 1], dk[d][4 * i + 2], dk[d][4 * i + 3]};
                        *reinterpret_cast<v4f*>(p + z.D + e) = v4f{dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]};
                    }
                }
        }
        return;
    }
    const bool there = key < z.N;
    store_rows<DT, DP>(dk, z.scale, there ? z.dk.p + b * z.dk.sb + hk * z.dk.sh + key * z.dk.st : nullptr, z.D, lane);
    store_rows<DT, DP>(dv, 1.0f, there ? z.dv.p + b * z.dv.sb + hk * z.dv.sh + key * z.dv.st : nullptr, z.D, lane);
}

// Few keys (32 W of them at most): all gradients in one pass over the rows, five products instead of seven, and Q, dO and O read
// once. A wave owns 32 keys, as above; dS of a tile of TR rows goes to LDS as [key][row], from where (turned while it is read,
// like K) it is an operand of dQ^T = K^T dS^T. A wave forms one 32 x 32 block of dQ^T over a part of the keys; where more waves
// share a block, the others' sums go through LDS to the first. delta comes from the same tile's O and dO. A workgroup walks over
// a part of its unit's tiles; the parts' dK and dV are added by the kernel below.
//
// Heads of more than 64 have tiles of 32 rows, K's operands from LDS, O and dO for delta only asked for behind the products and
// the compiler's order of instructions: what two waves on a SIMD have registers for, but for 14 (2 x 32 heads of 128, 6144 rows, 128
// keys bf16: 130 to 142 us; with the groups kept apart 147 to 151; fp16, whose powers cost 14 more of them, 172).
//
// bf16, 2 x 32 heads of 64, 6144 rows, 256 keys, ragged: 93 to 118 us and 7 for the parts (274 MB; the matrix pipes are busy 27 % of
// the time, the vector units 37 %, LDS 30 %: between the two barriers of a tile the two waves of a SIMD are in the same phase).
template <int DT, int DP, int W>
__global__ __launch_bounds__(W * 64, 2) void cross_attn_bwd_few_keys_kernel(XBwd a, int parts) {
    constexpr bool LONG = DP > 64;
    constexpr int KS = DP / 16, DTL = DP / 32, TR = !LONG || (DP == 96 && W == 8) ? 64 : 32, ELEMS = TR * DP;
    constexpr int RB = TR / 32, NB = RB * DTL, KG = W / NB, STEPS = W * 2 / KG;  // blocks of dQ^T, waves that share one, 16-key steps of each
    constexpr int CL = DP == 32 ? 4 : DP == 64 ? 8 : 16;  // lanes that share a row of dO and O, for delta
    constexpr int CHUNKS = TR * CL / (W * 64) > 0 ? TR * CL / (W * 64) : 1;
    __shared__ __align__(16) uint16_t q0[ELEMS], q1[ELEMS], g0[ELEMS], g1[ELEMS], kt[W * 32 * DP], ds[W * 32 * TR];
    __shared__ __align__(16) float lse0[TR], lse1[TR], delta0[TR], delta1[TR];  // -lse and -delta of the tile's rows
    constexpr bool SHIFT = DT == Q8_F16;
    __shared__ float size0[SHIFT ? TR : 1], size1[SHIFT ? TR : 1], vsize[SHIFT ? W : 1];  // |dO|^2 of the tile's rows, largest |V|^2 of a wave's keys
    __shared__ __align__(16) float sums[KG > 1 ? (KG - 1) * NB * 1024 : 4];
    const int unit = blockIdx.x / parts, part = blockIdx.x - unit * parts;
    const int b = unit / a.Hkv, hk = unit - b * a.Hkv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int key = wave * 32 + (lane & 31);
    const int len = a.keys.length(b);
    const uint8_t* mask = a.keys.row(b);
    const bool counts = key < len && (mask == nullptr || mask[key]);
    const uint32_t keep = counts ? ~0u : 0u;
    const bool idle = __builtin_amdgcn_ballot_w64(counts) == 0;  // no key of this wave counts
    const int head_tiles = (a.M + TR - 1) / TR, tiles = a.G * head_tiles, per = (tiles + parts - 1) / parts;
    const int t0 = part * per, t1 = t0 + per < tiles ? t0 + per : tiles;

    v4u kf[LONG ? 1 : KS], vf[KS];
    {
        const uint16_t* kp = a.k.p + b * a.k.sb + hk * a.k.sh + key * a.k.st + half * 8;
        const uint16_t* vp = a.v.p + b * a.v.sb + hk * a.v.sh + key * a.v.st + half * 8;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const bool in = counts && s * 16 + half * 8 < a.D;
            const v4u x = in ? *reinterpret_cast<const v4u*>(kp + s * 16) : v4u{0u, 0u, 0u, 0u};
            if constexpr (!LONG) kf[s] = x;
            vf[s] = in ? *reinterpret_cast<const v4u*>(vp + s * 16) : v4u{0u, 0u, 0u, 0u};
            *reinterpret_cast<v4u*>(kt + wave * 32 * DP + tile_at<DP>(lane & 31, 2 * s + half)) = x;
        }
    }
    if constexpr (SHIFT) {
        float n = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) n = square_sum<DT>(vf[s][i], n);
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(n), __float_as_uint(n), false, false);
        n = group_max<32>(__uint_as_float(r[0]) + __uint_as_float(r[1]));
        if (lane == 0) vsize[wave] = n;
    }
    if (idle) {  // its part of dS stays zero
        for (int i = lane; i < 32 * TR / 8; i += 64) *reinterpret_cast<v4u*>(ds + wave * 32 * TR + i * 8) = v4u{0u, 0u, 0u, 0u};
    }

    Copies<DP, TR, W> copies;
    copies.wave = wave;
    copies.D = a.D;
    int rows = 0;
    float row_lse = 0.f;
    v4u dor[CHUNKS], orr[CHUNKS];
    v2i lowr[CHUNKS];
    const uint16_t *qp = a.q.p + b * a.q.sb + (int64_t)hk * a.G * a.q.sh, *gp = a.g.p + b * a.g.sb + (int64_t)hk * a.G * a.g.sh;
    const uint16_t* op = a.o.p + b * a.o.sb + (int64_t)hk * a.G * a.o.sh;
    const uint8_t* lp = a.o_low + (int64_t)unit * a.R * a.D;
    const int chunk = (int)threadIdx.x % CL, crow = (int)threadIdx.x / CL;  // of delta: rows crow + k W 64 / CL
    // the tile that is next (t past the end: empty)
    auto aim = [&](int t) {
        const int g = t / head_tiles, m = (t - g * head_tiles) * TR;
        rows = t < t1 ? a.M - m : 0;
        if (rows > TR) rows = TR;
        const int last = rows - 1, n = (int)threadIdx.x & (TR - 1);
        row_lse = a.lse[(int64_t)unit * a.R + (rows ? g * a.M + m + (n < rows ? n : last) : 0)];
    };
    // what its delta is formed of
    auto ask = [&](int t) {
        const int g = t / head_tiles, m = (t - g * head_tiles) * TR, last = rows - 1;
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const int r = crow + k * (W * 64 / CL), i = m + (r < last ? r : last);
            const bool in = rows > 0 && chunk * 8 < a.D;
            dor[k] = in ? *reinterpret_cast<const v4u*>(gp + g * a.g.sh + i * a.g.st + chunk * 8) : v4u{0u, 0u, 0u, 0u};
            orr[k] = in ? *reinterpret_cast<const v4u*>(op + g * a.o.sh + i * a.o.st + chunk * 8) : v4u{0u, 0u, 0u, 0u};
            lowr[k] = in ? *reinterpret_cast<const v2i*>(lp + ((int64_t)g * a.M + i) * a.D + chunk * 8) : v2i{0, 0};
        }
    };
    auto tile_of = [&](const uint16_t* p, const XTensor& x, int t) {
        const int g = t / head_tiles, m = (t - g * head_tiles) * TR;
        return XTile(p + g * x.sh + m * x.st, x.st, rows, a.D, TR);
    };
    auto finish = [&](float* lt, float* dt, float* st) {
        wait_loads();
        if (threadIdx.x < TR) lt[threadIdx.x] = (int)threadIdx.x < rows ? kShiftP<DT> - row_lse : -__builtin_inff();
#pragma unroll
        for (int k = 0; k < CHUNKS; ++k) {
            const float d = group_sum<CL>(dot_sum<DT>(dor[k], orr[k], lowr[k], 0.f));
            const int r = crow + k * (W * 64 / CL);
            if (chunk == 0 && r < TR) dt[r] = r < rows ? -d : 0.f;
            if constexpr (SHIFT) {
                float n = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) n = square_sum<DT>(dor[k][i], n);
                n = group_sum<CL>(n);
                if (chunk == 0 && r < TR) st[r] = r < rows && n < __builtin_inff() ? n : 0.f;  // (a row that is not finite says nothing of the others)
            }
        }
    };

    v16f dk[DTL], dv[DTL];
#pragma unroll
    for (int t = 0; t < DTL; ++t) { dk[t] = splat16(0.f); dv[t] = splat16(0.f); }
    if (t0 < t1) {
        aim(t0);
        ask(t0);
        copies.group(0, 1, tile_of(qp, a.q, t0), tile_of(gp, a.g, t0), 0, q0, g0);
        finish(lse0, delta0, size0);
    }
    wait_loads();
    __syncthreads();
    int shift = kMostShift, least = kMostShift;  // log2 of the present factor of dS, and the least that a tile so far asked for

    LaneOffsets<DP> at(lane);
    LaneOffsets<TR> ds_at(lane);
    Operands<DP, LONG ? 2 : 4> ops;
    auto keep_apart = [] { if constexpr (!LONG) fence(); };
    auto step = [&](int t, auto buffer, auto exact) {
        constexpr int BUF = decltype(buffer)::value;
        at.fresh();
        const uint16_t *ql = BUF ? q1 : q0, *gl = BUF ? g1 : g0;
        const float *lt = BUF ? lse1 : lse0, *dt = BUF ? delta1 : delta0;
        uint16_t *qnext = BUF ? q0 : q1, *gnext = BUF ? g0 : g1;
        const int g = t / head_tiles, m = (t - g * head_tiles) * TR, here = rows;
        aim(t + 1);
        if constexpr (!LONG) ask(t + 1);
        copies.group(0, 1, tile_of(qp, a.q, t + 1), tile_of(gp, a.g, t + 1), 0, qnext, gnext);
        float factor = 1.0f;  // of dS beside the shifted P's
        if constexpr (SHIFT) {
            // The power that brings the bound to 2^14 .. 2^15, but no more than 40 above the least one, so that the sums so far stay in range.
            float most_v = 0.f;  // (read again for every tile: no register for it between the products)
#pragma unroll
            for (int i = 0; i < W; ++i) most_v = fmaxf(most_v, vsize[i]);
            const float rows_most = group_max<64>((BUF ? size1 : size0)[lane & (TR - 1)]);
            const float bound = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(rows_most * most_v)));
            const int x = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(bound));
            const int own = bound > 0.f ? min(15 - ((x + 1) >> 1), kMostShift) : kMostShift;
            least = min(least, own);
            const int next = min(own, least + 40);
            if (shift != next) {
                scale_all(dk, __builtin_ldexpf(1.0f, next - shift));
                shift = next;
            }
            factor = power_of_two(shift - kShiftP<DT>);
        }
        if (!idle) {
#pragma unroll
            for (int u = 0; u < RB; ++u) {
                v16f s = splat16(0.f), dp = bias16(dt, u, half);
                int w = 0;  // the place of the operands that are next
                if (u == 0) ops.rows(0, ql, 0, 0, at);
#pragma unroll
                for (int i = 0; i < ops.RN; ++i, w ^= 1) {
                    v4u k[ops.RG];
#pragma unroll
                    for (int j = 0; j < ops.RG; ++j) {
                        if constexpr (LONG) k[j] = lds_rows<DP>(kt, wave * 32, i * ops.RG + j, at);
                        else k[j] = kf[i * ops.RG + j];
                    }
                    if (i + 1 < ops.RN) ops.rows(w ^ 1, ql, u * 32, i + 1, at);
                    else ops.rows(w ^ 1, gl, u * 32, 0, at);
                    keep_apart();
#pragma unroll
                    for (int j = 0; j < ops.RG; ++j) s = mfma16<DT>(ops.f[w][j], k[j], s);
                    keep_apart();
                }
#pragma unroll
                for (int i = 0; i < ops.RN; ++i, w ^= 1) {
                    if (i + 1 < ops.RN) ops.rows(w ^ 1, gl, u * 32, i + 1, at);
                    else ops.cols(w ^ 1, gl, u * 32, 0, at);
                    keep_apart();
#pragma unroll
                    for (int j = 0; j < ops.RG; ++j) dp = mfma16<DT>(ops.f[w][j], vf[i * ops.RG + j], dp);
                    // P, a part of it beside each group
#pragma unroll
                    for (int q = i * 4 / ops.RN; q < (i + 1) * 4 / ops.RN; ++q) {
                        const v4f x = *reinterpret_cast<const v4f*>(&lt[u * 32 + q * 8 + half * 4]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[q * 4 + j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[q * 4 + j], a.c, x[j]));
                    }
                    keep_apart();
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const v4u p = pack_step<DT>(s, k);
#pragma unroll
                    for (int c = 0; c < ops.CN; ++c, w ^= 1) {
                        if (c + 1 < ops.CN) ops.cols(w ^ 1, gl, u * 32 + k * 16, c + 1, at);
                        else if (k == 0) ops.cols(w ^ 1, gl, u * 32 + 16, 0, at);
                        else ops.cols(w ^ 1, ql, u * 32, 0, at);
                        keep_apart();
#pragma unroll
                        for (int d = 0; d < ops.CG; ++d) dv[c * ops.CG + d] = mfma16<DT>(ops.f[w][d], p, dv[c * ops.CG + d]);
                        if (k == 0 && c == 0) {  // dS, beside them (P's second half is still needed as it is)
                            if constexpr (exact) {  // all keys are in this wave: what their dS adds up to is the error of delta
#pragma unroll
                                for (int i = 0; i < 16; ++i)
                                    dp[i] -= group_sum<32>(__uint_as_float(__float_as_uint(dp[i] * s[i]) & keep)) * kUnshiftP<DT>;
                            }
#pragma unroll
                            for (int i = 0; i < 16; ++i) dp[i] *= SHIFT ? s[i] * factor : s[i];
                        }
                        keep_apart();
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    v4u p = pack_step<DT>(dp, k);
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[i] &= keep;  // a key that does not count may hold anything here
                    // rows u * 32 + 8 (2 k) + 4 half .. + 3 and the 4 rows 8 further, of this lane's key
                    *reinterpret_cast<v2i*>(ds + wave * 32 * TR + tile_at<TR>(lane & 31, u * 4 + 2 * k) + half * 4) = v2i{(int)p[0], (int)p[1]};
                    *reinterpret_cast<v2i*>(ds + wave * 32 * TR + tile_at<TR>(lane & 31, u * 4 + 2 * k + 1) + half * 4) = v2i{(int)p[2], (int)p[3]};
#pragma unroll
                    for (int c = 0; c < ops.CN; ++c, w ^= 1) {
                        if (c + 1 < ops.CN) ops.cols(w ^ 1, ql, u * 32 + k * 16, c + 1, at);
                        else if (k == 0) ops.cols(w ^ 1, ql, u * 32 + 16, 0, at);
                        else if (u + 1 < RB) ops.rows(w ^ 1, ql, 32, 0, at);
                        keep_apart();
#pragma unroll
                        for (int d = 0; d < ops.CG; ++d) dk[c * ops.CG + d] = mfma16<DT>(ops.f[w][d], p, dk[c * ops.CG + d]);
                        keep_apart();
                    }
                }
                // (an even number of groups: the next rows are in place 0)
            }
        }
        if constexpr (LONG) ask(t + 1);  // (here: before, there are no registers for it)
        barrier();
        // dQ^T: this wave's block of rows and elements, over its part of the keys
        const int block = wave % NB, kg = wave / NB, rb = block % RB, db = block / RB;  // (kg = KG: a wave without one)
        v16f dq = splat16(0.f);
        if (kg < KG)
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const int key0 = (kg * STEPS + i) * 16;
            dq = mfma16<DT>(lds_cols<DP>(kt, key0, db, at), lds_cols<TR>(ds, key0, rb, ds_at), dq);
        }
        auto store = [&] {
            const int r = rb * 32 + (lane & 31);
            uint16_t* p = a.dq.p + b * a.dq.sb + (int64_t)(hk * a.G + g) * a.dq.sh + (int64_t)(m + r) * a.dq.st + db * 32;
            store_rows<DT, 32>({dq}, SHIFT ? __builtin_ldexpf(a.scale, -shift) : a.scale, r < here ? p : nullptr, a.D - db * 32, lane);
        };
        // Behind the barrier the next tile is whole and dS has been read. (The sums have been when their writers come back to them:
        // the barrier in front of the product lies between.)
        if constexpr (KG == 1) {
            if (kg == 0) store();
            finish(BUF ? lse0 : lse1, BUF ? delta0 : delta1, BUF ? size0 : size1);
            barrier();
        } else {
            finish(BUF ? lse0 : lse1, BUF ? delta0 : delta1, BUF ? size0 : size1);
            if (kg > 0 && kg < KG) {
                float* to = sums + ((kg - 1) * NB + block) * 1024 + lane * 4;
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<v4f*>(to + i * 256) = v4f{dq[4 * i], dq[4 * i + 1], dq[4 * i + 2], dq[4 * i + 3]};
            }
            barrier();
            if (kg == 0) {
#pragma unroll
                for (int o = 0; o < KG - 1; ++o) {
                    const float* from = sums + (o * NB + block) * 1024 + lane * 4;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const v4f x = *reinterpret_cast<const v4f*>(from + i * 256);
#pragma unroll
                        for (int j = 0; j < 4; ++j) dq[4 * i + j] += x[j];
                    }
                }
                store();
            }
        }
    };
    auto walk = [&](auto exact) {
        for (int t = t0; t < t1; t += 2) {
            step(t, std::integral_constant<int, 0>{}, exact);
            if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{}, exact);
        }
    };
    if (len <= kXExact) walk(std::true_type{});
    else walk(std::false_type{});
    if (!counts) {  // a key that does not count has no gradient, whatever its column holds
#pragma unroll
        for (int t = 0; t < DTL; ++t) { dk[t] = splat16(0.f); dv[t] = splat16(0.f); }
    }
    if constexpr (SHIFT) {
        scale_all(dv, kUnshiftP<DT>);
        scale_all(dk, __builtin_ldexpf(1.0f, -shift));
    }
    const XBwd& z = arguments_again<XBwd>();
    if (key >= z.N) return;
    if (parts > 1) {
        const int kb = wave / kXWaves;  // the block of 128 keys that the kernel below counts in
        float* p = z.part + (((int64_t)part * z.plan.tail + (unsigned)(unit * z.blocks + kb)) * kXRows + (wave & 3) * 32 + (lane & 31)) * 2 * z.D;
#pragma unroll
        for (int d = 0; d < DTL; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int e = d * 32 + i * 8 + half * 4;
                if (e < z.D) {
                    *reinterpret_cast<v4f*>(p + e) = v4f{dk[d][4 * i], dk[d][4 * i + 1], dk[d][4 * i + 2], dk[d][4 * i + 3]};
                    *reinterpret_cast<v4f*>(p + z.D + e) = v4f{dv[d][4 * i], dv[d][4 * i + 1], dv[d][4 * i + 2], dv[d][4 * i + 3]};
                }
            }
        return;
    }
    store_rows<DT, DP>(dk, z.scale, z.dk.p + b * z.dk.sb + hk * z.dk.sh + key * z.dk.st, z.D, lane);
    store_rows<DT, DP>(dv, 1.0f, z.dv.p + b * z.dv.sb + hk * z.dv.sh + key * z.dv.st, z.D, lane);
}

// Adds the parts of dQ (WIDTH = 1) or of dK and dV (WIDTH = 2): one thread for 4 elements of a row.
template <int DT, int WIDTH>
__global__ __launch_bounds__(256) void cross_attn_add_kernel(XBwd a) {
    const int64_t rows = (int64_t)a.plan.tail * kXRows;
    const int quads = WIDTH * a.D / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = i / quads;
    const unsigned tail = (unsigned)(n / kXRows), block = a.plan.full + tail;
    const int unit = block / a.blocks, r = (block - unit * a.blocks) * kXRows + (int)(n - (int64_t)tail * kXRows);
    if (n >= rows || r >= (WIDTH == 1 ? a.R : a.N)) return;
    int e = (int)(i - n * quads) * 4;
    v4f s = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < a.plan.splits; ++k) {
        const v4f p = *reinterpret_cast<const v4f*>(a.part + ((int64_t)k * rows + n) * (WIDTH * a.D) + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] += p[j];
    }
    const bool is_v = WIDTH == 2 && e >= a.D;
    const float f = is_v ? 1.0f : a.scale;
    if (is_v) e -= a.D;
    const int b = unit / a.Hkv, hk = unit - b * a.Hkv;
    uint16_t* p;
    if constexpr (WIDTH == 1) {
        const int g = r / a.M;
        p = a.dq.p + b * a.dq.sb + (int64_t)(hk * a.G + g) * a.dq.sh + (r - g * a.M) * a.dq.st;
    } else {
        const XOut& x = is_v ? a.dv : a.dk;
        p = x.p + b * x.sb + hk * x.sh + r * x.st;
    }
    *reinterpret_cast<v2i*>(p + e) = v2i{(int)pack2<DT>(s[0] * f, s[1] * f), (int)pack2<DT>(s[2] * f, s[3] * f)};
}

struct XPlan {
    int64_t units, rows, dq_blocks, kv_blocks, parts;  // blocks of a unit; floats of partial results
    int few;  // waves of the kernel for few keys, 0: not taken
    XSchedule dq, kv;
};
static XPlan plan(int64_t B, int H, int Hkv, int M, int N, int D) {
    XPlan p{};
    p.units = B * Hkv;
    p.rows = (int64_t)(H / Hkv) * M;
    p.dq_blocks = (p.rows + kXRows - 1) / kXRows;
    p.kv_blocks = ((int64_t)N + kXRows - 1) / kXRows;
    const int64_t tiles = (int64_t)(H / Hkv) * (((int64_t)M + kXTile - 1) / kXTile);
    // The kernel for few keys, a workgroup for four tiles of 64 rows or more: one of 8 waves on a CU, or two of 4 (LDS). bf16 times,
    // this kernel against the other two, with their additions (B x H x M x N x D), us:
    //   2 x 32 x 6144 x 256 x 64   120, 178     2 x 32 x 6144 x 128 x 64   81, 122    2 x 32 x 6144 x 128 x 128   154, 273
    //   2 x 32 x 6144 x 256 x 128  233, 326     2 x 32 x 6144 x 256 x 96  155, 231    11 x 32 on 4 x 2836 x 16 x 128  368, 475
    //   1 x 32 x 2048 x 128 x 64   28, 36       1 x 16 x 1024 x 64 x 64   20.6, 22.8  16 x 32 x 256 x 128 x 64   31, 51
    // and in fp16 2 x 32 x 6144 x 256 x 64 145, 194; 6144 x 128 x 128 184, 272; 6144 x 256 x 128 292, 343. With 129 to 256 keys it takes
    // 1024 tiles to be faster for certain: 8 x 8192 x 256 x 64 39.5 against 44.8; with 512 either is, 16 x 2048 x 256 x 64 31.2 against
    // 32.6, 16 x 2048 x 256 x 128 54.9 against 55.0, and 8 x 512 x 256 x 64 (64 tiles) 26.3 against 26.1.
    const int at_once = N > kXRows ? 256 : 512;
    if (p.units > 0 && M > 0 && N > 0 && (N <= kXRows || (N <= 2 * kXRows && p.units * tiles >= 4 * at_once)) && p.units <= kXMostBlocks / 2) {
        p.few = N > kXRows ? 8 : 4;
        p.kv.full = 0;
        p.kv.tail = (unsigned)(p.units * p.kv_blocks);
        p.kv.splits = walk_parts(p.units, tiles, at_once, 4);
        p.parts = p.kv.parts() * kXRows * 2 * D;
        return p;
    }
    // Workgroups that run at once on the 256 CUs, by the registers of a lane. A tile takes these kernels 1.3 and 1.7 times what it
    // takes the forward, which is what the floats of a part (for dK and dV twice as many) are weighed with: 8 heads of 128,
    // 1024 x 1024 60 us, dK and dV in 4 parts or more; 77 with none divided.
    p.dq = schedule(p.units * p.dq_blocks, N, D <= 32 ? 1024 : D <= 64 ? 768 : 512, 0.75 * (p.rows < kXRows ? p.rows : kXRows) * D);
    p.kv = schedule(p.units * p.kv_blocks, tiles * kXTile, D <= 32 ? 1024 : 512, (double)(N < kXRows ? N : kXRows) * D);
    const int64_t dq = p.dq.parts() * kXRows * D, kv = p.kv.parts() * kXRows * 2 * D;
    p.parts = dq > kv ? dq : kv;  // one after the other in the same place
    return p;
}
static int64_t delta_floats(const XPlan& p) { return p.few ? 0 : (p.units * p.rows + 3) / 4 * 4; }

struct XBackward {
    const void* grad; const int64_t* grad_strides;
    const void* q; const int64_t* q_strides;
    const void* k; const int64_t* k_strides;
    const void* v; const int64_t* v_strides;
    const void* o; const int64_t* o_strides;
    const void* o_low;  // NULL: formed here, by the forward once more
    const float* lse;
    void* dq; const int64_t* dq_strides;
    void* dk; const int64_t* dk_strides;
    void* dv; const int64_t* dv_strides;
    const int32_t* kv_lens; const uint8_t* key_mask; int64_t mask_row_stride;
    int dt; float softmax_scale;
    int64_t B; int H, Hkv, M, N, D;
    void* workspace; int64_t workspace_bytes;
    hipStream_t stream;
};

static bool fits(const XPlan& p) { return p.units * p.dq_blocks <= kXMostBlocks && p.units * p.kv_blocks <= kXMostBlocks; }
static int64_t plan_bytes(const XPlan& p) { return (delta_floats(p) + p.parts) * (int64_t)sizeof(float); }
static int64_t low_bytes(int64_t B, int H, int M, int D) { return (B * H * M * D + 15) / 16 * 16; }
// with o_low formed here: it, and behind it what the forward and then the backward use
static int64_t whole_bytes(int64_t B, int H, int Hkv, int M, int N, int D) {
    const int64_t fwd = cross_attn_forward_workspace(B, H, Hkv, M, N, D), bwd = plan_bytes(plan(B, H, Hkv, M, N, D));
    return low_bytes(B, H, M, D) + (fwd > bwd ? fwd : bwd);
}

static int cross_attn_backward(const char* who, const XBackward& c) {
    if (int e = x_sizes(who, c.dt, c.B, c.H, c.Hkv, c.M, c.N, c.D, c.softmax_scale)) return e;
    const int M = c.M, N = c.N, D = c.D;
    if (c.B == 0 || (M == 0 && N == 0)) return Q8_OK;
    static const int64_t none[3] = {0, 0, 0};
    if (M) {
        if (int e = x_tensor(who, "grad", c.grad, c.grad_strides, c.B, c.H, M, D)) return e;
        if (int e = x_tensor(who, "q", c.q, c.q_strides, c.B, c.H, M, D)) return e;
        if (int e = x_tensor(who, "o", c.o, c.o_strides, c.B, c.H, M, D)) return e;
        if (int e = x_tensor(who, "dq", c.dq, c.dq_strides, c.B, c.H, M, D)) return e;
        if (c.lse == nullptr) return fail(Q8_ERR_NULL, "%s: lse is NULL", who);
        if (!aligned16(c.o_low)) return fail(Q8_ERR_ALIGN, "%s: o_low must be 16-byte aligned", who);
    }
    if (N) {
        if (int e = x_tensor(who, "k", c.k, c.k_strides, c.B, c.Hkv, N, D)) return e;
        if (int e = x_tensor(who, "v", c.v, c.v_strides, c.B, c.Hkv, N, D)) return e;
        if (int e = x_tensor(who, "dk", c.dk, c.dk_strides, c.B, c.Hkv, N, D)) return e;
        if (int e = x_tensor(who, "dv", c.dv, c.dv_strides, c.B, c.Hkv, N, D)) return e;
    }
    if ((reinterpret_cast<uintptr_t>(c.lse) & 3) || (reinterpret_cast<uintptr_t>(c.kv_lens) & 3)) return fail(Q8_ERR_ALIGN, "%s: lse or kv_lens not aligned", who);
    if (c.key_mask && (c.mask_row_stride < 0 || (c.B > 1 && c.mask_row_stride > INT64_MAX / 2 / c.B))) return fail(Q8_ERR_SHAPE, "%s: row stride of the mask", who);
    const XPlan p = plan(c.B, c.H, c.Hkv, M, N, D);
    const bool form_low = c.o_low == nullptr && M;
    const int64_t need = form_low ? whole_bytes(c.B, c.H, c.Hkv, M, N, D) : plan_bytes(p);
    if (need && c.workspace == nullptr) return fail(Q8_ERR_NULL, "%s: a workspace of %lld bytes is needed", who, (long long)need);
    if (c.workspace_bytes < need) return fail(Q8_ERR_SHAPE, "%s: workspace of %lld bytes, %lld needed", who, (long long)c.workspace_bytes, (long long)need);
    if (!aligned16(c.workspace)) return fail(Q8_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
    if (!fits(p)) return fail(Q8_ERR_SHAPE, "%s: sizes out of range", who);
    char* work = static_cast<char*>(c.workspace);
    const void* o_low = c.o_low;
    if (form_low) {
        o_low = work;
        work += low_bytes(c.B, c.H, M, D);
        if (int e = cross_attn_forward(who, XForward{c.q, c.q_strides, c.k, c.k_strides, c.v, c.v_strides, nullptr, nullptr, c.workspace, nullptr, c.kv_lens, c.key_mask,
                                                     c.mask_row_stride, c.dt, c.softmax_scale, c.B, c.H, c.Hkv, M, N, D, work,
                                                     c.workspace_bytes - low_bytes(c.B, c.H, M, D), c.stream}))
            return e;
    }
    XBwd a{};
    auto in = [&](const void* x, const int64_t* s, int n) {
        const int64_t* t = n ? s : none;
        return XTensor{static_cast<const uint16_t*>(x), t[0], t[1], t[2]};
    };
    auto out = [&](void* x, const int64_t* s, int n) {
        const int64_t* t = n ? s : none;
        return XOut{static_cast<uint16_t*>(x), t[0], t[1], t[2]};
    };
    a.q = in(c.q, c.q_strides, M);
    a.o = in(c.o, c.o_strides, M);
    a.o_low = static_cast<const uint8_t*>(o_low);
    a.g = in(c.grad, c.grad_strides, M);
    a.k = in(c.k, c.k_strides, N);
    a.v = in(c.v, c.v_strides, N);
    a.dq = out(c.dq, c.dq_strides, M);
    a.dk = out(c.dk, c.dk_strides, N);
    a.dv = out(c.dv, c.dv_strides, N);
    a.lse = c.lse;
    a.delta = reinterpret_cast<float*>(work);
    a.part = a.delta + delta_floats(p);
    a.keys = XKeys{c.kv_lens, c.key_mask, c.mask_row_stride, N};
    a.c = c.softmax_scale * kLog2e;
    a.scale = c.softmax_scale;
    a.Hkv = c.Hkv;
    a.G = c.H / c.Hkv;
    a.M = M;
    a.N = N;
    a.D = D;
    a.R = (int)p.rows;
    hipStream_t st = c.stream;
#define X_BWD(NAME, DT)                                                       \
    switch (padded_head(D)) {                                                 \
        case 32: NAME<DT, 32><<<grid, kXThreads, 0, st>>>(a); break;          \
        case 64: NAME<DT, 64><<<grid, kXThreads, 0, st>>>(a); break;          \
        case 96: NAME<DT, 96><<<grid, kXThreads, 0, st>>>(a); break;          \
        default: NAME<DT, 128><<<grid, kXThreads, 0, st>>>(a);                \
    }
    if (p.few) {
        a.blocks = (int)p.kv_blocks;
        a.plan = p.kv;
        const unsigned grid = (unsigned)(p.units * p.kv.splits);
#define X_FEW(DT, W)                                                                                                           \
    do {                                                                                                                       \
        switch (padded_head(D)) {                                                                                              \
            case 32: cross_attn_bwd_few_keys_kernel<DT, 32, W><<<grid, W * 64, 0, st>>>(a, p.kv.splits); break;                \
            case 64: cross_attn_bwd_few_keys_kernel<DT, 64, W><<<grid, W * 64, 0, st>>>(a, p.kv.splits); break;                \
            case 96: cross_attn_bwd_few_keys_kernel<DT, 96, W><<<grid, W * 64, 0, st>>>(a, p.kv.splits); break;                \
            default: cross_attn_bwd_few_keys_kernel<DT, 128, W><<<grid, W * 64, 0, st>>>(a, p.kv.splits);                      \
        }                                                                                                                      \
    } while (0)
        if (p.few == 4) {
            if (c.dt == Q8_BF16) X_FEW(Q8_BF16, 4); else X_FEW(Q8_F16, 4);
        } else {
            if (c.dt == Q8_BF16) X_FEW(Q8_BF16, 8); else X_FEW(Q8_F16, 8);
        }
#undef X_FEW
        if (int e = launch_status(who)) return e;
    }
    if (M && !p.few) {
        a.blocks = (int)p.dq_blocks;
        a.plan = p.dq;
        const unsigned grid = a.plan.grid();
        if (c.dt == Q8_BF16) { X_BWD(cross_attn_dq_kernel, Q8_BF16) } else { X_BWD(cross_attn_dq_kernel, Q8_F16) }
        if (int e = launch_status(who)) return e;
        if (a.plan.parts()) {
            const unsigned n = a.plan.tail * (D / 8);  // 128 rows of D / 4 threads
            if (c.dt == Q8_BF16) cross_attn_add_kernel<Q8_BF16, 1><<<n, 256, 0, st>>>(a);
            else cross_attn_add_kernel<Q8_F16, 1><<<n, 256, 0, st>>>(a);
            if (int e = launch_status(who)) return e;
        }
    }
    if (N) {
        a.blocks = (int)p.kv_blocks;
        a.plan = p.kv;
        if (!p.few) {
            const unsigned grid = a.plan.grid();
            if (c.dt == Q8_BF16) { X_BWD(cross_attn_dkdv_kernel, Q8_BF16) } else { X_BWD(cross_attn_dkdv_kernel, Q8_F16) }
            if (int e = launch_status(who)) return e;
        }
        if (a.plan.parts()) {
            const unsigned n = a.plan.tail * (D / 4);
            if (c.dt == Q8_BF16) cross_attn_add_kernel<Q8_BF16, 2><<<n, 256, 0, st>>>(a);
            else cross_attn_add_kernel<Q8_F16, 2><<<n, 256, 0, st>>>(a);
            if (int e = launch_status(who)) return e;
        }
    }
#undef X_BWD
    return Q8_OK;
}

}  // namespace q8

using namespace q8;

extern "C" int64_t q8_cross_attn_backward_workspace(int64_t B, int H, int Hkv, int M, int N, int D) {
    const char* who = "q8_cross_attn_backward_workspace";
    if (int e = x_sizes(who, Q8_BF16, B, H, Hkv, M, N, D, 1.f)) return e;
    if (!fits(plan(B, H, Hkv, M, N, D))) return fail(Q8_ERR_SHAPE, "%s: sizes out of range", who);
    return whole_bytes(B, H, Hkv, M, N, D);
}

extern "C" int64_t q8_cross_attn_train_backward_workspace(int64_t B, int H, int Hkv, int M, int N, int D) {
    const char* who = "q8_cross_attn_train_backward_workspace";
    if (int e = x_sizes(who, Q8_BF16, B, H, Hkv, M, N, D, 1.f)) return e;
    const XPlan p = plan(B, H, Hkv, M, N, D);
    return fits(p) ? plan_bytes(p) : fail(Q8_ERR_SHAPE, "%s: sizes out of range", who);
}

extern "C" int q8_cross_attn_backward(const void* grad, const int64_t* grad_strides, const void* q, const int64_t* q_strides, const void* k,
                                      const int64_t* k_strides, const void* v, const int64_t* v_strides, const void* o, const int64_t* o_strides,
                                      const float* lse, void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                                      const int64_t* dv_strides, const int32_t* kv_lens, const uint8_t* key_mask, int64_t mask_row_stride, int dt,
                                      float softmax_scale, int64_t B, int H, int Hkv, int M, int N, int D, void* workspace, int64_t workspace_bytes,
                                      q8_stream_t stream) {
    return cross_attn_backward("q8_cross_attn_backward",
                               XBackward{grad, grad_strides, q, q_strides, k, k_strides, v, v_strides, o, o_strides, nullptr, lse, dq, dq_strides, dk, dk_strides, dv,
                                         dv_strides, kv_lens, key_mask, mask_row_stride, dt, softmax_scale, B, H, Hkv, M, N, D, workspace, workspace_bytes,
                                         static_cast<hipStream_t>(stream)});
}

extern "C" int q8_cross_attn_train_backward(const void* grad, const int64_t* grad_strides, const void* q, const int64_t* q_strides, const void* k,
                                            const int64_t* k_strides, const void* v, const int64_t* v_strides, const void* o, const int64_t* o_strides,
                                            const void* o_low, const float* lse, void* dq, const int64_t* dq_strides, void* dk, const int64_t* dk_strides,
                                            void* dv, const int64_t* dv_strides, const int32_t* kv_lens, const uint8_t* key_mask, int64_t mask_row_stride,
                                            int dt, float softmax_scale, int64_t B, int H, int Hkv, int M, int N, int D, void* workspace,
                                            int64_t workspace_bytes, q8_stream_t stream) {
    const char* who = "q8_cross_attn_train_backward";
    if (int e = x_sizes(who, dt, B, H, Hkv, M, N, D, softmax_scale)) return e;
    if (B && M && o_low == nullptr) return fail(Q8_ERR_NULL, "%s: o_low is NULL", who);
    return cross_attn_backward(who, XBackward{grad, grad_strides, q, q_strides, k, k_strides, v, v_strides, o, o_strides, o_low, lse, dq, dq_strides, dk, dk_strides,
                                              dv, dv_strides, kv_lens, key_mask, mask_row_stride, dt, softmax_scale, B, H, Hkv, M, N, D, workspace,
                                              workspace_bytes, static_cast<hipStream_t>(stream)});
}
