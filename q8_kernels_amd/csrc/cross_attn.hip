// 16-bit cross attention, forward: O = softmax(scale Q K^T) V over the keys that count, any number of queries and keys.
//
// One pass over the keys with the running maximum and sum of the softmax. A workgroup holds 128 query rows, 32 a wave; Q^T
// stays in registers, K and V go through LDS in tiles of 64 keys (double-buffered, the next tile's loads in flight during the
// present one's arithmetic). S^T = K Q^T leaves a query's scores in one lane pair, P^T = exp2(S^T c - m) goes on as the B
// operand of O^T = V^T P^T without leaving registers. Scores, maxima, sums and O are fp32; P is rounded to 16 bits for the
// product (as its operand has to be), relative to a maximum that trails the running one by at most 2^8 (fp16: to 2^-7 of it, so
// what is 2^-21 of the largest is still a normal number), so the rounding is a relative one. O is rescaled only when the
// maximum has grown beyond that.
//
// O is divided by the sum of the rounded P, so it is a mean of the values with weights that add up to one: with relative
// roundings r_j it is off by sum_j r_j P_j (v_j - O), not by sum_j r_j P_j v_j, and what a training step forms from it,
// delta = dO . O, by sum_j r_j dS_j. (The log-sum has the sum of the unrounded P, which the backward forms P from.) The
// rounding of O itself would be an error of every score's gradient in the row, which where few keys count or a few take most
// of the row is larger than the gradient's own rounding: 2 to 6 roundings. So a training step keeps 8 bits of what it left off.
//
// Row blocks that do not fill the card: their keys are divided over several workgroups, whose unnormalised results, maxima and
// sums a second kernel joins.
#include "cross_attn_common.h"

#include <type_traits>

namespace q8 {

struct XFwd {
    XTensor q, k, v;
    XOut o;              // p NULL: not wanted
    uint8_t* o_low;      // [units, R, D]: what the rounding of O to 16 bits left off. NULL: not wanted
    float* lse;          // [units, R]: log2 of the sum of exp2 (c s); +inf: no key counts. NULL: not wanted
    XKeys keys;
    float c;             // softmax scale * log2 e
    int Hkv, G, M, D, R;
    int row_blocks;         // of a unit
    XSchedule plan;
    float *part, *pm, *pw, *pl;  // divided blocks: [splits, tail, 128, D], [splits, tail, 128] three times
};

// One wave's rows: Q^T as operands, the running state of their softmax. STATS: the log-sum is wanted.
template <int DT, int DP, bool STATS>
struct Rows32 {
    static constexpr int KS = DP / 16, DTL = DP / 32;
    v4u qf[KS];
    v16f acc[DTL];
    float m, w, l;  // m, less kShiftM, in units of log2; w, l: the sums of P as it is rounded and as it was, over this lane's half of the keys

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int t = 0; t < DTL; ++t) acc[t] = splat16(0.f);
        m = -3.0e38f;
        w = l = 0.f;
    }
    __device__ __forceinline__ void load(const XFwd& a, int b, int hk, int row, int half) {
        const int g = row < a.R ? row / a.M : 0, i = row - g * a.M;
        const uint16_t* p = a.q.p + b * a.q.sb + (int64_t)(hk * a.G + g) * a.q.sh + i * a.q.st + half * 8;
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = (row < a.R && s * 16 + half * 8 < a.D) ? *reinterpret_cast<const v4u*>(p + s * 16) : v4u{0u, 0u, 0u, 0u};
    }
    // One tile of 64 keys: whole (all of them count) or with a bias of 0 and -infinity. copies(i, n): what goes to memory
    // beside group i of the n that form the scores.
    template <typename Copy>
    __device__ __forceinline__ void tile(const uint16_t* kl, const uint16_t* vl, bool whole, const float* bias, float c, const LaneOffsets<DP>& at, int half,
                                         Copy copies) {
        Operands<DP, 4> ops;
        v16f s[2];
        auto scores = [&](auto masked) {
            ops.rows(0, kl, 0, 0, at);
#pragma unroll
            for (int i = 0; i < 2 * ops.RN; ++i) {
                const int u = i / ops.RN, g = i % ops.RN;
                if (i + 1 < 2 * ops.RN) ops.rows((i + 1) & 1, kl, (i + 1) / ops.RN * 32, (i + 1) % ops.RN, at);
                else ops.cols(0, vl, 0, 0, at);
                copies(i, 2 * ops.RN);
                if (g == 0) {
                    if constexpr (masked) s[u] = bias16(bias, u, half);
                    else s[u] = splat16(0.f);
                }
                fence();
#pragma unroll
                for (int j = 0; j < ops.RG; ++j) s[u] = mfma16<DT>(ops.f[i & 1][j], qf[g * ops.RG + j], s[u]);
                fence();
            }
        };
        if (whole) scores(std::false_type{});
        else scores(std::true_type{});
        float top = s[0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = max_ieee(top, s[0][i]);
#pragma unroll
        for (int i = 0; i < 16; ++i) top = max_ieee(top, s[1][i]);
        top = half_pair_max(top) * c;
        const bool grown = top > m + (8 + kShiftM<DT>);
        if (__builtin_amdgcn_ballot_w64(grown) != 0) {
            const float next = grown ? top - kShiftM<DT> : m, f = __builtin_amdgcn_exp2f(m - next);
            m = next;
            w *= f;
            if constexpr (STATS) l *= f;
#pragma unroll
            for (int d = 0; d < DTL; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[d][i] *= f;
        }
        auto weights = [&](int u) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], c, -m));
                if constexpr (STATS) l += s[u][i];
            }
        };
        weights(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const v4u p = pack_step<DT>(s[i / 2], i % 2);
            if (i < 3) ops.cols((i + 1) & 1, vl, (i + 1) * 16, 0, at);
            fence();
            if (i == 0) weights(1);  // beside the matrix instructions of the first half
#pragma unroll
            for (int d = 0; d < DTL; ++d) acc[d] = mfma16<DT>(ops.f[i & 1][d], p, acc[d]);
#pragma unroll
            for (int j = 0; j < 4; ++j) w = add_pair<DT>(p[j], w);
            if (i == 0) {
#pragma unroll
                for (int d = 0; d < DTL; ++d) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x402, 48 / DTL, 0);
                }
            }
            fence();
        }
    }
    // the sums over all keys
    static __device__ __forceinline__ float both_halves(float x) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    __device__ __forceinline__ void join_halves() {
        w = both_halves(w);
        if constexpr (STATS) l = both_halves(l);
    }
    // log-sum and O
    __device__ __forceinline__ void finish(const XFwd& a, int unit, int b, int hk, int row, int lane) const {
        const bool in = row < a.R;
        const int64_t at = (int64_t)unit * a.R + row;
        if constexpr (STATS) {
            if (in && lane < 32) a.lse[at] = l == 0.f ? __builtin_inff() : m + __builtin_log2f(l);
        }
        const int g = in ? row / a.M : 0;
        const float inv = w == 0.f ? 0.f : 1.0f / w;
        if (a.o.p != nullptr) store_rows<DT, DP>(acc, inv, in ? a.o.p + b * a.o.sb + (int64_t)(hk * a.G + g) * a.o.sh + (row - g * a.M) * a.o.st : nullptr, a.D, lane);
        if (a.o_low != nullptr) store_rests<DT, DP>(acc, inv, in ? a.o_low + at * a.D : nullptr, a.D, lane);
    }
};

// us: 2 x 16 heads of 128 on 4, 4096 x 4096 fp16 298, with the log-sum and the rest of O 313, bf16 with both 303 to 318 (860 to 910
// TFLOP/s; the matrix pipes are busy 45 % of the time, the vector units 52 %; the matrix instructions alone would take 131 at 2.1 GHz, a
// rate that their own load does not leave the clock at); 2 x 16 of 64 on 4, 4096 x 4096 bf16 186, with both 190; 8 single tokens, 32 heads
// of 128 on 8, 8192 ragged keys bf16 28 to 38 (4.0 to 5.3 TB/s of keys and values: HBM).
template <int DT, int DP, bool STATS>
__global__ __launch_bounds__(kXThreads, 2) void cross_attn_fwd_kernel(XFwd a) {
    constexpr int ELEMS = kXTile * DP;
    __shared__ __align__(16) uint16_t k0[ELEMS], k1[ELEMS], v0[ELEMS], v1[ELEMS];
    __shared__ __align__(16) float bias0[kXTile], bias1[kXTile];
    unsigned block;
    int split, of;
    if (!a.plan.item(block, split, of)) return;
    const int unit = block / a.row_blocks, rb = block - unit * a.row_blocks;
    const int b = unit / a.Hkv, hk = unit - b * a.Hkv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int row0 = rb * kXRows + wave * 32, row = row0 + (lane & 31);

    Rows32<DT, DP, STATS> rows;
    rows.load(a, b, hk, row, half);
    KVTiles<DP> kv;
    kv.len = a.keys.length(b);
    kv.mask = a.keys.row(b);
    kv.copies.D = a.D;
    kv.copies.wave = wave;
    kv.kp = a.k.p + b * a.k.sb + hk * a.k.sh;
    kv.vp = a.v.p + b * a.v.sb + hk * a.v.sh;
    kv.kst = a.k.st;
    kv.vst = a.v.st;
    const int tiles = (kv.len + kXTile - 1) / kXTile, per = (tiles + of - 1) / of;
    const int t0 = split * per, t1 = t0 + per < tiles ? t0 + per : tiles;
    if (t0 < t1) kv.first(t0, k0, v0, bias0);
    rows.clear();
    wait_loads();
    __syncthreads();

    LaneOffsets<DP> at(lane);
    auto step = [&](int t, auto buffer, auto with_rows) {
        constexpr int BUF = decltype(buffer)::value;
        at.fresh();
        // (past the last tile of this workgroup the copies are of a tile that nobody reads, or empty)
        kv.bias_of(kv.live[1], BUF ? bias0 : bias1);
        kv.ask(t + 2);
        const XTile knext = kv.k_tile(t + 1), vnext = kv.v_tile(t + 1);
        auto copies = [&](int i, int n) { kv.copies.group(i, n, knext, vnext, ~kv.live[1], BUF ? k0 : k1, BUF ? v0 : v1); };
        if constexpr (with_rows) rows.tile(BUF ? k1 : k0, BUF ? v1 : v0, kv.live[0] == ~(uint64_t)0, BUF ? bias1 : bias0, a.c, at, half, copies);
        else copies(0, 1);
        kv.end(t);
        __syncthreads();
    };
    auto walk = [&](auto with_rows) {
        for (int t = t0; t < t1; t += 2) {
            step(t, std::integral_constant<int, 0>{}, with_rows);
            if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{}, with_rows);
        }
    };
    // a wave without rows only copies (it meets the same barriers: they count waves)
    if (row0 < a.R) walk(std::true_type{});
    else walk(std::false_type{});
    rows.join_halves();
    const XFwd& z = arguments_again<XFwd>();
    if (of > 1) {
        if (row < z.R) {
            const int64_t to = ((int64_t)split * z.plan.tail + (block - z.plan.full)) * kXRows + wave * 32 + (lane & 31);
            if (half == 0) {
                z.pm[to] = rows.m;
                z.pw[to] = rows.w;
                if constexpr (STATS) z.pl[to] = rows.l;
            }
            float* p = z.part + to * z.D;
#pragma unroll
            for (int d = 0; d < rows.DTL; ++d)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = d * 32 + i * 8 + half * 4;
                    if (e < z.D) *reinterpret_cast<v4f*>(p + e) = v4f{rows.acc[d][4 * i], rows.acc[d][4 * i + 1], rows.acc[d][4 * i + 2], rows.acc[d][4 * i + 3]};
                }
        }
        return;
    }
    rows.finish(z, unit, b, hk, row, lane);
}

// Few keys (NT tiles at most): all of K and V stay in LDS, and a workgroup walks over the rows of its unit instead, each wave
// by itself, without a barrier; the next 32 rows of Q are on their way meanwhile. The kernel above would fill LDS again for
// every 128 rows. bf16, 2 x 32 heads of 64: 6144 x 128 keys (NT = 2, three workgroups on a CU) 32 us here and 40 there (ragged lengths
// 31, 40), 6144 x 256 keys (NT = 4, two workgroups) 52 and 53 (ragged 40, 52).
template <int DT, int DP, int NT, bool STATS>
__global__ __launch_bounds__(kXThreads, 2) void cross_attn_few_keys_kernel(XFwd a, int parts) {
    constexpr int ELEMS = kXTile * DP, KS = DP / 16;
    __shared__ __align__(16) uint16_t k[NT * ELEMS], v[NT * ELEMS];
    __shared__ __align__(16) float bias[NT * kXTile];
    const int unit = blockIdx.x / parts, part = blockIdx.x - unit * parts;
    const int b = unit / a.Hkv, hk = unit - b * a.Hkv;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int step = parts * kXRows;
    int row = part * kXRows + wave * 32 + (lane & 31);

    Rows32<DT, DP, STATS> rows;
    rows.load(a, b, hk, row, half);
    KVTiles<DP> kv;
    kv.len = a.keys.length(b);
    kv.mask = a.keys.row(b);
    kv.copies.D = a.D;
    kv.copies.wave = wave;
    kv.kp = a.k.p + b * a.k.sb + hk * a.k.sh;
    kv.vp = a.v.p + b * a.v.sb + hk * a.v.sh;
    kv.kst = a.k.st;
    kv.vst = a.v.st;
    const int tiles = (kv.len + kXTile - 1) / kXTile;  // at most NT
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t >= tiles) break;
        if (kv.mask != nullptr) kv.ask(t);
        const uint64_t live = kv.counted(t);
        kv.copies.group(0, 1, kv.k_tile(t), kv.v_tile(t), ~live, k + t * ELEMS, v + t * ELEMS);
        if (threadIdx.x < kXTile) bias[t * kXTile + threadIdx.x] = (live >> threadIdx.x) & 1 ? 0.f : -__builtin_inff();
    }
    wait_loads();
    __syncthreads();

    LaneOffsets<DP> at(lane);
    for (int row0 = part * kXRows + wave * 32; row0 < a.R; row0 += step, row += step) {
        Rows32<DT, DP, STATS> ahead;
        ahead.load(a, b, hk, row + step, half);
        rows.clear();
        for (int t = 0; t < tiles; ++t) {
            at.fresh();
            rows.tile(k + t * ELEMS, v + t * ELEMS, kv.mask == nullptr && (t + 1) * kXTile <= kv.len, bias + t * kXTile, a.c, at, half, [](int, int) {});
        }
        rows.join_halves();
        rows.finish(a, unit, b, hk, row, lane);
#pragma unroll
        for (int s = 0; s < KS; ++s) rows.qf[s] = ahead.qf[s];
    }
}

// Joins the parts of a row: weights exp2(m_i - max m). D / 4 threads a row, 4 elements each, BATCH parts at a time, their loads
// all under way together. Two parts of 2 x 23732 rows of 64: 7.9 us (30 MB; with batches
// of 8 for them too 9.7), 8 parts of 8 x 1024 rows of 128 5.6 us.
template <int DT, int BATCH>
__global__ __launch_bounds__(256) void cross_attn_join_kernel(XFwd a) {
    const unsigned lanes = (unsigned)a.D / 4, id = blockIdx.x * 256 + threadIdx.x, n = id / lanes, all = a.plan.tail * kXRows;
    const unsigned tail = n / kXRows, block = a.plan.full + tail;
    const int unit = block / a.row_blocks, r = (int)(block - unit * a.row_blocks) * kXRows + (int)(n - tail * kXRows);
    if (n >= all || r >= a.R) return;
    const int e = (int)(id - n * lanes) * 4;
    float m = -3.0e38f, w = 0.f, l = 0.f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
    const float* pls = a.lse != nullptr ? a.pl : a.pw;  // (without a log-sum: anything)
    for (int i0 = 0; i0 < a.plan.splits; i0 += BATCH) {
        float pm[BATCH], pw[BATCH], pl[BATCH];
        v4f po[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const bool in = i0 + i < a.plan.splits;
            const int64_t at = (int64_t)(in ? i0 + i : i0) * all + n;
            pm[i] = in ? a.pm[at] : -3.0e38f;
            pw[i] = in ? a.pw[at] : 0.f;
            pl[i] = in ? pls[at] : 0.f;
            po[i] = *reinterpret_cast<const v4f*>(a.part + at * a.D + e);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) top = max_ieee(top, pm[i]);
        const float f = __builtin_amdgcn_exp2f(m - top);
        m = top;
        w *= f;
        l *= f;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] *= f;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const float share = i0 + i < a.plan.splits ? __builtin_amdgcn_exp2f(pm[i] - m) : 0.f;
            w += share * pw[i];
            l += share * pl[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += share * po[i][j];
        }
    }
    if (a.lse != nullptr && e == 0) a.lse[(int64_t)unit * a.R + r] = l == 0.f ? __builtin_inff() : m + __builtin_log2f(l);
    const float inv = w == 0.f ? 0.f : 1.0f / w;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] *= inv;
    const int g = r / a.M, b = unit / a.Hkv, hk = unit - b * a.Hkv;
    const uint32_t x = pack2<DT>(o[0], o[1]), y = pack2<DT>(o[2], o[3]);
    if (a.o.p != nullptr) *reinterpret_cast<v2i*>(a.o.p + b * a.o.sb + (int64_t)(hk * a.G + g) * a.o.sh + (int64_t)(r - g * a.M) * a.o.st + e) = v2i{(int)x, (int)y};
    if (a.o_low != nullptr)
        *reinterpret_cast<uint32_t*>(a.o_low + ((int64_t)unit * a.R + r) * a.D + e) = rests_of<DT>(o[0], o[1], o[2], o[3], x, y);
}

// The kernel for few keys: 256 for heads up to 64, 128 for longer ones (two workgroups on a CU, by LDS), and how many of its
// workgroups run at once. bf16, us, this kernel and the general one, heads of 64: 2 x 32, 6144 x 128 31.7, 39.9; 6144 x 256 51.7, 52.5;
// 32 x 32, 64 x 64 11.8, 13.0; 64 x 32 on 8, 1 x 100 6.6, 7.0; the other way round 16, 1024 x 128 6.9, 6.4 and 16 x 16, 300 x 128 12.0, 11.4.
// Of 128: 2 x 32, 6144 x 128 64, 67; 32, 1 x 128 7.2, 7.5. Of 96: 2 x 32, 6144 x 128 48, 61; 32 x 32, 64 x 64 16.9, 16.6; 13 x 16 on 8,
// 3610 x 1 109, 89.
static bool few_keys(int N, int D) { return N <= (D <= 64 ? 4 : 2) * kXTile; }
static int few_blocks(int N, int D) { return D <= 64 && N <= 2 * kXTile ? 768 : 512; }

static XSchedule fwd_plan(int64_t units, int64_t rows, int N, int D) {
    // workgroups that run at once, by the registers of a lane
    return schedule(units * ((rows + kXRows - 1) / kXRows), N, D <= 32 ? 1024 : D <= 64 ? 768 : 512, (double)(rows < kXRows ? rows : kXRows) * D);
}

static int64_t part_bytes(const XSchedule& plan, int D) { return plan.parts() * kXRows * (D + 3) * (int64_t)sizeof(float); }

int64_t cross_attn_forward_workspace(int64_t B, int H, int Hkv, int M, int N, int D) {
    return few_keys(N, D) ? 0 : part_bytes(fwd_plan(B * Hkv, (int64_t)(H / Hkv) * M, N, D), D);
}

int cross_attn_forward(const char* who, const XForward& c) {
    if (int e = x_sizes(who, c.dt, c.B, c.H, c.Hkv, c.M, c.N, c.D, c.softmax_scale)) return e;
    const int N = c.N, D = c.D;
    if (c.B == 0 || c.M == 0) return Q8_OK;
    if (int e = x_tensor(who, "q", c.q, c.q_strides, c.B, c.H, c.M, D)) return e;
    if (c.o != nullptr || c.o_low == nullptr)
        if (int e = x_tensor(who, "o", c.o, c.o_strides, c.B, c.H, c.M, D)) return e;
    if (N) {
        if (int e = x_tensor(who, "k", c.k, c.k_strides, c.B, c.Hkv, N, D)) return e;
        if (int e = x_tensor(who, "v", c.v, c.v_strides, c.B, c.Hkv, N, D)) return e;
    }
    if (!aligned16(c.o_low)) return fail(Q8_ERR_ALIGN, "%s: o_low must be 16-byte aligned", who);
    if ((reinterpret_cast<uintptr_t>(c.lse) & 3) || (reinterpret_cast<uintptr_t>(c.kv_lens) & 3)) return fail(Q8_ERR_ALIGN, "%s: lse or kv_lens not aligned", who);
    if (c.key_mask && (c.mask_row_stride < 0 || (c.B > 1 && c.mask_row_stride > INT64_MAX / 2 / c.B))) return fail(Q8_ERR_SHAPE, "%s: row stride of the mask", who);
    XFwd a{};
    static const int64_t none[3] = {0, 0, 0};
    const int64_t *ks = N ? c.k_strides : none, *vs = N ? c.v_strides : none, *os = c.o ? c.o_strides : none;
    a.q = XTensor{static_cast<const uint16_t*>(c.q), c.q_strides[0], c.q_strides[1], c.q_strides[2]};
    a.k = XTensor{static_cast<const uint16_t*>(c.k), ks[0], ks[1], ks[2]};
    a.v = XTensor{static_cast<const uint16_t*>(c.v), vs[0], vs[1], vs[2]};
    a.o = XOut{static_cast<uint16_t*>(c.o), os[0], os[1], os[2]};
    a.o_low = static_cast<uint8_t*>(c.o_low);
    a.lse = c.lse;
    a.keys = XKeys{c.kv_lens, c.key_mask, c.mask_row_stride, N};
    a.c = c.softmax_scale * kLog2e;
    a.Hkv = c.Hkv;
    a.G = c.H / c.Hkv;
    a.M = c.M;
    a.D = D;
    a.R = a.G * c.M;
    a.row_blocks = (a.R + kXRows - 1) / kXRows;
    const int64_t units = c.B * c.Hkv;
    if (units * a.row_blocks > kXMostBlocks) return fail(Q8_ERR_SHAPE, "%s: too many rows", who);
    const bool stats = c.lse != nullptr, bf16 = c.dt == Q8_BF16;
    if (few_keys(N, D)) {
        const int64_t parts = walk_parts(units, a.row_blocks, few_blocks(N, D), 1);
        if (units * parts > kXMostBlocks) return fail(Q8_ERR_SHAPE, "%s: too many heads", who);
        const unsigned grid = (unsigned)(units * parts);
#define X_FEW(DT, NT, STATS)                                                                                               \
    do {                                                                                                                   \
        if (D <= 32) cross_attn_few_keys_kernel<DT, 32, NT, STATS><<<grid, kXThreads, 0, c.stream>>>(a, (int)parts);       \
        else if (D <= 64) cross_attn_few_keys_kernel<DT, 64, NT, STATS><<<grid, kXThreads, 0, c.stream>>>(a, (int)parts);  \
        else if (D <= 96) cross_attn_few_keys_kernel<DT, 96, 2, STATS><<<grid, kXThreads, 0, c.stream>>>(a, (int)parts);   \
        else cross_attn_few_keys_kernel<DT, 128, 2, STATS><<<grid, kXThreads, 0, c.stream>>>(a, (int)parts);               \
    } while (0)
#define X_FEW_TYPE(NT, STATS)                                                       \
    do {                                                                            \
        if (bf16) X_FEW(Q8_BF16, NT, STATS); else X_FEW(Q8_F16, NT, STATS);         \
    } while (0)
        if (N <= 2 * kXTile) {
            if (stats) X_FEW_TYPE(2, true); else X_FEW_TYPE(2, false);
        } else {
            if (stats) X_FEW_TYPE(4, true); else X_FEW_TYPE(4, false);
        }
#undef X_FEW_TYPE
#undef X_FEW
        return launch_status(who);
    }
    a.plan = fwd_plan(units, a.R, N, D);
    if (a.plan.parts()) {
        const int64_t need = part_bytes(a.plan, D), n = a.plan.parts() * kXRows;
        if (c.workspace == nullptr) return fail(Q8_ERR_NULL, "%s: a workspace of %lld bytes is needed", who, (long long)need);
        if (c.workspace_bytes < need) return fail(Q8_ERR_SHAPE, "%s: workspace of %lld bytes, %lld needed", who, (long long)c.workspace_bytes, (long long)need);
        if (!aligned16(c.workspace)) return fail(Q8_ERR_ALIGN, "%s: workspace must be 16-byte aligned", who);
        a.part = static_cast<float*>(c.workspace);
        a.pm = a.part + n * D;
        a.pw = a.pm + n;
        a.pl = a.pw + n;
    }
    const unsigned grid = a.plan.grid();
#define X_FWD(DT, STATS)                                                                              \
    switch (padded_head(D)) {                                                                         \
        case 32: cross_attn_fwd_kernel<DT, 32, STATS><<<grid, kXThreads, 0, c.stream>>>(a); break;    \
        case 64: cross_attn_fwd_kernel<DT, 64, STATS><<<grid, kXThreads, 0, c.stream>>>(a); break;    \
        case 96: cross_attn_fwd_kernel<DT, 96, STATS><<<grid, kXThreads, 0, c.stream>>>(a); break;    \
        default: cross_attn_fwd_kernel<DT, 128, STATS><<<grid, kXThreads, 0, c.stream>>>(a);          \
    }
    if (bf16) {
        if (stats) { X_FWD(Q8_BF16, true) } else { X_FWD(Q8_BF16, false) }
    } else {
        if (stats) { X_FWD(Q8_F16, true) } else { X_FWD(Q8_F16, false) }
    }
#undef X_FWD
    if (int e = launch_status(who)) return e;
    if (a.plan.parts()) {
        const unsigned n = a.plan.tail * (D / 8);  // 128 rows of D / 4 threads
        const bool two = a.plan.splits == 2;
        if (bf16) { if (two) cross_attn_join_kernel<Q8_BF16, 2><<<n, 256, 0, c.stream>>>(a); else cross_attn_join_kernel<Q8_BF16, 8><<<n, 256, 0, c.stream>>>(a); }
        else { if (two) cross_attn_join_kernel<Q8_F16, 2><<<n, 256, 0, c.stream>>>(a); else cross_attn_join_kernel<Q8_F16, 8><<<n, 256, 0, c.stream>>>(a); }
        return launch_status(who);
    }
    return Q8_OK;
}

}  // namespace q8

using namespace q8;

extern "C" int64_t q8_cross_attn_workspace(int64_t B, int H, int Hkv, int M, int N, int D) {
    if (int e = x_sizes("q8_cross_attn_workspace", Q8_BF16, B, H, Hkv, M, N, D, 1.f)) return e;
    return cross_attn_forward_workspace(B, H, Hkv, M, N, D);
}

extern "C" int q8_cross_attn(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                             void* o, const int64_t* o_strides, float* lse, const int32_t* kv_lens, const uint8_t* key_mask, int64_t mask_row_stride,
                             int dt, float softmax_scale, int64_t B, int H, int Hkv, int M, int N, int D, void* workspace, int64_t workspace_bytes,
                             q8_stream_t stream) {
    return cross_attn_forward("q8_cross_attn", XForward{q, q_strides, k, k_strides, v, v_strides, o, o_strides, nullptr, lse, kv_lens, key_mask, mask_row_stride, dt,
                                                        softmax_scale, B, H, Hkv, M, N, D, workspace, workspace_bytes, static_cast<hipStream_t>(stream)});
}

extern "C" int q8_cross_attn_train(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                   void* o, const int64_t* o_strides, void* o_low, float* lse, const int32_t* kv_lens, const uint8_t* key_mask,
                                   int64_t mask_row_stride, int dt, float softmax_scale, int64_t B, int H, int Hkv, int M, int N, int D, void* workspace,
                                   int64_t workspace_bytes, q8_stream_t stream) {
    const char* who = "q8_cross_attn_train";
    if (int e = x_sizes(who, dt, B, H, Hkv, M, N, D, softmax_scale)) return e;
    if (B && M && (o == nullptr || o_low == nullptr || lse == nullptr)) return fail(Q8_ERR_NULL, "%s: o, o_low and lse are needed", who);
    return cross_attn_forward(who, XForward{q, q_strides, k, k_strides, v, v_strides, o, o_strides, o_low, lse, kv_lens, key_mask, mask_row_stride, dt,
                                            softmax_scale, B, H, Hkv, M, N, D, workspace, workspace_bytes, static_cast<hipStream_t>(stream)});
}
