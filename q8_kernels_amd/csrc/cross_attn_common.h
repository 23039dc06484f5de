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
// Tiles in LDS are row-major with rows of DP elements (DP: the head size D padded to 32, 64, 96 or 128) in 16-byte chunks, chunk
// c of row r at c ^ f(r) (tile_at). LDS serves 16 lanes x 16 bytes, or 32 lanes x 8 bytes, at a time from 64 banks: the
// operand reads take one chunk of 16 consecutive rows, the transposing reads 4 aligned chunks of 4 consecutive rows, and f
// spreads either over all banks (rows padded by 32 bytes instead: 40 % of the LDS cycles were bank conflicts).
#pragma once
#include "q8_common.h"
#include "q8_host.h"

namespace q8 {

constexpr int kXThreads = 256, kXWaves = 4, kXTile = 64, kXRows = 128;  // a workgroup; rows of a staged tile; rows (keys) a workgroup owns, 32 a wave
constexpr int64_t kXMostBlocks = 0xff0000;  // workgroups of a launch: below 2^32 threads, with room for the divided walks
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
// fp16 has its normal numbers down to 2^-14 only: probabilities enter their products times 2^kShiftP (backward, where they are at
// most 1) or relative to 2^-kShiftM of the maximum (forward, where they are at most 2^8 beside it). bf16 has fp32's range.
template <int DT>
constexpr int kShiftP = DT == Q8_F16 ? 14 : 0;
template <int DT>
constexpr int kShiftM = DT == Q8_F16 ? 7 : 0;
template <int DT>
__device__ __forceinline__ float unpack(uint32_t h) { return DT == Q8_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h); }
// c + both values of a pair: exact products, one fp32 rounding to nearest
template <int DT>
__device__ __forceinline__ float add_pair(uint32_t p, float c) {
    if constexpr (DT == Q8_BF16) {
        typedef __bf16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, 0x3f803f80u), c, false);
    } else {
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, 0x3c003c00u), c, false);
    }
}
// c + the squares of both values of a pair
template <int DT>
__device__ __forceinline__ float square_sum(uint32_t p, float c) {
    if constexpr (DT == Q8_BF16) {
        typedef __bf16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, p), c, false);
    } else {
        typedef _Float16 v2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, p), c, false);
    }
}
// What rounding x to 16 bits, code h, left off, as one byte: 8 bits more of the mantissa, signed (values next to a tie give the
// nearest byte there is). fp32 codes of one sign are in the order of their values, so it is a difference of codes, and with_rest
// is an addition to one. fp16 below 2^-14, whose step is 2^-24 whatever the value, gets the largest byte where that does not
// reach: some of the way. (The difference to zero is 0 or more, so zero's byte is.)
template <int DT>
constexpr int kRestShift = DT == Q8_BF16 ? 8 : 5;
template <int DT>
__device__ __forceinline__ uint32_t rest_of(float x, uint32_t h) {  // in bits 8 .. 15
    constexpr int up = 8 - kRestShift<DT>, most = 0x7f7f >> up, least = -(0x8000 >> up);
    const int d = (int)(__float_as_uint(x) - __float_as_uint(unpack<DT>(h)));
    return ((uint32_t)(d < least ? least : d < most ? d : most) << up) + 0x80u;
}
template <int DT>
__device__ __forceinline__ float with_rest(uint32_t h, uint32_t bytes, int k) {
    return __uint_as_float(__float_as_uint(unpack<DT>(h)) + (uint32_t)(((int)(bytes << (24 - 8 * k)) >> 24) << kRestShift<DT>));
}
// the bytes of x0 .. x3, whose codes are in lo and hi
template <int DT>
__device__ __forceinline__ uint32_t rests_of(float x0, float x1, float x2, float x3, uint32_t lo, uint32_t hi) {
    const uint32_t a = __builtin_amdgcn_perm(rest_of<DT>(x1, lo >> 16), rest_of<DT>(x0, lo & 0xffffu), 0x0c0c0501u);
    const uint32_t b = __builtin_amdgcn_perm(rest_of<DT>(x3, hi >> 16), rest_of<DT>(x2, hi & 0xffffu), 0x05010c0cu);
    return a | b;
}

__device__ __forceinline__ v16f splat16(float v) {
    v16f r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = v;
    return r;
}

template <int DP>
__device__ __forceinline__ int tile_f(int r) {
    return DP == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : DP == 64 ? ((r & 2) << 1) | ((r >> 2) & 3) : (r >> 2) & 3;
}
// element offset of chunk c of row r
template <int DP>
__device__ __forceinline__ int tile_at(int r, int c) { return r * DP + ((c ^ tile_f<DP>(r)) << 3); }
// A lane's byte offsets in a tile, for its chunk of elements 0 .. 15 (rows) and columns 0 .. 31 (cols). The other operands
// are an XOR of a constant away (an addition where f leaves the bits alone), which is cheaper than keeping 16 addresses in
// registers: fresh() keeps the compiler from doing that.
template <int DP>
struct LaneOffsets {
    unsigned rows, cols;
    __device__ __forceinline__ explicit LaneOffsets(int lane) {
        rows = (unsigned)tile_at<DP>(lane & 31, lane >> 5) * 2u;
        cols = (unsigned)tile_at<DP>(((lane >> 5) << 2) + ((lane & 15) >> 2), ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) * 2u + ((lane & 1) << 3);
    }
    __device__ __forceinline__ void fresh() {
        asm volatile("" : "+v"(rows));
        asm volatile("" : "+v"(cols));
    }
};
// A operand: rows row0 + l % 32 (row0 a multiple of 32), elements 16 s + 8 (l / 32) .. + 7
template <int DP>
__device__ __forceinline__ v4u lds_rows(const uint16_t* tile, int row0, int s, const LaneOffsets<DP>& at) {
    const unsigned o = DP == 96 ? (at.rows ^ ((s & 1) << 5)) + ((s >> 1) << 6) : at.rows ^ (s << 5);
    return *reinterpret_cast<const v4u*>(reinterpret_cast<const char*>(tile + row0 * DP) + o);
}
// A operand of the transposed tile: column 32 d + l % 32 over the 16 rows from row0 (a multiple of 16), in the order of a
// score column's results: 4 rows, and the 4 rows 8 further, where f differs in its second bit
template <int DP>
__device__ __forceinline__ v4u lds_cols(const uint16_t* tile, int row0, int d, const LaneOffsets<DP>& at) {
    const unsigned o = DP == 96 ? at.cols + (d << 6) : at.cols ^ (d << 6);
    const char* p = reinterpret_cast<const char*>(tile + row0 * DP);
    const v4s16 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s16*)(p + o));
    const v4s16 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s16*)(p + 16 * DP + (o ^ 32u)));
    const v2i x = __builtin_bit_cast(v2i, a), y = __builtin_bit_cast(v2i, b);
    return v4u{(unsigned)x[0], (unsigned)x[1], (unsigned)y[0], (unsigned)y[1]};
}

// Operands of a group of matrix instructions (at most G), read one group ahead of their use: left alone, the compiler reads
// each right before its instruction, which then waits out the LDS latency. fence() keeps the groups apart.
template <int DP, int G>
struct Operands {
    static constexpr int KS = DP / 16, DTL = DP / 32;
    static constexpr int RG = KS <= G ? KS : KS % G == 0 ? G : 3, CG = DTL <= G ? DTL : DTL % G == 0 ? G : 1;  // instructions of a group
    static constexpr int RN = KS / RG, CN = DTL / CG;  // groups of a product over the head, and of one over 16 rows
    static_assert(RG * RN == KS && CG * CN == DTL, "whole groups");
    v4u f[2][RG > CG ? RG : CG];
    __device__ __forceinline__ void rows(int to, const uint16_t* tile, int row0, int group, const LaneOffsets<DP>& at) {
#pragma unroll
        for (int j = 0; j < RG; ++j) f[to][j] = lds_rows<DP>(tile, row0, group * RG + j, at);
    }
    __device__ __forceinline__ void cols(int to, const uint16_t* tile, int row0, int group, const LaneOffsets<DP>& at) {
#pragma unroll
        for (int j = 0; j < CG; ++j) f[to][j] = lds_cols<DP>(tile, row0, group * CG + j, at);
    }
};
// The kernel's arguments (its first parameter) read again from memory: what is only needed behind a loop then takes no scalar
// registers in it (they are spilled into vector registers otherwise, and read back in every turn).
template <typename Args>
__device__ __forceinline__ const Args& arguments_again() {
    auto p = (const __attribute__((address_space(4))) Args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Args*)p;
}
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// Waits until at most LEFT (below 16) of the loads and copies so far are under way.
template <int LEFT = 0>
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70 | LEFT); }

// A barrier that leaves copies under way (__syncthreads waits for all of them): LDS accesses before it are done, and the
// compiler moves none across it.
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The B operand that results 8 s .. 8 s + 7 of a score column make
template <int DT>
__device__ __forceinline__ v4u pack_step(const v16f& v, int s) {
    return v4u{pack2<DT>(v[8 * s], v[8 * s + 1]), pack2<DT>(v[8 * s + 2], v[8 * s + 3]), pack2<DT>(v[8 * s + 4], v[8 * s + 5]),
               pack2<DT>(v[8 * s + 6], v[8 * s + 7])};
}

// Copies of TR rows to an LDS tile that do not pass through registers: one fills 64 consecutive 16-byte places with the rows
// from 64 / CPR * idx on; the chunk that belongs into a place is chosen by the lane's source offset. They are buffer loads:
// what lies outside the tile's bytes (rows past the end, and the offsets given to chunks past the head size and to rows that
// do not count) comes as zeros and is not read. So a copy is one instruction whatever the tile, without a branch, which
// would make the compiler wait for every LDS read under way at its end. They are done after wait_loads.
//
// Two tensors (K and V, or Q and dO) go together: a wave's share of both is COPIES instructions, which are spread over the
// work on the tile before, because a burst of them stops the wave until the memory path has taken them.
struct XTile {
    __amdgpu_buffer_rsrc_t bytes;
    unsigned st2;  // bytes between rows
    __device__ __forceinline__ XTile(const uint16_t* base, int64_t st, int rows, int D, int most = kXTile) {
        const int n = rows < most ? rows : most;
        st2 = (unsigned)st * 2u;  // (st below 2^24: a tile stays below 2^31 bytes)
        bytes = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, n > 0 ? (int)((unsigned)(n - 1) * st2 + (unsigned)D * 2u) : 0, 0x00020000);
    }
};
template <int DP, int TR = kXTile, int W = kXWaves>
struct Copies {
    static constexpr int CPR = DP / 8, ALONE = TR * CPR / 64, COPIES = 2 * ALONE / W;
    static constexpr bool EVEN = 64 % CPR == 0;  // a copy is whole rows
    static_assert(2 * ALONE % W == 0, "whole copies for every wave");
    int wave, D;
    // copy idx (0 .. ALONE - 1) of a tile; rows with a bit in `dead` become zeros
    __device__ __forceinline__ void one(const XTile& x, int idx, uint64_t dead, uint16_t* tile) const {
        const int lane = threadIdx.x & 63;
        const int row = EVEN ? lane / CPR : (idx * 64 + lane) / CPR;  // EVEN: of the copy
        // (idx is wave + a multiple of 4, and f looks at rows modulo 16: the lane's part is the same for all its copies)
        const int f = EVEN ? tile_f<DP>((wave & 3) * (64 / CPR) + row) : tile_f<DP>(row);
        const int chunk = (EVEN ? lane % CPR : (idx * 64 + lane) % CPR) ^ f;
        unsigned off = (unsigned)row * x.st2 + (chunk * 8 < D ? (unsigned)chunk * 16u : 0x80000000u);
        const int row0 = EVEN ? idx * (64 / CPR) : 0;
        off += (unsigned)row0 * x.st2;
        if constexpr (EVEN) {
            const int word = row0 < 32 ? (int)dead : (int)(dead >> 32);  // a copy's rows lie in one half of the tile
            off |= (unsigned)__builtin_amdgcn_sbfe(word, (unsigned)((row0 & 31) + row), 1u);
        } else {
            off |= (dead >> row) & 1 ? ~0u : 0u;
        }
        __builtin_amdgcn_raw_ptr_buffer_load_lds(x.bytes, (__attribute__((address_space(3))) void*)(tile + idx * 512), 16, (int)off, 0, 0, 0);
    }
    // share i of the wave's COPIES
    __device__ __forceinline__ void share(int i, const XTile& x, const XTile& y, uint64_t dead, uint16_t* xt, uint16_t* yt) const {
        const int idx = wave + i * W;
        if (idx < ALONE) one(x, idx, dead, xt);
        else one(y, idx - ALONE, dead, yt);
    }
    // the shares that go with group g of `of`
    __device__ __forceinline__ void group(int g, int of, const XTile& x, const XTile& y, uint64_t dead, uint16_t* xt, uint16_t* yt) const {
#pragma unroll
        for (int i = 0; i < COPIES; ++i)
            if (i * of / COPIES == g) share(i, x, y, dead, xt, yt);
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

// K and V in tiles of 64 keys, in two buffers: while one tile is worked on, the next one's copies run, and the mask bytes of
// the one after that are on their way, for the copies have to know which keys count. The buffers are arrays of their own: the
// compiler waits for all copies before a read of LDS that it cannot tell from their targets.
template <int DP>
struct KVTiles {
    static constexpr int ELEMS = kXTile * DP;
    Copies<DP> copies;
    const uint16_t *kp, *vp;
    int64_t kst, vst;
    const uint8_t* mask;
    int len;
    uint8_t byte;
    uint64_t live[2];  // of the present tile and of the next one
    // requests the mask bytes of tile t (any t: of an existing key)
    __device__ __forceinline__ void ask(int t) {
        const int key = t * kXTile + (int)(threadIdx.x & 63), last = len - 1;  // (t0 < t1: len is 1 or more)
        // (without a mask some byte of K: a load under a condition would be waited for at its end)
        byte = *(mask != nullptr ? mask + (key < last ? key : last) : reinterpret_cast<const uint8_t*>(kp));
    }
    // which keys of tile t count, from its bytes
    __device__ __forceinline__ uint64_t counted(int t) const {
        return __builtin_amdgcn_ballot_w64(t * kXTile + (int)(threadIdx.x & 63) < len && (mask == nullptr || byte != 0));
    }
    // tile t of K and of V (any t: past the end they are empty)
    __device__ __forceinline__ XTile k_tile(int t) const { return XTile(kp + (int64_t)t * kXTile * kst, kst, len - t * kXTile, copies.D); }
    __device__ __forceinline__ XTile v_tile(int t) const { return XTile(vp + (int64_t)t * kXTile * vst, vst, len - t * kXTile, copies.D); }
    // the bias of a tile's scores
    static __device__ __forceinline__ void bias_of(uint64_t alive, float* bias) {
        if (alive != ~(uint64_t)0 && threadIdx.x < kXTile) bias[threadIdx.x] = (alive >> threadIdx.x) & 1 ? 0.f : -__builtin_inff();
    }
    // the first tile, whole and in place after the barrier
    __device__ __forceinline__ void first(int t, uint16_t* kt, uint16_t* vt, float* bias) {
        if (mask != nullptr) ask(t);  // (without a mask nothing is waited for)
        live[0] = counted(t);
        copies.group(0, 1, k_tile(t), v_tile(t), ~live[0], kt, vt);
        bias_of(live[0], bias);
        ask(t + 1);
        wait_loads();
        live[1] = counted(t + 1);
    }
    // before the barrier at the end of tile t
    __device__ __forceinline__ void end(int t) {
        wait_loads();
        live[0] = live[1];
        live[1] = counted(t + 2);
    }
};
// the start of a tile's scores: the bias of rows 32 u .. 32 u + 31
__device__ __forceinline__ v16f bias16(const float* bias, int u, int half) {
    v16f s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const v4f w = *reinterpret_cast<const v4f*>(bias + u * 32 + i * 8 + half * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i * 4 + j] = w[j];
    }
    return s;
}

// Which block (128 rows or keys of a unit) a workgroup works on, and which part of its walk. The blocks that fill the card
// whole times (`full`, a multiple of the workgroups that run at once) are walked by one workgroup each; those left (`tail`),
// which would leave most of it idle for another whole turn, are divided over `splits` workgroups each. Workgroups go to the 8
// XCDs in turn: consecutive blocks are given to the same XCD, whose L2 then holds the K and V (or Q and dO) that they share.
struct XSchedule {
    unsigned full, tail;
    int splits;
    __device__ __forceinline__ bool item(unsigned& block, int& split, int& of) const {
        const unsigned id = blockIdx.x;
        of = 1;
        split = 0;
        if (id < full) {
            block = (id & 7u) * (full >> 3) + (id >> 3);
            return true;
        }
        const unsigned j = id - full, n = tail * splits, per = (n + 7) / 8, k = (j & 7u) * per + (j >> 3);
        if ((j >> 3) >= per || k >= n) return false;
        split = (int)(k / tail);
        block = full + k - split * tail;
        of = splits;
        return true;
    }
    unsigned grid() const { return full + 8u * ((tail * splits + 7) / 8); }
    int64_t parts() const { return splits > 1 ? (int64_t)tail * splits : 0; }  // blocks of partial results
};
// `slots`: workgroups that run at once on the 256 CUs; `length`: of a walk; `floats`: of a block's partial result. The blocks left
// are divided (into parts of four tiles or more) with the number that ends first by this estimate, in tiles: a workgroup takes one
// tile's time longer than its walk; a CU with one workgroup on it works a tile off faster than one with all its slots taken (half
// the slots: 0.6 of the time); parts are written, read and joined: 6 tiles' time for 128 x 128 floats of every slot, and 2 for the
// launch. Forward, bf16, us with the join: 3 x 16 heads of 128, 700 x 700 (288 blocks) 32 whole, 47 in two parts, 52 in three; 8 x 16
// heads of 64, 512 x 2048 (512 blocks) 55 whole, 68 in two; 8 single tokens, 32 heads of 128 on 8, 8192 keys (64 blocks) 59 in 8 parts, 64
// in 4, 63 in 16, 72 in 32.
inline XSchedule schedule(int64_t blocks, int64_t length, int slots, double floats) {
    XSchedule s;
    s.full = (unsigned)(blocks / slots * slots);
    s.tail = (unsigned)(blocks - s.full);
    s.splits = 1;
    const int64_t tiles = (length + kXTile - 1) / kXTile, most = (tiles + 3) / 4;
    double cost = 1e300;
    for (int cus = 0; s.tail && cus <= 2 * slots; cus += 256) {  // whole, or the most parts that so many places take
        int64_t n = cus / s.tail;
        n = n < most ? n : most;
        n = n < 1 ? 1 : n;
        const double groups = (double)s.tail * n, load = (groups > 256 ? groups : 256) / slots;
        const double turns = load <= 1 ? 0.25 + 0.75 * load : (double)(int64_t)((groups + slots - 1) / slots);
        const double c = turns * ((double)((tiles + n - 1) / n) + 1) + (n > 1 ? 6 * groups / slots * floats / (kXRows * 128) + 2 : 0);
        if (c < cost) { cost = c; s.splits = (int)n; }
    }
    return s;
}
// Into how many parts each of `units` walks of `steps` goes, `least` steps each or more, when `slots` workgroups run at once: the
// number with which the last one ends first, a workgroup costing about two steps beside its walk. (44 walks of 360 tiles on 512
// slots, backward with 16 keys of 128: 11 parts 372 us; 12, whose last 16 workgroups wait for a free place, 548.)
inline int walk_parts(int64_t units, int64_t steps, int slots, int least) {
    const int64_t most = steps > least ? (steps + least - 1) / least : 1;
    int64_t best = 1, cost = INT64_MAX;
    for (int turns = 1; turns <= 8; ++turns) {  // the most parts that take so many turns of the card, or one
        int64_t n = (int64_t)slots * turns / units;
        n = n < 1 ? 1 : n < most ? n : most;
        const int64_t c = (units * n + slots - 1) / slots * ((steps + n - 1) / n + 2);
        if (c < cost) { best = n; cost = c; }
    }
    return (int)best;
}

// One 32 x D result of a wave (columns = rows of the output, results = its elements) to memory. Lanes l and l + 32 hold 4
// elements each of the same 8: two half exchanges make 16 consecutive bytes of either, 8 elements of group i in the low lane
// and those of group i + 1 in the high one. p: the lane's output row (of column l % 32), NULL where there is none.
template <int DT, int DP>
__device__ __forceinline__ void store_rows(const v16f (&acc)[DP / 32], float scale, uint16_t* p, int D, int lane) {
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            uint32_t w[2][2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int r = 4 * (i + k);
                w[k][0] = pack2<DT>(acc[t][r] * scale, acc[t][r + 1] * scale);
                w[k][1] = pack2<DT>(acc[t][r + 2] * scale, acc[t][r + 3] * scale);
            }
            const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
            const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
            const int e = t * 32 + (i + (lane >> 5)) * 8;
            if (p != nullptr && e < D) *reinterpret_cast<v4u*>(p + e) = v4u{x[0], y[0], x[1], y[1]};
        }
}

// What that left off: 16 bytes of a lane, elements 0 .. 15 of 32 in the low lane, 16 .. 31 in the high one
template <int DT, int DP>
__device__ __forceinline__ void store_rests(const v16f (&acc)[DP / 32], float scale, uint8_t* p, int D, int lane) {
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x0 = acc[t][4 * i] * scale, x1 = acc[t][4 * i + 1] * scale, x2 = acc[t][4 * i + 2] * scale, x3 = acc[t][4 * i + 3] * scale;
            w[i] = rests_of<DT>(x0, x1, x2, x3, pack2<DT>(x0, x1), pack2<DT>(x2, x3));
        }
        // lanes l and l + 32: elements 8 i .. + 3 and 8 i + 4 .. + 7; first exchanged into 8 and 8, then into 16 and 16
        const auto a = __builtin_amdgcn_permlane32_swap(w[0], w[1], false, false), b = __builtin_amdgcn_permlane32_swap(w[2], w[3], false, false);
        const auto x = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false), y = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
        typedef int v4i8 __attribute__((ext_vector_type(4), aligned(8)));
        const int e = t * 32 + (lane >> 5) * 16;
        if (p != nullptr) {  // (D is a multiple of 8)
            if (e + 8 < D) *reinterpret_cast<v4i8*>(p + e) = v4i8{(int)x[0], (int)y[0], (int)x[1], (int)y[1]};
            else if (e < D) *reinterpret_cast<v2i*>(p + e) = v2i{(int)x[0], (int)y[0]};
        }
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
    if (t > 1 && s[2] >= (1 << 24)) return fail(Q8_ERR_SHAPE, "%s: token stride of %s (below 2^24 elements)", who, name);
    if (e > (INT64_MAX >> 4)) return fail(Q8_ERR_SHAPE, "%s: strides of %s", who, name);
    if (!aligned16(p)) return fail(Q8_ERR_ALIGN, "%s: %s must be 16-byte aligned", who, name);
    return Q8_OK;
}

inline int x_sizes(const char* who, int dt, int64_t B, int H, int Hkv, int M, int N, int D, float scale) {
    if (dt != Q8_BF16 && dt != Q8_F16) return fail(Q8_ERR_DTYPE, "%s: element type %d (bf16 or fp16)", who, dt);
    if (B < 0 || H < 1 || Hkv < 1 || M < 0 || N < 0) return fail(Q8_ERR_SHAPE, "%s: B %lld, heads %d and %d, M %d, N %d", who, (long long)B, H, Hkv, M, N);
    if (H % Hkv) return fail(Q8_ERR_SHAPE, "%s: %d query heads on %d key heads (a multiple is needed)", who, H, Hkv);
    if (D < 8 || D > 128 || D % 8) return fail(Q8_ERR_SHAPE, "%s: head dim %d (a multiple of 8 up to 128)", who, D);
    if (!(scale > 0.f) || scale > 1e38f) return fail(Q8_ERR_SHAPE, "%s: softmax scale %g (positive and finite)", who, (double)scale);
    // rows, units and the fp32 scratch stay in 32-bit counts
    if ((int64_t)(H / Hkv) * M > 0x3fffffff || N > 0x3fffffff || (B && (int64_t)Hkv > 0x3fffffff / B) ||
        (B && M && (int64_t)H > ((int64_t)1 << 40) / B / M))
        return fail(Q8_ERR_SHAPE, "%s: sizes out of range", who);
    return Q8_OK;
}

// The forward (cross_attn.hip) with every output optional but o or o_low; what the backward runs where it was not given o_low.
struct XForward {
    const void* q; const int64_t* q_strides;
    const void* k; const int64_t* k_strides;
    const void* v; const int64_t* v_strides;
    void* o; const int64_t* o_strides;
    void* o_low;
    float* lse;
    const int32_t* kv_lens; const uint8_t* key_mask; int64_t mask_row_stride;
    int dt; float softmax_scale;
    int64_t B; int H, Hkv, M, N, D;
    void* workspace; int64_t workspace_bytes;
    hipStream_t stream;
};
int cross_attn_forward(const char* who, const XForward& c);
int64_t cross_attn_forward_workspace(int64_t B, int H, int Hkv, int M, int N, int D);  // bytes, of sizes that x_sizes takes

inline int padded_head(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

}  // namespace q8
