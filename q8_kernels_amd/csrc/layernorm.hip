// Layer norm over the last dimension, forward and backward with the parameters' gradients.
//
//   mu = mean_j x_j, rstd = 1 / sqrt(mean_j (x_j - mu)^2 + eps), h_j = (x_j - mu) rstd, y_j = h_j w_j + b_j
//   with u_j = g_j w_j:  dx_j = rstd (u_j - mean(u) - h_j mean(u h)),  dw_j = sum_rows g_j h_j,  db_j = sum_rows g_j
//
// HBM-bound: the forward reads x and writes y, the backward reads x and g and writes dx, all of them once. A row therefore
// stays in the registers of the T threads that own it (16 to 1024, at most 32 elements each) between the
// passes over it: the variance is the mean of the squared distances from the finished mean, not E x^2 - mu^2, which
// cancels. All sums are fp32. Rows whose length or address does not allow 16-byte accesses take element accesses instead
// (VEC = 1), strided by T so that a wave still covers consecutive addresses.
//
// The parameters' gradients are sums over rows. A workgroup of the backward walks over rows and keeps the sums of its
// columns in registers, adds the groups of threads that hold the same columns in LDS, one after the other, and writes one
// row of partial sums to the workspace; a second kernel adds those in a fixed order. No atomics: the same inputs give the
// same bits. The number of workgroups (ln_blocks) trades rows in flight against the partial sums' traffic. Rows of more than
// 16384 elements (8192 where accesses are by element) leave no registers for the sums: a kernel of its own reads x and g once
// more for them (1000 x 30000 bf16: 37 and 30 us; in one kernel, an earlier build whose registers spilled, 172).
//
// bf16, 12288 x 2048, inputs that no cache holds: forward 22 to 23 us (4.4 TB/s), backward 33 and 4 to 5 for the parameters' sums
// (4.0 TB/s of what it has to move; a copy reaches 5.1). What bounds it: HBM, and at the smallest sizes the launches.
#include "q8_common.h"
#include "q8_host.h"

namespace q8 {

constexpr int kLnMaxDim = 32768;

__device__ __forceinline__ uint16_t f32_to_f16_bits(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }

// The elements of a row that one thread holds, as they are in memory: 8 * CH of them, element i of thread t is
// ((i / 8) * T + t) * 8 + i % 8 (VEC = 8) or i * T + t (VEC = 1).
template <int DT, int VEC, int T, int CH>
struct RowPart {
    static constexpr int N = 8 * CH;
    static constexpr int WORDS = VEC == 1 ? N : (DT == Q8_F32 ? N : N / 2);
    uint32_t r[WORDS];

    static __device__ __forceinline__ int index(int i, int t) { return VEC == 1 ? i * T + t : ((i >> 3) * T + t) * 8 + (i & 7); }

    // elements past the row's end are zeros; row_ok false: all of them are
    __device__ __forceinline__ void load(const void* p, int64_t first, int t, int dim, bool row_ok) {
        if constexpr (VEC == 8) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int e = (c * T + t) * 8;
                constexpr int Q = DT == Q8_F32 ? 2 : 1;  // 16-byte accesses of 8 elements
                v4u w[Q];
#pragma unroll
                for (int q = 0; q < Q; ++q) w[q] = v4u{0u, 0u, 0u, 0u};
                if (row_ok && e < dim) {
                    const v4u* s = reinterpret_cast<const v4u*>(static_cast<const char*>(p) + (first + e) * (DT == Q8_F32 ? 4 : 2));
#pragma unroll
                    for (int q = 0; q < Q; ++q) w[q] = s[q];
                }
#pragma unroll
                for (int q = 0; q < Q; ++q)
#pragma unroll
                    for (int k = 0; k < 4; ++k) r[(c * Q + q) * 4 + k] = w[q][k];
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = i * T + t;
                r[i] = 0u;
                if (row_ok && e < dim) {
                    if constexpr (DT == Q8_F32) r[i] = static_cast<const uint32_t*>(p)[first + e];
                    else r[i] = static_cast<const uint16_t*>(p)[first + e];
                }
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (DT == Q8_F32) return __uint_as_float(r[i]);
        const uint32_t h = VEC == 1 ? r[i] : ((i & 1) ? r[i >> 1] >> 16 : r[i >> 1] & 0xffffu);
        return DT == Q8_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
    }
    static __device__ __forceinline__ void store(void* p, int64_t first, int t, int dim, const float (&v)[N]) {
        if constexpr (VEC == 8) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int e = (c * T + t) * 8;
                if (e >= dim) continue;
                v4u* s = reinterpret_cast<v4u*>(static_cast<char*>(p) + (first + e) * (DT == Q8_F32 ? 4 : 2));
                if constexpr (DT == Q8_F32) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        v4u w;
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] = __float_as_uint(v[c * 8 + q * 4 + k]);
                        s[q] = w;
                    }
                } else {
                    v4u w;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        w[k] = DT == Q8_BF16 ? pack2_bf16(v[c * 8 + 2 * k], v[c * 8 + 2 * k + 1])
                                             : f32_to_f16_bits(v[c * 8 + 2 * k]) | ((uint32_t)f32_to_f16_bits(v[c * 8 + 2 * k + 1]) << 16);
                    *s = w;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = i * T + t;
                if (e >= dim) continue;
                if constexpr (DT == Q8_F32) static_cast<float*>(p)[first + e] = v[i];
                else static_cast<uint16_t*>(p)[first + e] = DT == Q8_BF16 ? (uint16_t)(pack2_bf16(v[i], 0.f) & 0xffffu) : f32_to_f16_bits(v[i]);
            }
        }
    }
};

// The thread's elements of a parameter vector in fp32; absent (NULL): all `none`. Parameters are fp32 or of x's type.
template <int DT, int VEC, int T, int CH>
__device__ __forceinline__ void load_param(const void* p, bool f32, int t, int dim, float none, float (&v)[8 * CH]) {
    if (p == nullptr) {
#pragma unroll
        for (int i = 0; i < 8 * CH; ++i) v[i] = none;
    } else if (f32) {
        RowPart<Q8_F32, VEC, T, CH> w;
        w.load(p, 0, t, dim, true);
#pragma unroll
        for (int i = 0; i < 8 * CH; ++i) v[i] = w.get(i);
    } else {
        RowPart<DT, VEC, T, CH> w;
        w.load(p, 0, t, dim, true);
#pragma unroll
        for (int i = 0; i < 8 * CH; ++i) v[i] = w.get(i);
    }
}

// Sums of NV values over the T threads of a row. T > 64: one barrier; `slot` alternates between calls so that a wave that
// runs ahead does not overwrite what a slower one still reads (two slots do: it cannot pass the next call's barrier).
template <int T, int NV>
__device__ __forceinline__ void row_sums(float (&v)[NV], float (*red)[NV][16], int slot) {
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] = group_sum<(T < 64 ? T : 64)>(v[k]);
    if constexpr (T > 64) {
        constexpr int W = T / 64;
        const int wave = threadIdx.x >> 6, first = threadIdx.x / T * W;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < NV; ++k) red[slot][k][wave] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float s = red[slot][k][first];
#pragma unroll
            for (int i = 1; i < W; ++i) s += red[slot][k][first + i];
            v[k] = s;
        }
    }
}

// Whether the backward's threads have registers for the parameters' gradients beside the row (128 each with 1024 threads).
template <int VEC, int T, int CH>
constexpr bool ln_fused() { return T < 1024 || CH == 1 || (CH == 2 && VEC == 8); }

template <int T>
constexpr int ln_threads() { return T < 256 ? 256 : T; }

template <int DT, int VEC, int T, int CH>
__global__ __launch_bounds__(ln_threads<T>()) void layernorm_kernel(const void* __restrict__ x, int64_t x_stride, const void* __restrict__ w,
                                                                  const void* __restrict__ b, int w_f32, void* __restrict__ y,
                                                                  float* __restrict__ mean, float* __restrict__ rstd, int64_t rows, int dim, float eps) {
    constexpr int N = 8 * CH, G = ln_threads<T>() / T;
    __shared__ float red[2][1][16];
    const int t = threadIdx.x % T;
    const int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / T;
    const bool row_ok = row < rows;
    RowPart<DT, VEC, T, CH> xr;
    xr.load(x, row * x_stride, t, dim, row_ok);
    float v[N], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = xr.get(i);
        s[0] += v[i];
    }
    row_sums<T, 1>(s, red, 0);
    const float mu = s[0] / (float)dim;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] -= mu;
        if (RowPart<DT, VEC, T, CH>::index(i, t) < dim) s[0] += v[i] * v[i];
    }
    row_sums<T, 1>(s, red, 1);
    const float rs = 1.0f / sqrtf(s[0] / (float)dim + eps);
    if (!row_ok) return;
    float wv[N], bv[N];
    load_param<DT, VEC, T, CH>(w, w_f32, t, dim, 1.0f, wv);
    load_param<DT, VEC, T, CH>(b, w_f32, t, dim, 0.0f, bv);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] * rs * wv[i] + bv[i];
    RowPart<DT, VEC, T, CH>::store(y, row * dim, t, dim, v);
    if (t == 0 && mean != nullptr) {
        mean[row] = mu;
        rstd[row] = rs;
    }
}

// partials: [gridDim.x][2][dim] fp32 (sums of g h, sums of g), or NULL when no parameter needs a gradient.
// dx NULL: not wanted. The next row is requested before the present one's sums are formed, where the registers
// hold both (1000 x 16384 fp32, 1024 threads with 16 elements: 62 us without, 85 with).
template <int DT, int VEC, int T, int CH>
__global__ __launch_bounds__(ln_threads<T>()) void layernorm_backward_kernel(const void* __restrict__ g, int64_t g_stride, const void* __restrict__ x,
                                                                           int64_t x_stride, const void* __restrict__ w, int w_f32,
                                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                           void* __restrict__ dx, float* __restrict__ partials, int64_t rows, int dim) {
    constexpr int N = 8 * CH, G = ln_threads<T>() / T;
    constexpr bool FUSED = ln_fused<VEC, T, CH>(), AHEAD = T < 1024 || CH == 1;
    using Part = RowPart<DT, VEC, T, CH>;
    __shared__ float red[2][2][16];
    __shared__ float cols[G > 1 ? 2 * T * N : 1];
    const int t = threadIdx.x % T, grp = threadIdx.x / T;
    const float inv_dim = 1.0f / (float)dim;
    float wv[N], dw[N], db[N];
    load_param<DT, VEC, T, CH>(w, w_f32, t, dim, 1.0f, wv);
#pragma unroll
    for (int i = 0; i < N; ++i) { dw[i] = 0.f; db[i] = 0.f; }
    const int64_t step = (int64_t)gridDim.x * G;
    int64_t row = (int64_t)blockIdx.x * G + grp;
    const int64_t turns = (rows + step - 1) / step;  // the same for all threads: every wave meets every barrier
    Part xr, gr;
    float mu = 0.f, rs = 0.f;
    if constexpr (AHEAD) {
        xr.load(x, row * x_stride, t, dim, row < rows);
        gr.load(g, row * g_stride, t, dim, row < rows);
        if (row < rows) { mu = mean[row]; rs = rstd[row]; }
    }
    for (int64_t it = 0; it < turns; ++it, row += step) {
        const bool row_ok = row < rows;
        Part xn, gn;
        float mn = 0.f, rn = 0.f;
        if constexpr (AHEAD) {
            const int64_t next = row + step;
            xn.load(x, next * x_stride, t, dim, next < rows);
            gn.load(g, next * g_stride, t, dim, next < rows);
            if (next < rows) { mn = mean[next]; rn = rstd[next]; }
        } else {
            xr.load(x, row * x_stride, t, dim, row_ok);
            gr.load(g, row * g_stride, t, dim, row_ok);
            if (row_ok) { mu = mean[row]; rs = rstd[row]; }
        }
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            // (past the row's end g is zero, so u and every sum is too, whatever h is: h is finite there)
            const float gv = gr.get(i), h = (xr.get(i) - mu) * rs, u = gv * wv[i];
            s[0] += u;
            s[1] += u * h;
            if constexpr (FUSED) {
                dw[i] += gv * h;
                db[i] += gv;
            }
        }
        row_sums<T, 2>(s, red, (int)(it & 1));
        if (row_ok && dx != nullptr) {
            const float mu_u = s[0] * inv_dim, mu_uh = s[1] * inv_dim;
            float o[N];
    #pragma unroll
            for (int i = 0; i < N; ++i) {
                const float h = (xr.get(i) - mu) * rs;
                o[i] = rs * (gr.get(i) * wv[i] - mu_u - h * mu_uh);
            }
            Part::store(dx, row * dim, t, dim, o);
        }
        if constexpr (AHEAD) { xr = xn; gr = gn; mu = mn; rs = rn; }
    }
    if (!FUSED || partials == nullptr) return;
    if constexpr (G > 1) {
        for (int k = 0; k < G; ++k) {
            if (grp == k) {
#pragma unroll
                for (int i = 0; i < N; ++i) {  // a column belongs to the thread t of every group: no other thread touches its slot
                    const int s = i * T + t;
                    cols[s] = k == 0 ? dw[i] : cols[s] + dw[i];
                    cols[T * N + s] = k == 0 ? db[i] : cols[T * N + s] + db[i];
                }
            }
            __syncthreads();
        }
        if (grp != 0) return;
#pragma unroll
        for (int i = 0; i < N; ++i) { dw[i] = cols[i * T + t]; db[i] = cols[T * N + i * T + t]; }
    }
    float* out = partials + (int64_t)blockIdx.x * 2 * dim;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = Part::index(i, t);
        if (e < dim) { out[e] = dw[i]; out[dim + e] = db[i]; }
    }
}

// VEC consecutive elements in fp32
template <int DT, int VEC>
__device__ __forceinline__ void load_columns(const void* p, int64_t at, float (&v)[VEC == 8 ? 8 : 1]) {
    if constexpr (VEC == 1) {
        if constexpr (DT == Q8_F32) v[0] = static_cast<const float*>(p)[at];
        else v[0] = DT == Q8_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(p)[at]) : f16_bits_to_f32(static_cast<const uint16_t*>(p)[at]);
    } else if constexpr (DT == Q8_F32) {
        const v4f a = *reinterpret_cast<const v4f*>(static_cast<const float*>(p) + at), b = *reinterpret_cast<const v4f*>(static_cast<const float*>(p) + at + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[i + 4] = b[i]; }
    } else {
        const v4u a = *reinterpret_cast<const v4u*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = DT == Q8_BF16 ? bf16_bits_to_f32(a[i] & 0xffffu) : f16_bits_to_f32(a[i] & 0xffffu);
            v[2 * i + 1] = DT == Q8_BF16 ? bf16_bits_to_f32(a[i] >> 16) : f16_bits_to_f32(a[i] >> 16);
        }
    }
}

// The partial sums of a part of the rows alone, for rows too long for the kernel above: a thread holds VEC columns.
template <int DT, int VEC>
__global__ __launch_bounds__(256) void layernorm_columns_kernel(const void* __restrict__ g, int64_t g_stride, const void* __restrict__ x, int64_t x_stride,
                                                                const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                float* __restrict__ partials, int64_t rows, int dim) {
    constexpr int BATCH = 4, N = VEC == 8 ? 8 : 1;
    const int col = (blockIdx.x * 256 + threadIdx.x) * VEC;
    if (col >= dim) return;
    const int64_t per = (rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    float dw[N], db[N];
#pragma unroll
    for (int i = 0; i < N; ++i) { dw[i] = 0.f; db[i] = 0.f; }
    for (int64_t r = r0; r < r1; r += BATCH) {
        float xv[BATCH][N], gv[BATCH][N], mu[BATCH], rs[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const bool ok = r + k < r1;
            const int64_t row = ok ? r + k : r;
            load_columns<DT, VEC>(x, row * x_stride + col, xv[k]);
            load_columns<DT, VEC>(g, row * g_stride + col, gv[k]);
            mu[k] = mean[row];
            rs[k] = ok ? rstd[row] : 0.f;
            if (!ok) {
#pragma unroll
                for (int i = 0; i < N; ++i) xv[k][i] = gv[k][i] = mu[k] = 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                dw[i] += gv[k][i] * ((xv[k][i] - mu[k]) * rs[k]);
                db[i] += gv[k][i];
            }
    }
    float* out = partials + (int64_t)blockIdx.y * 2 * dim + col;
#pragma unroll
    for (int i = 0; i < N; ++i) { out[i] = dw[i]; out[dim + i] = db[i]; }
}

__device__ __forceinline__ void store_any(void* p, int dt, int64_t e, float v) {
    if (dt == Q8_F32) static_cast<float*>(p)[e] = v;
    else static_cast<uint16_t*>(p)[e] = dt == Q8_BF16 ? (uint16_t)(pack2_bf16(v, 0.f) & 0xffffu) : f32_to_f16_bits(v);
}

// out[column] = sum of the partial rows: 32 columns x 32 groups of rows per workgroup, then the groups in order.
__global__ __launch_bounds__(1024) void layernorm_params_kernel(const float* __restrict__ partials, int blocks, void* __restrict__ dw,
                                                                void* __restrict__ db, int dt, int dim) {
    __shared__ float part[32][33];
    const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + c;  // 0 .. 2 dim - 1: dw's columns, then db's
    float s = 0.f;
    if (col < 2 * dim) {
        const float* p = partials + (int64_t)k * 2 * dim + col;
        int r = k;
        for (; r + 7 * 32 < blocks; r += 8 * 32, p += (int64_t)8 * 32 * 2 * dim) {  // 8 loads under way at once
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = p[(int64_t)i * 32 * 2 * dim];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += v[i];
        }
        for (; r < blocks; r += 32, p += (int64_t)32 * 2 * dim) s += *p;
    }
    part[k][c] = s;
    __syncthreads();
    if (k != 0 || col >= 2 * dim) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += part[i][c];
    void* out = col < dim ? dw : db;
    if (out != nullptr) store_any(out, dt, col < dim ? col : col - dim, s);
}

// The threads of a row, as LN_BY_DIM below chooses them with the chunks of 8 elements that each holds. The forward takes few
// threads with up to 32 elements; the backward holds six times as many registers an element, so it takes more threads with 8
// or 16, which leaves two waves or more on a SIMD. Kernel times in us, forward / backward and the parameters' sums, of threads that
// each hold the fewest chunks that cover the row; bf16 unless fp32 is said, inputs that no cache holds:
//   12288 x 2048: 64 threads 23.5 / 35.6, 128 22.1 / 37.2, 256 23.7 / 43.6     4099 x 1155 fp32: 64 15.2 / 37.4, 128 11.8 / 21.8
//   8192 x 4096:  256 30.1 / 48.8, 512 31.8 / 48.3                             4000 x 3001: 256 28.6 / 30.7, 512 28.3 / 27.6
//   4096 x 8192:  256 30.8 / 70.3 (256 workgroups: 60.7), 1024 35.2 / 55.4     2000 x 5001: 256 35.5 / 52.4, 512 36.7 / 34.9, 1024 26.1 / 27.0
//   65536 x 128:  16 8.9 / 21.2, 64 21.4 / 38.3
static int ln_fwd_threads(int dim) { return dim <= 128 ? 16 : dim <= 1024 ? 64 : dim <= 2048 ? 128 : dim <= 8192 ? 256 : 1024; }
static int ln_threads_of(int dim, bool vec) { return dim <= 128 ? 16 : dim <= 1024 ? 64 : dim <= 2048 ? 128 : dim <= 4096 ? 512 : dim <= 8192 && !vec ? 512 : 1024; }

// Workgroups of the backward: two rows or more for each group of threads (300 x 2048: 10.3 us, with four 14.2), and few enough
// that the partial sums stay small beside the rows: 512 (12288 x 2048: 256 49.5 us, 512 37.5, 1024 44.0), 256 of 1024 threads
// (4096 x 8192 with 256 threads: 512 70 us, 256 61), 128 of the longest rows (2000 x 16384: 68 us).
static int64_t ln_blocks(int64_t rows, int dim, bool vec) {
    const int t = ln_threads_of(dim, vec), groups = (t < 256 ? 256 : t) / t;
    const int64_t most = t < 1024 ? 512 : dim <= 8192 ? 256 : 128, b = (rows + 2 * groups - 1) / (2 * groups);
    return b < 1 ? 1 : b < most ? b : most;
}
// Parts of the rows for the kernel that forms the partial sums alone: 32 rows or more, at most 128.
static int64_t ln_parts(int64_t rows) { return rows <= 32 ? 1 : rows < 4096 ? (rows + 31) / 32 : 128; }
// workspace for either kind of access: the call may be of an unaligned tensor (which needs no more for long rows)
static int64_t ln_partials(int64_t rows, int dim) {
    const int64_t a = ln_blocks(rows, dim, true), b = ln_blocks(rows, dim, false);
    return (a > b ? a : b) * 2 * dim * (int64_t)sizeof(float);
}

static int ln_check(const char* who, int dt, int w_dtype, bool has_param, int64_t rows, int dim) {
    if (rows < 0 || dim < 1 || dim > kLnMaxDim) return fail(Q8_ERR_SHAPE, "%s: rows %lld, dim %d (1 .. %d)", who, (long long)rows, dim, kLnMaxDim);
    if (rows > (int64_t)0x7fffffff) return fail(Q8_ERR_SHAPE, "%s: too many rows (%lld)", who, (long long)rows);
    if (dt != Q8_BF16 && dt != Q8_F16 && dt != Q8_F32) return fail(Q8_ERR_DTYPE, "%s: element type %d (bf16, fp16 or fp32)", who, dt);
    if (has_param && w_dtype != Q8_F32 && w_dtype != dt) return fail(Q8_ERR_DTYPE, "%s: parameters are fp32 or of x's type, got %d", who, w_dtype);
    return Q8_OK;
}

// a row stride: at least dim (one row: anything), and such that the last element's byte offset fits 63 bits
static bool ln_stride_ok(int64_t stride, int64_t rows, int dim) {
    return rows <= 1 || (stride >= dim && stride <= INT64_MAX / 8 / rows);
}

static bool elem_aligned(const void* p, int dt) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(elem_size(dt) - 1)) == 0; }

}  // namespace q8

using namespace q8;

#define LN_BY_DIM(DT, VEC, FWD, ...)                                                                        \
    do {                                                                                                    \
        if (dim <= 128) { constexpr int T = 16, CH = 1; __VA_ARGS__(DT, VEC); }                             \
        else if (dim <= 512) { constexpr int T = 64, CH = 1; __VA_ARGS__(DT, VEC); }                        \
        else if (dim <= 1024) { constexpr int T = 64, CH = 2; __VA_ARGS__(DT, VEC); }                       \
        else if (dim <= 2048) { constexpr int T = 128, CH = 2; __VA_ARGS__(DT, VEC); }                      \
        else if (dim <= 4096) { constexpr int T = FWD ? 256 : 512, CH = 512 / T; __VA_ARGS__(DT, VEC); }    \
        else if (dim <= 8192) { constexpr int T = FWD ? 256 : VEC == 8 ? 1024 : 512, CH = 1024 / T; __VA_ARGS__(DT, VEC); } \
        else if (dim <= 16384) { constexpr int T = 1024, CH = 2; __VA_ARGS__(DT, VEC); }                    \
        else { constexpr int T = 1024, CH = 4; __VA_ARGS__(DT, VEC); }                                      \
    } while (0)
#define LN_BY_TYPE(vec, FWD, ...)                                    \
    do {                                                             \
        if (vec) {                                                   \
            if (dt == Q8_BF16) LN_BY_DIM(Q8_BF16, 8, FWD, __VA_ARGS__);      \
            else if (dt == Q8_F16) LN_BY_DIM(Q8_F16, 8, FWD, __VA_ARGS__);   \
            else LN_BY_DIM(Q8_F32, 8, FWD, __VA_ARGS__);             \
        } else {                                                     \
            if (dt == Q8_BF16) LN_BY_DIM(Q8_BF16, 1, FWD, __VA_ARGS__);      \
            else if (dt == Q8_F16) LN_BY_DIM(Q8_F16, 1, FWD, __VA_ARGS__);   \
            else LN_BY_DIM(Q8_F32, 1, FWD, __VA_ARGS__);             \
        }                                                            \
    } while (0)

extern "C" int q8_layernorm(const void* x, int dt, int64_t x_row_stride, const void* w, const void* b, int w_dtype, void* y, float* mean,
                            float* rstd, int64_t rows, int dim, float eps, q8_stream_t stream) {
    if (int e = ln_check("q8_layernorm", dt, w_dtype, w || b, rows, dim)) return e;
    if (rows == 0) return Q8_OK;
    if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return fail(Q8_ERR_NULL, "q8_layernorm: null pointer (mean and rstd: both or neither)");
    if (!ln_stride_ok(x_row_stride, rows, dim)) return fail(Q8_ERR_SHAPE, "q8_layernorm: row stride %lld", (long long)x_row_stride);
    const int wd = w_dtype == Q8_F32 ? Q8_F32 : dt;
    if (!elem_aligned(x, dt) || !elem_aligned(y, dt) || (w && !elem_aligned(w, wd)) || (b && !elem_aligned(b, wd)) || !elem_aligned(mean, Q8_F32) ||
        !elem_aligned(rstd, Q8_F32))
        return fail(Q8_ERR_ALIGN, "q8_layernorm: pointer not aligned to its element type");
    if (!(eps >= 0.f)) return fail(Q8_ERR_SHAPE, "q8_layernorm: eps %g", (double)eps);
    const bool vec = dim % 8 == 0 && (rows == 1 || x_row_stride % 8 == 0) && aligned16(x) && aligned16(y) && aligned16(w) && aligned16(b);
    const int t = ln_fwd_threads(dim), groups = (t < 256 ? 256 : t) / t;
    const int64_t blocks = (rows + groups - 1) / groups;
    if (blocks > most_blocks(t < 256 ? 256 : t)) return fail(Q8_ERR_SHAPE, "q8_layernorm: too many rows (%lld of %d elements)", (long long)rows, dim);
    const dim3 grid((unsigned)blocks);
    hipStream_t s = static_cast<hipStream_t>(stream);
#define LN_FWD(DT, VEC) \
    layernorm_kernel<DT, VEC, T, CH><<<grid, ln_threads<T>(), 0, s>>>(x, x_row_stride, w, b, w_dtype == Q8_F32, y, mean, rstd, rows, dim, eps)
    LN_BY_TYPE(vec, true, LN_FWD);
#undef LN_FWD
    return launch_status("q8_layernorm");
}

extern "C" int64_t q8_layernorm_backward_workspace(int64_t rows, int dim) {
    if (rows < 0 || rows > (int64_t)0x7fffffff || dim < 1 || dim > kLnMaxDim) return fail(Q8_ERR_SHAPE, "q8_layernorm_backward_workspace: rows %lld, dim %d", (long long)rows, dim);
    return ln_partials(rows, dim);
}

extern "C" int q8_layernorm_backward(const void* grad, int64_t grad_row_stride, const void* x, int dt, int64_t x_row_stride, const void* w, int w_dtype,
                                     const float* mean, const float* rstd, void* dx, void* dw, void* db, void* workspace, int64_t workspace_bytes,
                                     int64_t rows, int dim, q8_stream_t stream) {
    const bool params = dw || db;
    if (int e = ln_check("q8_layernorm_backward", dt, w_dtype, w || params, rows, dim)) return e;
    if (!dx && !params) return Q8_OK;
    if (rows == 0 && !params) return Q8_OK;
    if ((rows && (!grad || !x || !mean || !rstd)) || (params && !workspace)) return fail(Q8_ERR_NULL, "q8_layernorm_backward: null pointer");
    if (!ln_stride_ok(x_row_stride, rows, dim) || !ln_stride_ok(grad_row_stride, rows, dim)) return fail(Q8_ERR_SHAPE, "q8_layernorm_backward: row stride");
    const int wd = w_dtype == Q8_F32 ? Q8_F32 : dt;
    if (!elem_aligned(grad, dt) || !elem_aligned(x, dt) || !elem_aligned(dx, dt) || (w && !elem_aligned(w, wd)) || (dw && !elem_aligned(dw, wd)) ||
        (db && !elem_aligned(db, wd)) || !elem_aligned(mean, Q8_F32) || !elem_aligned(rstd, Q8_F32) || (params && !elem_aligned(workspace, Q8_F32)))
        return fail(Q8_ERR_ALIGN, "q8_layernorm_backward: pointer not aligned to its element type");
    if (params && workspace_bytes < ln_partials(rows, dim))
        return fail(Q8_ERR_SHAPE, "q8_layernorm_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                    (long long)ln_partials(rows, dim));
    const bool vec = dim % 8 == 0 && (rows <= 1 || (x_row_stride % 8 == 0 && grad_row_stride % 8 == 0)) && aligned16(x) && aligned16(grad) &&
                     aligned16(dx) && aligned16(w);
    const bool fused = dim <= (vec ? 16384 : 8192);
    const int parts = (int)(fused ? ln_blocks(rows, dim, vec) : ln_parts(rows));
    const int blocks = fused ? parts : (int)(rows < 512 ? rows : 512);
    float* partials = params ? static_cast<float*>(workspace) : nullptr;
    hipStream_t s = static_cast<hipStream_t>(stream);
#define LN_BWD(DT, VEC)                                                                                                                                    \
    do {                                                                                                                                                   \
        constexpr bool fused = ln_fused<VEC, T, CH>();                                                                                                     \
        if (fused || (dx && rows))                                                                                                                         \
            layernorm_backward_kernel<DT, VEC, T, CH><<<blocks, ln_threads<T>(), 0, s>>>(grad, grad_row_stride, x, x_row_stride, w, w_dtype == Q8_F32, mean, \
                                                                                         rstd, dx, partials, rows, dim);                                  \
        if (!fused && params)                                                                                                                              \
            layernorm_columns_kernel<DT, VEC><<<dim3((unsigned)((dim + 256 * VEC - 1) / (256 * VEC)), (unsigned)parts), 256, 0, s>>>(                       \
                grad, grad_row_stride, x, x_row_stride, mean, rstd, partials, rows, dim);                                                                  \
    } while (0)
    LN_BY_TYPE(vec, false, LN_BWD);
#undef LN_BWD
    if (int e = launch_status("q8_layernorm_backward")) return e;
    if (params) {
        layernorm_params_kernel<<<(2 * dim + 31) / 32, 1024, 0, s>>>(partials, parts, dw, db, wd, dim);
        return launch_status("q8_layernorm_backward");
    }
    return Q8_OK;
}
