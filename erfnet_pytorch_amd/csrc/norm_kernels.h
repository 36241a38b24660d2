// Layer norm over the last axis of dense rows [rows][C]: y = (x - mean) * rstd * w + b, rstd = 1 / sqrt(var + eps)
// with the biased variance, and its gradients
//   dx = rstd * (g w - mean(g w) - xhat * mean(g w xhat)),   dw = sum over rows of g xhat,   db = sum over rows of g.
//
// Bound by memory: forward reads x and writes y, backward reads x and g and writes dx; a row stays in registers
// between its statistics and its result, so nothing is read twice.  Statistics, products and sums are fp32; the mean
// is taken first and the squares of the differences after it (E[x^2] - mean^2 loses the variance of a row whose level
// is far from zero).  The first mean carries its sum's roundings, which are small against the level and not against the spread:
// the differences' own sum, behind the same barrier as their squares, takes them out of mean, variance and differences.
// Equal values have themselves as their mean, no variance and y = b.  (fp32 rows of level 1000 and spread 0.01: y off by
// 1e-2 without, 4e-6 with it; 49152 x 128 9.2 -> 9.8 us, 20000 x 1030 31.7 -> 33.4, others within 1 %.)
#pragma once
#include "vec16.h"
#include "wave.h"

#define NORM_BLOCK 256
#define NORM_MAX_C 16384

struct NormDesc {
    const void *x, *gy;         // [rows][C], storage type T
    void *y;                    // forward: y; backward: dx
    const float *w, *b;         // [C] or null
    float *mean, *rstd;         // [rows]; forward may leave them null
    float *partial;             // backward: [blocks][2][C] sums of g xhat and of g
    long long rows, safe_rows;  // of the first safe_rows rows, a vector that begins in the row ends in the tensor
    int C;
    float eps;
};

// s / C from 1 / C, the product's remainder added back: a sum that is exact has its mean rounded once.
__device__ __forceinline__ float norm_mean(float s, float c, float inv_c)
{
    const float q = s * inv_c;
    return __builtin_fmaf(__builtin_fmaf(-q, c, s), inv_c, q);
}

// Sums of one or two values over LANES lanes, or over a block of whole waves (0); `red` holds a slot per wave and value
// and alternates between calls.
template <int LANES, int M> __device__ __forceinline__ void norm_sum(float (&v)[M], float (&red)[M][16])
{
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] = wave_sum(v[m], LANES ? LANES : 64);
    if (LANES) return;
    if ((threadIdx.x & 63) == 0)
        for (int m = 0; m < M; ++m) red[m][threadIdx.x >> 6] = v[m];
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] = 0.0f;
    for (int i = 0; i < (int)(blockDim.x >> 6); ++i)
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] += red[m][i];
}

// The vectors of one row that a thread holds: R of them, `threads` apart, this thread's first at vector `me`.  EVEN: C is a
// multiple of the vector.  Otherwise a row's last vector reads on into the next rows (where there are any: safe_rows), and
// what it reads of them is cut off where it is unpacked (norm_unpack): the load itself has no wait.
template <typename T, int R, bool EVEN>
__device__ __forceinline__ void norm_load(u32x4 (&raw)[R], const NormDesc &d, const void *base, long long row, int me, int threads)
{
    const T *x = (const T *)base + row * d.C;
    const bool inside = row < d.safe_rows;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = (r * threads + me) * Vec16<T>::N;
        if constexpr (EVEN) {
            raw[r] = (u32x4){0u, 0u, 0u, 0u};
            if (c < d.C) raw[r] = reinterpret_cast<const typename Vec16<T>::Raw *>(x + c)->v;
        } else {
            raw[r] = ld16(x + c, d.C - c, inside);
        }
    }
}
template <typename T, bool EVEN> __device__ __forceinline__ void norm_unpack(u32x4 raw, float (&f)[Vec16<T>::N], int left)
{
    if (!EVEN && left < Vec16<T>::N) raw = first16<T>(raw, left);
    Vec16<T>::unpack(raw, f);
}
template <typename T, bool EVEN> __device__ __forceinline__ void norm_store(T *p, const float (&f)[Vec16<T>::N], int left)
{
    if constexpr (EVEN) {
        if (left > 0) reinterpret_cast<typename Vec16<T>::Raw *>(p)->v = Vec16<T>::pack(f);
    } else {
        st16(p, f, left);
    }
}

// N parameters from channel c on, `none` where there are none.  (16 bytes a load: one by one, the weight and bias of 8191 x 2048
// bf16, read for two rows a block, took most of its 37 us.)
template <int N, bool EVEN>
__device__ __forceinline__ void norm_params(float (&f)[N], const float *p, int c, int C, float none)
{
    struct __attribute__((packed, aligned(4))) Four { f32x4 v; };
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        f32x4 v = {none, none, none, none};
        if (p && c + i + 3 < C) v = reinterpret_cast<const Four *>(p + c + i)->v;
        else if (p && !EVEN)
            for (int j = 0; j < 3; ++j)
                if (c + i + j < C) v[j] = p[c + i + j];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[i + j] = v[j];
    }
}

// LANES > 0: one row per LANES lanes of a wave; 0: one row per block.  Every thread walks over rows and has
// the next row's loads in flight while it works on one, so the latency of memory and of the two sums behind one
// another overlaps with the loads; weight and bias stay in registers.  (Short rows are bound by instructions as much as by
// memory: with the lane count and the shape of a row's end known to the compiler, 990099 x 101 fp32 takes 173 us instead
// of 209.)
template <typename T, int R, int LANES, bool EVEN>
__global__ __launch_bounds__(LANES ? NORM_BLOCK : 1024) void norm_fwd_kernel(const NormDesc d)
{
    // (bf16: sums of up to 2^14 values of 8 bits need no rounding where the values are equal, and little where they are close)
    constexpr bool BLOCK = LANES == 0, AGAIN = sizeof(T) == 4;
    constexpr int N = Vec16<T>::N;
    __shared__ float red1[1][16], red2[AGAIN ? 2 : 1][16];
    const int C = d.C, threads = BLOCK ? (int)blockDim.x : LANES;
    const int me = BLOCK ? (int)threadIdx.x : (int)threadIdx.x & (LANES - 1);
    constexpr int rows_per_block = BLOCK ? 1 : NORM_BLOCK / (BLOCK ? 1 : LANES);
    const long long stride = (long long)gridDim.x * rows_per_block;
    long long row = (long long)blockIdx.x * rows_per_block + (BLOCK ? 0 : threadIdx.x / (BLOCK ? 1 : LANES));
    if (row >= d.rows) return;                  // (in a block kernel the grid has no more blocks than rows)
    u32x4 next[R];
    norm_load<T, R, EVEN>(next, d, d.x, row, me, threads);
    float w[R][N], b[R][N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        norm_params<N, EVEN>(w[r], d.w, (r * threads + me) * N, C, 1.0f);
        norm_params<N, EVEN>(b[r], d.b, (r * threads + me) * N, C, 0.0f);
    }
    const float inv_c = 1.0f / (float)C;
    for (; row < d.rows; row += stride) {
        float v[R][N], s[1] = {0.0f};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            norm_unpack<T, EVEN>(next[r], v[r], C - (r * threads + me) * N);
#pragma unroll
            for (int i = 0; i < N; ++i) s[0] += v[r][i];
        }
        if (row + stride < d.rows) norm_load<T, R, EVEN>(next, d, d.x, row + stride, me, threads);
        norm_sum<LANES>(s, red1);
        const float mean = norm_mean(s[0], (float)C, inv_c);
        // (above 2^60 the differences are taken 2^-64 fold, so that the squares of a few units in the last place stay inside fp32)
        const bool high = AGAIN && fabsf(mean) > 1.152921504606846976e18f;
        const float unit = high ? 5.42101086242752217e-20f : 1.0f, whole = high ? 18446744073709551616.0f : 1.0f;
        float q[AGAIN ? 2 : 1] = {0.0f};        // squares of the differences, and the differences
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * threads + me) * N;
            const float from = c < C ? -mean * unit : 0.0f;     // (behind the row there are zeros)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[r][i] = __builtin_fmaf(v[r][i], unit, EVEN || c + i < C ? from : 0.0f);
                q[0] += v[r][i] * v[r][i];
                if (AGAIN) q[1] += v[r][i];
            }
        }
        norm_sum<LANES>(q, red2);
        float rest = 0.0f, left = q[0];
        if (AGAIN) {
            rest = norm_mean(q[1], (float)C, inv_c);
            left = __builtin_fmaf(-q[1], rest, q[0]);
            // (rounded below zero: none left; infinity minus infinity: the squares were beyond fp32, and stay so)
            left = left >= 0.0f ? left : left < 0.0f ? 0.0f : q[0];
        }
        const float rstd = rsqrtf(left * inv_c * whole * whole + d.eps), scale = rstd * whole;
        if (me == 0 && d.mean) { d.mean[row] = mean + rest * whole; d.rstd[row] = rstd; }
        T *y = (T *)d.y + row * C;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * threads + me) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) v[r][i] = (AGAIN ? v[r][i] - rest : v[r][i]) * scale * w[r][i] + b[r][i];
            norm_store<T, EVEN>(y + c, v[r], C - c);
        }
    }
}

// Backward, the same walk, from the last row to the first: what was read and written last is what the 256 MB cache
// still has (8191 x 8192 bf16, forward and backward: 136 -> 131 us).  Every thread keeps the weight's and bias's gradient of its own channels in registers over
// all rows it meets; the block's sums go to partial, and norm_grad_sum_kernel adds the blocks in order.
// THREADS: most threads of a block kernel (0: wave kernel).  Beyond 8192 channels bf16 takes 32 elements a thread, whose 256
// registers hold the sums and the next row's loads, fp32 1024 threads with 128 registers for the sums alone; the weight is read again for
// every row (4000 x 12000, 1024 / 512 threads: bf16 83 / 73 us, fp32 120 / 124).
template <typename T, int R, int LANES, int THREADS, bool EVEN>
__global__ __launch_bounds__(THREADS ? THREADS : NORM_BLOCK) void norm_bwd_kernel(const NormDesc d)
{
    constexpr bool BLOCK = THREADS != 0, HELD = THREADS != 1024 && R * Vec16<T>::N <= 16, AHEAD = THREADS != 1024;
    static_assert(BLOCK == (LANES == 0), "one of the two");
    constexpr int N = Vec16<T>::N;
    extern __shared__ float acc[];              // wave kernel: [4 waves][2][C]
    __shared__ float red[2][2][16];
    const int C = d.C, threads = BLOCK ? (int)blockDim.x : LANES;
    const int me = BLOCK ? (int)threadIdx.x : (int)threadIdx.x & (LANES - 1);
    constexpr int rows_per_block = BLOCK ? 1 : NORM_BLOCK / (BLOCK ? 1 : LANES);
    const long long stride = (long long)gridDim.x * rows_per_block;
    long long row = (long long)blockIdx.x * rows_per_block + (BLOCK ? 0 : threadIdx.x / (BLOCK ? 1 : LANES));
    u32x4 nx[R], ng[R];
    float nmean = 0.0f, nrstd = 0.0f;
    auto fetch = [&](long long row) __attribute__((always_inline)) {
        const long long at = d.rows - 1 - row;
        norm_load<T, R, EVEN>(nx, d, d.x, at, me, threads);
        norm_load<T, R, EVEN>(ng, d, d.gy, at, me, threads);
        nmean = d.mean[at];
        nrstd = d.rstd[at];
    };
    if (AHEAD && row < d.rows) fetch(row);
    float w[R][N], dw[R][N], db[R][N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (HELD) norm_params<N, EVEN>(w[r], d.w, (r * threads + me) * N, C, 1.0f);
#pragma unroll
        for (int i = 0; i < N; ++i) dw[r][i] = db[r][i] = 0.0f;
    }
    const float inv_c = 1.0f / (float)C;
    int turn = 0;
    for (; row < d.rows; row += stride, turn ^= 1) {
        if (!AHEAD) fetch(row);
        const float mean = nmean, rstd = nrstd;
        float h[R][N], g[R][N], s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * threads + me) * N;
            norm_unpack<T, EVEN>(nx[r], h[r], C - c);
            norm_unpack<T, EVEN>(ng[r], g[r], C - c);         // zero beyond the row: nothing below counts it
            if (!HELD) norm_params<N, EVEN>(w[r], d.w, c, C, 1.0f);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                // (s1 without rstd: behind the row's end, where x and g are zero, 0 - mean in units of the row's spread may pass the
                // type's range, and infinity times zero would be counted.  Differences are below 2^64 wherever fp32 holds their
                // squares; where it does not, rstd is 0 and s1 with it.)
                const float off = h[r][i] - mean;
                h[r][i] = off * rstd;
                dw[r][i] += g[r][i] * h[r][i];
                db[r][i] += g[r][i];
                g[r][i] *= w[r][i];
                s0 += g[r][i];
                s1 += g[r][i] * off;
            }
        }
        if (AHEAD && row + stride < d.rows) fetch(row + stride);
        s0 = wave_sum(s0, BLOCK ? 64 : LANES);
        s1 = wave_sum(s1, BLOCK ? 64 : LANES);
        if (BLOCK) {
            // both sums behind one barrier; the slots alternate, so a wave that is a row ahead cannot overwrite them
            if ((threadIdx.x & 63) == 0) { red[turn][0][threadIdx.x >> 6] = s0; red[turn][1][threadIdx.x >> 6] = s1; }
            __syncthreads();
            s0 = s1 = 0.0f;
            for (int i = 0; i < (int)(blockDim.x >> 6); ++i) { s0 += red[turn][0][i]; s1 += red[turn][1][i]; }
        }
        s0 *= inv_c;
        s1 = rstd > 0.0f ? s1 * (inv_c * rstd) : 0.0f;
        T *dx = (T *)d.y + (d.rows - 1 - row) * C;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * threads + me) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) g[r][i] = rstd * (g[r][i] - s0 - h[r][i] * s1);
            if (d.y) norm_store<T, EVEN>(dx + c, g[r], C - c);
        }
    }
    if (!d.partial) return;
    float *out = d.partial + (long long)blockIdx.x * 2 * C;
    if (BLOCK) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * threads + me) * N;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (c + i < C) { out[c + i] = dw[r][i]; out[C + c + i] = db[r][i]; }
        }
        return;
    }
    // the rows of one wave, then the four waves
    float *mine = acc + (threadIdx.x >> 6) * 2 * C;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = (r * threads + me) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float a = dw[r][i], b = db[r][i];
#pragma unroll
            for (int o = BLOCK ? 64 : LANES; o < 64; o <<= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
            if ((threadIdx.x & 63) < threads && c + i < C) { mine[c + i] = a; mine[C + c + i] = b; }
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * C; j += NORM_BLOCK) out[j] = acc[j] + acc[2 * C + j] + acc[4 * C + j] + acc[6 * C + j];
}

// dw[c], db[c] = sum over blocks of partial[block][0 / 1][c]: COLS columns x 1024 / COLS rows of threads a block, each row's
// blocks in a fixed order, then the rows in order.  Few columns want many rows (there are few blocks to hide the latency of
// a row's loads), many columns want whole cache lines.
template <int COLS>
__global__ __launch_bounds__(1024) void norm_grad_sum_kernel(const float *partial, int nblocks, int C, float *dw, float *db)
{
    constexpr int ROWS = 1024 / COLS;
    __shared__ float red[ROWS][COLS + 1];
    const int col = threadIdx.x % COLS, part = threadIdx.x / COLS, j = blockIdx.x * COLS + col;
    float s = 0.0f;
    if (j < 2 * C) {
#pragma unroll 8
        for (int i = part; i < nblocks; i += ROWS) s += partial[(long long)i * 2 * C + j];
    }
    red[part][col] = s;
    __syncthreads();
    if (part == 0 && j < 2 * C) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) t += red[i][col];
        if (j < C) { if (dw) dw[j] = t; }
        else if (db) db[j - C] = t;
    }
}
