// Layer norm over the last axis of dense rows [rows][C]: y = (x - mean) * rstd * w + b, rstd = 1 / sqrt(var + eps)
// with the biased variance, and its gradients
//   dx = rstd * (g w - mean(g w) - xhat * mean(g w xhat)),   dw = sum over rows of g xhat,   db = sum over rows of g.
//
// Bound by memory: forward reads x and writes y, backward reads x and g and writes dx; a row stays in registers
// between its statistics and its result, so nothing is read twice.  Statistics, products and sums are fp32; the mean
// is taken first and the squares of the differences after it (E[x^2] - mean^2 loses the variance of a row whose level
// is far from zero), and it is a quotient, not a product with 1 / C: the mean of equal values is that value.
#pragma once
#include "vec16.h"

#define NORM_BLOCK 256
#define NORM_MAX_C 16384

struct NormDesc {
    const void *x, *gy;         // [rows][C], storage type T
    void *y;                    // forward: y; backward: dx
    const float *w, *b;         // [C] or null
    float *mean, *rstd;         // [rows]; forward may leave them null
    float *partial;             // backward: [blocks][2][C] sums of g xhat and of g
    long long rows;
    int C, lanes, lane_bits;    // lanes (a power of two) share a row in the wave kernels
    float eps;
};

__device__ __forceinline__ float norm_group_sum(float v, int lanes)
{
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// One row per `lanes` lanes of a wave, R vectors a lane.
template <typename T, int R>
__global__ __launch_bounds__(NORM_BLOCK) void norm_fwd_wave_kernel(const NormDesc d)
{
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & (d.lanes - 1), C = d.C;
    const int rows_per_block = NORM_BLOCK >> d.lane_bits;
    float w[R][N], b[R][N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = (r * d.lanes + lane) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[r][i] = d.w && c + i < C ? d.w[c + i] : 1.0f;
            b[r][i] = d.b && c + i < C ? d.b[c + i] : 0.0f;
        }
    }
    const float inv_c = 1.0f / (float)C;
    for (long long row = (long long)blockIdx.x * rows_per_block + (threadIdx.x >> d.lane_bits); row < d.rows;
         row += (long long)gridDim.x * rows_per_block) {
        const T *x = (const T *)d.x + row * C;
        float v[R][N], s = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * d.lanes + lane) * N;
            Vec16<T>::unpack(ld16(x + c, C - c), v[r]);
#pragma unroll
            for (int i = 0; i < N; ++i) s += v[r][i];
        }
        const float mean = norm_group_sum(s, d.lanes) / (float)C;
        float q = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * d.lanes + lane) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[r][i] = c + i < C ? v[r][i] - mean : 0.0f;
                q += v[r][i] * v[r][i];
            }
        }
        const float rstd = 1.0f / sqrtf(norm_group_sum(q, d.lanes) * inv_c + d.eps);
        if (lane == 0 && d.mean) { d.mean[row] = mean; d.rstd[row] = rstd; }
        T *y = (T *)d.y + row * C;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * d.lanes + lane) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) v[r][i] = v[r][i] * rstd * w[r][i] + b[r][i];
            if (c < C) st16(y + c, v[r], C - c);
        }
    }
}

// Sum over a block of whole waves; `red` holds a slot per wave and alternates between calls.
__device__ __forceinline__ float norm_block_sum(float v, float *red)
{
    v = norm_group_sum(v, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
    for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += red[i];
    return s;
}

// One row per block, R vectors a thread.
template <typename T, int R>
__global__ __launch_bounds__(1024) void norm_fwd_block_kernel(const NormDesc d)
{
    constexpr int N = Vec16<T>::N;
    __shared__ float red[2][16];
    const int C = d.C;
    const float inv_c = 1.0f / (float)C;
    for (long long row = blockIdx.x; row < d.rows; row += gridDim.x) {
        const T *x = (const T *)d.x + row * C;
        float v[R][N], s = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * (int)blockDim.x + (int)threadIdx.x) * N;
            Vec16<T>::unpack(ld16(x + c, C - c), v[r]);
#pragma unroll
            for (int i = 0; i < N; ++i) s += v[r][i];
        }
        const float mean = norm_block_sum(s, red[0]) / (float)C;
        float q = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * (int)blockDim.x + (int)threadIdx.x) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[r][i] = c + i < C ? v[r][i] - mean : 0.0f;
                q += v[r][i] * v[r][i];
            }
        }
        const float rstd = 1.0f / sqrtf(norm_block_sum(q, red[1]) * inv_c + d.eps);
        if (threadIdx.x == 0 && d.mean) { d.mean[row] = mean; d.rstd[row] = rstd; }
        T *y = (T *)d.y + row * C;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * (int)blockDim.x + (int)threadIdx.x) * N;
            if (c >= C) continue;
            float o[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int j = c + i < C ? c + i : C - 1;
                o[i] = v[r][i] * rstd * (d.w ? d.w[j] : 1.0f) + (d.b ? d.b[j] : 0.0f);
            }
            st16(y + c, o, C - c);
        }
    }
}

// Backward, one row per `lanes` lanes.  Every thread keeps the weight's and bias's gradient of its own channels in
// registers over all rows it meets; the block's sums go to partial, and norm_grad_sum_kernel adds the blocks in order.
template <typename T, int R>
__global__ __launch_bounds__(NORM_BLOCK) void norm_bwd_wave_kernel(const NormDesc d)
{
    constexpr int N = Vec16<T>::N;
    extern __shared__ float acc[];              // [4 waves][2][C]
    const int lane = threadIdx.x & (d.lanes - 1), C = d.C;
    const int rows_per_block = NORM_BLOCK >> d.lane_bits;
    float w[R][N], dw[R][N], db[R][N];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = (r * d.lanes + lane) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[r][i] = d.w && c + i < C ? d.w[c + i] : 1.0f;
            dw[r][i] = db[r][i] = 0.0f;
        }
    }
    const float inv_c = 1.0f / (float)C;
    for (long long row = (long long)blockIdx.x * rows_per_block + (threadIdx.x >> d.lane_bits); row < d.rows;
         row += (long long)gridDim.x * rows_per_block) {
        const T *x = (const T *)d.x + row * C, *gy = (const T *)d.gy + row * C;
        const float mean = d.mean[row], rstd = d.rstd[row];
        float h[R][N], g[R][N], s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * d.lanes + lane) * N;
            Vec16<T>::unpack(ld16(x + c, C - c), h[r]);
            Vec16<T>::unpack(ld16(gy + c, C - c), g[r]);        // zero beyond the row: nothing below counts it
#pragma unroll
            for (int i = 0; i < N; ++i) {
                h[r][i] = (h[r][i] - mean) * rstd;
                dw[r][i] += g[r][i] * h[r][i];
                db[r][i] += g[r][i];
                g[r][i] *= w[r][i];
                s0 += g[r][i];
                s1 += g[r][i] * h[r][i];
            }
        }
        s0 = norm_group_sum(s0, d.lanes) * inv_c;
        s1 = norm_group_sum(s1, d.lanes) * inv_c;
        T *dx = (T *)d.y + row * C;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * d.lanes + lane) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) g[r][i] = rstd * (g[r][i] - s0 - h[r][i] * s1);
            if (c < C && d.y) st16(dx + c, g[r], C - c);
        }
    }
    if (!d.partial) return;
    // the rows of one wave, then the four waves
    float *mine = acc + (threadIdx.x >> 6) * 2 * C;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = (r * d.lanes + lane) * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float a = dw[r][i], b = db[r][i];
            for (int o = d.lanes; o < 64; o <<= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
            if ((threadIdx.x & 63) < d.lanes && c + i < C) { mine[c + i] = a; mine[C + c + i] = b; }
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * C; j += NORM_BLOCK)
        d.partial[(long long)blockIdx.x * 2 * C + j] = acc[j] + acc[2 * C + j] + acc[4 * C + j] + acc[6 * C + j];
}

template <typename T, int R>
__global__ __launch_bounds__(1024) void norm_bwd_block_kernel(const NormDesc d)
{
    constexpr int N = Vec16<T>::N;
    __shared__ float red[2][2][16];
    const int C = d.C;
    float dw[R][N], db[R][N];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < N; ++i) dw[r][i] = db[r][i] = 0.0f;
    const float inv_c = 1.0f / (float)C;
    int turn = 0;
    for (long long row = blockIdx.x; row < d.rows; row += gridDim.x, turn ^= 1) {
        const T *x = (const T *)d.x + row * C, *gy = (const T *)d.gy + row * C;
        const float mean = d.mean[row], rstd = d.rstd[row];
        float h[R][N], g[R][N], s0 = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * (int)blockDim.x + (int)threadIdx.x) * N;
            Vec16<T>::unpack(ld16(x + c, C - c), h[r]);
            Vec16<T>::unpack(ld16(gy + c, C - c), g[r]);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                h[r][i] = (h[r][i] - mean) * rstd;
                dw[r][i] += g[r][i] * h[r][i];
                db[r][i] += g[r][i];
                if (d.w) g[r][i] *= d.w[c + i < C ? c + i : C - 1];
                s0 += g[r][i];
                s1 += g[r][i] * h[r][i];
            }
        }
        // both sums behind one barrier; the slots alternate, so a wave that is a row ahead cannot overwrite them
        s0 = norm_group_sum(s0, 64);
        s1 = norm_group_sum(s1, 64);
        if ((threadIdx.x & 63) == 0) { red[turn][0][threadIdx.x >> 6] = s0; red[turn][1][threadIdx.x >> 6] = s1; }
        __syncthreads();
        s0 = s1 = 0.0f;
        for (int i = 0; i < (int)(blockDim.x >> 6); ++i) { s0 += red[turn][0][i]; s1 += red[turn][1][i]; }
        s0 *= inv_c;
        s1 *= inv_c;
        T *dx = (T *)d.y + row * C;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = (r * (int)blockDim.x + (int)threadIdx.x) * N;
#pragma unroll
            for (int i = 0; i < N; ++i) g[r][i] = rstd * (g[r][i] - s0 - h[r][i] * s1);
            if (c < C && d.y) st16(dx + c, g[r], C - c);
        }
    }
    if (!d.partial) return;
    float *out = d.partial + (long long)blockIdx.x * 2 * C;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = (r * (int)blockDim.x + (int)threadIdx.x) * N;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (c + i < C) { out[c + i] = dw[r][i]; out[C + c + i] = db[r][i]; }
    }
}

// dw[c], db[c] = sum over blocks of partial[block][0 / 1][c]: 32 columns x 32 rows of threads a block, rows in a fixed
// order, then the 32 rows in order.
__global__ __launch_bounds__(1024) void norm_grad_sum_kernel(const float *partial, int nblocks, int C, float *dw, float *db)
{
    __shared__ float red[32][33];
    const int col = threadIdx.x & 31, part = threadIdx.x >> 5, j = blockIdx.x * 32 + col;
    float s = 0.0f;
    if (j < 2 * C)
        for (int i = part; i < nblocks; i += 32) s += partial[(long long)i * 2 * C + j];
    red[part][col] = s;
    __syncthreads();
    if (part == 0 && j < 2 * C) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += red[i][col];
        if (j < C) { if (dw) dw[j] = t; }
        else if (db) db[j - C] = t;
    }
}
