// Log probabilities of given classes, entropy and the likeliest alternatives of a softmax over a class axis, and the
// gradient of all three.  With m = max x, S = sum e^(x - m), A = sum e^(x - m) (x - m):
//   log p_i = x_i - m - log S        H = -sum p log p = log S - A / S
//   dx_i = -p_i (G + g_H (log p_i + H)) + [upstream gradients of the entries gathered at i],   G = their sum.
//
// Forward reads the logits once: a thread keeps (m, S, A) of what it has seen and moves them to a new maximum when one
// turns up; threads, waves and blocks join theirs the same way.  Backward reads the logits once more (m and log S are
// kept per row as two numbers: their sum would lose log S to the rounding of a large m) and writes the gradient.
//
// Entries of -infinity (masked classes) have probability 0 and add nothing; where all are -infinity the
// log probabilities are -infinity, the entropy 0 and the gradient 0.  A NaN or +infinity makes its row NaN.
// Alternatives are ordered by logit, larger first, NaN before all, equal ones by index: one 64-bit key per entry.
#pragma once
#include "vec16.h"

#define LP_BLOCK 256
#define LP_MAX_TOP 64
#define LP_LOWEST (-3.402823466e+38f)
// e^-200 is 0 in fp32: exponents stop here where they are also a factor, so that 0 * infinity cannot arise
#define LP_FLOOR (-200.0f)

struct LpDesc {
    const void *x;              // logits, storage type T
    const long long *target;    // [rows]
    float *log_prob, *entropy;  // [rows]
    float2 *stats;              // [rows] (m, log S); log S = -infinity marks a row with no class
    float *top_lp;              // row kernels [rows][k], pixel kernel [outer][k][inner]
    long long *top_idx;
    long long rows;             // row kernels: rows; pixel kernels: outer * inner
    long long ld;               // row kernels: elements from row to row
    long long inner;            // pixel kernels
    long long ignore;
    int V, k;
    int splits, seg;            // row kernels: blocks per row and elements of each
    float4 *part;               // splits > 1: [rows][splits] (m, S, A, -)
    unsigned long long *part_keys;  // [rows][splits][k]
    // backward
    const float *g_lp, *g_h, *g_top;    // null: zero
    void *dx;
};

__device__ __forceinline__ unsigned lp_key32(float x)
{
    // order of the values as an order of unsigned numbers; the two zeros are one, NaN is above all, no entry gives 0
    const unsigned u = __builtin_bit_cast(unsigned, x + 0.0f);
    return x != x ? 0xffffffffu : (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float lp_key_value(unsigned k)
{
    return __builtin_bit_cast(float, k == 0xffffffffu ? 0x7fc00000u : (k >> 31) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned long long lp_key(float x, int index)
{
    return (unsigned long long)lp_key32(x) << 32 | (unsigned)~index;
}

struct LpSums { float m, s, a; };

__device__ __forceinline__ float lp_exp(float t) { return __builtin_amdgcn_exp2f(t * 1.44269504088896341f); }

// Moves the sums to the maximum `m`, m >= r.m.
__device__ __forceinline__ void lp_move(LpSums &r, float m)
{
    const float t = fmaxf(r.m - m, LP_FLOOR), f = lp_exp(t);
    r.a = f * (r.a + r.s * t);
    r.s *= f;
    r.m = m;
}
__device__ __forceinline__ void lp_add(LpSums &r, float x)      // x <= r.m, or NaN
{
    const float t = x - r.m, e = lp_exp(t);
    r.s += e;
    r.a += e * fmaxf(t, LP_FLOOR);
}
__device__ __forceinline__ void lp_join(LpSums &r, LpSums o)
{
    const float m = fmaxf(r.m, o.m);
    lp_move(r, m);
    lp_move(o, m);
    r.s += o.s;
    r.a += o.a;
}

// ---------------------------------------------------------------------------------- a wave's list of the largest keys
// Lane i of `list` holds the i-th largest key seen so far (0: none).  New candidates gather in 64 slots of shared
// memory; a full buffer is sorted and merged into the list (bitonic networks over the lanes).
__device__ __forceinline__ unsigned long long lp_shfl_xor(unsigned long long v, int o)
{
    const unsigned lo = __shfl_xor((unsigned)v, o), hi = __shfl_xor((unsigned)(v >> 32), o);
    return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ unsigned long long lp_shfl(unsigned long long v, int src)
{
    const unsigned lo = __shfl((unsigned)v, src), hi = __shfl((unsigned)(v >> 32), src);
    return (unsigned long long)hi << 32 | lo;
}
// descending over the lanes from a bitonic sequence
__device__ __forceinline__ unsigned long long lp_bitonic_clean(unsigned long long v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long w = lp_shfl_xor(v, o);
        const bool keep_max = (lane & o) == 0;
        v = (v > w) == keep_max ? v : w;
    }
    return v;
}
__device__ __forceinline__ unsigned long long lp_sort64(unsigned long long v)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const unsigned long long w = lp_shfl_xor(v, o);
            const bool keep_max = ((lane & o) == 0) == ((lane & size) == 0);
            v = (v > w) == keep_max ? v : w;
        }
    return v;
}
// both descending; the 64 largest of the 128
__device__ __forceinline__ unsigned long long lp_merge(unsigned long long list, unsigned long long other)
{
    const unsigned long long r = lp_shfl(other, 63 - (int)(threadIdx.x & 63));
    return lp_bitonic_clean(list > r ? list : r);
}

struct LpList {
    unsigned long long list = 0, kth = 0;
    float bar = -INFINITY;      // a value below the k-th largest cannot enter (compared with !(x < bar): NaN passes)
    int count = 0;              // candidates in the buffer
    volatile unsigned long long *buf;

    __device__ __forceinline__ void flush(int k)
    {
        const int lane = threadIdx.x & 63;
        unsigned long long v = lane < count ? buf[lane] : 0ull;
        list = lp_merge(list, lp_sort64(v));
        kth = lp_shfl(list, k - 1);
        // (uniform over the wave; an unfilled list lets everything through)
        bar = kth ? lp_key_value((unsigned)(kth >> 32)) : -INFINITY;
        if (bar != bar) bar = INFINITY;         // k NaNs so far: only another NaN passes the bar, and the key decides
        count = 0;
    }
    // every lane offers one key (0: none)
    __device__ __forceinline__ void offer(unsigned long long key, int k)
    {
        unsigned long long mask = __ballot(key > kth);
        if (!mask) return;
        if (count + __popcll(mask) > 64) {
            flush(k);
            mask = __ballot(key > kth);
        }
        if (key > kth) {
            const int below = __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
            buf[count + below] = key;
        }
        count += __popcll(mask);
    }
};

// ---------------------------------------------------------------------------------- rows: the class axis is the last
// What one thread does with its share of elements [from, to) of a row: vectors `threads` apart.
template <typename T, bool TOP>
__device__ __forceinline__ LpSums lp_scan(const T *x, int from, int to, int me, int threads, int k, LpList &top)
{
    constexpr int N = Vec16<T>::N;
    LpSums r = {LP_LOWEST, 0.0f, 0.0f};
    // all lanes of a wave take every turn (the list's votes need them)
    for (int base = from; base < to; base += threads * N) {
        const int c = base + me * N;
        const int left = to - c;
        float v[N];
        Vec16<T>::unpack(ld16(x + c, left), v);
        if (left < N) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = i < left ? v[i] : -INFINITY;
        }
        float m = r.m;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, v[i]);
        if (m > r.m) lp_move(r, m);
#pragma unroll
        for (int i = 0; i < N; ++i) lp_add(r, v[i]);
        if (TOP) {
            float high = v[0];
#pragma unroll
            for (int i = 1; i < N; ++i) high = fmaxf(high, v[i]);
            // (a NaN is lost by fmaxf but not by the sums)
            if (__ballot(left > 0 && (!(high < top.bar) || r.s != r.s))) {
#pragma unroll
                for (int i = 0; i < N; ++i) top.offer(i < left ? lp_key(v[i], c + i) : 0ull, k);
            }
        }
    }
    return r;
}

__device__ __forceinline__ LpSums lp_wave_join(LpSums r)
{
    for (int o = 32; o > 0; o >>= 1) {
        LpSums q = {__shfl_xor(r.m, o), __shfl_xor(r.s, o), __shfl_xor(r.a, o)};
        lp_join(r, q);
    }
    return r;
}

// The row's results, by one whole wave.
template <typename T>
__device__ __forceinline__ void lp_write_row(const LpDesc &d, long long row, const LpSums &r, unsigned long long list)
{
    const int lane = threadIdx.x & 63;
    const bool none = r.s == 0.0f;
    const float log_s = none ? -INFINITY : logf(r.s);
    if (lane == 0) {
        d.stats[row] = make_float2(r.m, log_s);
        d.entropy[row] = none ? 0.0f : log_s - r.a / r.s;
        const long long t = d.target[row];
        float lp = 0.0f;
        if (t != d.ignore && t >= 0 && t < d.V)
            lp = none ? -INFINITY : Vec16<T>::get((const T *)d.x + row * d.ld + t) - r.m - log_s;
        d.log_prob[row] = lp;
    }
    if (lane < d.k) {
        const float x = lp_key_value((unsigned)(list >> 32));
        d.top_lp[row * d.k + lane] = none ? -INFINITY : x - r.m - log_s;
        d.top_idx[row * d.k + lane] = (long long)(unsigned)~(unsigned)list;
    }
}

// GROUP = 64: a wave takes a row, four rows a block.  GROUP = 256: a block takes one of `splits` segments of a row.
template <typename T, int GROUP, bool TOP>
__global__ __launch_bounds__(LP_BLOCK) void lp_rows_kernel(const LpDesc d)
{
    __shared__ unsigned long long buf[TOP ? 4 : 1][64];
    __shared__ LpSums sums[4];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    long long row;
    int split = 0, me, from = 0, to = d.V;
    if (GROUP == 64) {
        row = (long long)blockIdx.x * 4 + wave;
        if (row >= d.rows) return;              // no barrier below on this path
        me = lane;
    } else {
        row = blockIdx.x / d.splits;
        split = (int)(blockIdx.x - row * d.splits);
        me = threadIdx.x;
        from = split * d.seg;
        to = from + d.seg < d.V ? from + d.seg : d.V;
    }
    LpList top;
    top.buf = buf[TOP ? wave : 0];
    LpSums r = lp_scan<T, TOP>((const T *)d.x + row * d.ld, from, to, me, GROUP, d.k, top);
    if (TOP) top.flush(d.k);
    r = lp_wave_join(r);
    if (GROUP == 64) {
        lp_write_row<T>(d, row, r, top.list);
        return;
    }
    // the four waves: sums through shared memory, lists in two rounds of merging
    if (lane == 0) sums[wave] = r;
    if (TOP) {
        volatile unsigned long long *l = buf[wave];
        l[lane] = top.list;
        __syncthreads();
        if (wave < 2) {
            top.list = lp_merge(top.list, ((volatile unsigned long long *)buf[wave + 2])[lane]);
            l[lane] = top.list;
        }
    }
    __syncthreads();
    if (wave != 0) return;
    for (int w = 1; w < 4; ++w) lp_join(r, sums[w]);
    if (TOP) top.list = lp_merge(top.list, ((volatile unsigned long long *)buf[1])[lane]);
    if (d.splits == 1) {
        lp_write_row<T>(d, row, r, top.list);
        return;
    }
    const long long at = row * d.splits + split;
    if (lane == 0) d.part[at] = make_float4(r.m, r.s, r.a, 0.0f);
    if (lane < d.k) d.part_keys[at * d.k + lane] = top.list;
}

// Joins the segments of a row: one block a row.
template <typename T>
__global__ __launch_bounds__(LP_BLOCK) void lp_join_kernel(const LpDesc d)
{
    __shared__ unsigned long long buf[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long row = blockIdx.x;
    unsigned long long list = 0;
    if (d.k) {
        for (int s = wave; s < d.splits; s += 4) {
            const unsigned long long o = lane < d.k ? d.part_keys[(row * d.splits + s) * d.k + lane] : 0ull;
            list = lp_merge(list, o);
        }
        buf[wave][lane] = list;
        __syncthreads();
        if (wave == 0)
            for (int w = 1; w < 4; ++w) list = lp_merge(list, buf[w][lane]);
    }
    if (wave != 0) return;
    LpSums r = {LP_LOWEST, 0.0f, 0.0f};
    for (int s = lane; s < d.splits; s += 64) {
        const float4 p = d.part[row * d.splits + s];
        lp_join(r, LpSums{p.x, p.y, p.z});
    }
    lp_write_row<T>(d, row, lp_wave_join(r), list);
}

// ---------------------------------------------------------------------------------- backward over rows
// One entry's gradient without what was gathered there.
__device__ __forceinline__ float lp_grad(float x, float m, float log_s, float G, float gh, float H)
{
    const float lp = x - m - log_s, p = lp_exp(lp);
    return -p * (G + gh * (fmaxf(lp, LP_FLOOR) + H));
}

// GROUP threads take a segment of a row (GROUP = 64: the whole row).
template <typename T, int GROUP>
__global__ __launch_bounds__(LP_BLOCK) void lp_rows_bwd_kernel(const LpDesc d)
{
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 63;
    long long row;
    int me, from = 0, to = d.V;
    if (GROUP == 64) {
        row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
        me = lane;
    } else {
        row = blockIdx.x / d.splits;
        me = threadIdx.x;
        from = (int)(blockIdx.x - row * d.splits) * d.seg;
        to = from + d.seg < d.V ? from + d.seg : d.V;
    }
    const bool live = row < d.rows;
    const T *x = (const T *)d.x + row * d.ld;
    T *dx = (T *)d.dx + row * (long long)d.V;
    float2 st = make_float2(0.0f, 0.0f);
    float H = 0.0f, gh = 0.0f, glp = 0.0f, G = 0.0f;
    long long t = -1;
    if (live) {
        st = d.stats[row];
        H = d.entropy[row];
        if (d.g_h) gh = d.g_h[row];
        t = d.target[row];
        if (t == d.ignore || t < 0 || t >= d.V) t = -1;
        if (t >= 0 && d.g_lp) glp = d.g_lp[row];
        float g = 0.0f;
        if (d.g_top && lane < d.k) g = d.g_top[row * d.k + lane];
        for (int o = 32; o > 0; o >>= 1) g += __shfl_xor(g, o);
        G = glp + g;
        const bool none = st.y == -INFINITY;
        for (int c = from + me * N; c < to; c += GROUP * N) {
            float v[N];
            Vec16<T>::unpack(ld16(x + c, to - c), v);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = none ? 0.0f : lp_grad(v[i], st.x, st.y, G, gh, H);
            st16(dx + c, v, to - c);
        }
    }
    // the gathered entries of this segment again, with what was gathered: after the block's plain stores
    __syncthreads();
    if (!live || st.y == -INFINITY) return;
    for (int e = me; e <= d.k; e += GROUP) {        // the alternatives, then the target
        long long pos = t;
        float add = glp;
        if (e < d.k) {
            pos = d.top_idx[row * d.k + e];
            add = (d.g_top ? d.g_top[row * d.k + e] : 0.0f) + (pos == t ? glp : 0.0f);
        } else {
            for (int j = 0; j < d.k; ++j)
                if (d.top_idx[row * d.k + j] == t) pos = -1;        // among the alternatives: added there
        }
        if (pos >= from && pos < to)
            Vec16<T>::put(dx + pos, lp_grad(Vec16<T>::get(x + pos), st.x, st.y, G, gh, H) + add);
    }
}

// ---------------------------------------------------------------------------------- pixels: [outer][V][inner]
// A thread takes one pixel and walks the classes; neighbouring threads take neighbouring pixels.  K >= k alternatives
// in registers.
template <typename T, int K>
__global__ __launch_bounds__(LP_BLOCK) void lp_pixels_kernel(const LpDesc d)
{
    const long long p = (long long)blockIdx.x * LP_BLOCK + threadIdx.x;
    if (p >= d.rows) return;
    const long long n = p / d.inner, q = p - n * d.inner;
    const T *x = (const T *)d.x + n * d.V * d.inner + q;
    LpSums r = {LP_LOWEST, 0.0f, 0.0f};
    unsigned key[K > 0 ? K : 1];
    int idx[K > 0 ? K : 1];
#pragma unroll
    for (int j = 0; j < K; ++j) { key[j] = 0u; idx[j] = 0; }
    for (int c = 0; c < d.V; c += 4) {
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int cc = c + i < d.V ? c + i : d.V - 1;
            v[i] = Vec16<T>::get(x + (long long)cc * d.inner);
        }
        float m = r.m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (c + i >= d.V) v[i] = -INFINITY;
            m = fmaxf(m, v[i]);
        }
        if (m > r.m) lp_move(r, m);
#pragma unroll
        for (int i = 0; i < 4; ++i) lp_add(r, v[i]);
        if (K > 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                // strictly larger only: of equal entries the earlier one stays; what is displaced moves down one
                unsigned kk = c + i < d.V ? lp_key32(v[i]) : 0u;
                int ii = c + i;
                bool up = false;
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    up = up || kk > key[j];
                    const unsigned k0 = key[j];
                    const int i0 = idx[j];
                    key[j] = up ? kk : k0;
                    idx[j] = up ? ii : i0;
                    kk = up ? k0 : kk;
                    ii = up ? i0 : ii;
                }
            }
        }
    }
    const bool none = r.s == 0.0f;
    const float log_s = none ? -INFINITY : logf(r.s);
    d.stats[p] = make_float2(r.m, log_s);
    d.entropy[p] = none ? 0.0f : log_s - r.a / r.s;
    const long long t = d.target[p];
    float lp = 0.0f;
    if (t != d.ignore && t >= 0 && t < d.V) lp = none ? -INFINITY : Vec16<T>::get(x + t * d.inner) - r.m - log_s;
    d.log_prob[p] = lp;
    if (K > 0) {
#pragma unroll
        for (int j = 0; j < K; ++j)
            if (j < d.k) {
                const long long at = (n * d.k + j) * d.inner + q;
                d.top_lp[at] = none ? -INFINITY : lp_key_value(key[j]) - r.m - log_s;
                d.top_idx[at] = idx[j];
            }
    }
}

template <typename T, int K>
__global__ __launch_bounds__(LP_BLOCK) void lp_pixels_bwd_kernel(const LpDesc d)
{
    const long long p = (long long)blockIdx.x * LP_BLOCK + threadIdx.x;
    if (p >= d.rows) return;
    const long long n = p / d.inner, q = p - n * d.inner;
    const T *x = (const T *)d.x + n * d.V * d.inner + q;
    T *dx = (T *)d.dx + n * d.V * d.inner + q;
    const float2 st = d.stats[p];
    const float H = d.entropy[p], gh = d.g_h ? d.g_h[p] : 0.0f;
    const bool none = st.y == -INFINITY;
    long long t = d.target[p];
    if (t == d.ignore || t < 0 || t >= d.V) t = -1;
    const float glp = t >= 0 && d.g_lp ? d.g_lp[p] : 0.0f;
    float G = glp, gt[K > 0 ? K : 1];
    int idx[K > 0 ? K : 1];
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const long long at = (n * d.k + j) * d.inner + q;
        const bool on = j < d.k && d.g_top;
        gt[j] = on ? d.g_top[at] : 0.0f;
        idx[j] = on ? (int)d.top_idx[at] : -1;
        G += gt[j];
    }
#pragma unroll 4
    for (int c = 0; c < d.V; ++c) {
        float g = lp_grad(Vec16<T>::get(x + (long long)c * d.inner), st.x, st.y, G, gh, H);
        if (c == (int)t) g += glp;
#pragma unroll
        for (int j = 0; j < K; ++j) g += idx[j] == c ? gt[j] : 0.0f;
        Vec16<T>::put(dx + (long long)c * d.inner, none ? 0.0f : g);
    }
}
