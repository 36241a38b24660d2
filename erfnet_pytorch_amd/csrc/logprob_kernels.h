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
#include "wave.h"

#define LP_BLOCK 256
#define LP_MAX_TOP 64
#define LP_LOWEST (-3.402823466e+38f)
// e^-200 is 0 in fp32: exponents stop here where they are also a factor, so that 0 * infinity cannot arise
#define LP_FLOOR (-200.0f)

struct LpDesc {
    const void *x;              // logits, storage type T
    const long long *target;    // [rows]
    float *log_prob, *entropy;  // [rows]
    float2 *stats;              // [rows] (m, log S); log S = -infinity marks a row with no class.  Forward: may be null
    float *top_lp;              // row kernels [rows][k], pixel kernel [outer][k][inner]
    long long *top_idx;
    long long rows;             // row kernels: rows; pixel kernels: outer * inner
    long long ld;               // row kernels: elements from row to row
    long long inner, group, next;   // pixel kernels: pixel p is element (p / inner) * group + p % inner, its classes `next` apart
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

// ---------------------------------------------------------------------------------- the largest keys
// The scan itself looks for no alternatives: it leaves every thread with its maximum, and the k-th largest of those is a
// bar that at least k entries reach.  Only threads whose maximum reaches it can hold an alternative, about k of them, and only
// their entries are read again.  (Filtering entries against a running bar inside the scan took 240 us for 2047 rows of
// 100003 bf16 classes, k = 8, the bar 114 when it came in its place, the scan without alternatives 82.)
//
// Sorting networks over the 64 lanes, larger values in lower lanes.
template <int O> __device__ __forceinline__ unsigned lp_xor(unsigned v) { return wave_xor<O>(v); }
template <int O> __device__ __forceinline__ unsigned long long lp_xor(unsigned long long v)
{
    return (unsigned long long)wave_xor<O>((unsigned)(v >> 32)) << 32 | wave_xor<O>((unsigned)v);
}
__device__ __forceinline__ unsigned lp_reverse(unsigned v) { return wave_reverse(v); }
__device__ __forceinline__ unsigned long long lp_reverse(unsigned long long v)
{
    return (unsigned long long)wave_reverse((unsigned)(v >> 32)) << 32 | wave_reverse((unsigned)v);
}
// descending over aligned groups of 2 * O lanes, from bitonic sequences; `turn`: ascending instead
template <int O, typename K> __device__ __forceinline__ K lp_clean(K v, bool turn)
{
    const K w = lp_xor<O>(v);
    const bool keep_max = ((threadIdx.x & O) == 0) != turn;
    v = (v > w) == keep_max ? v : w;
    if constexpr (O > 1) return lp_clean<O / 2>(v, turn);
    return v;
}
template <typename K> __device__ __forceinline__ K lp_sort64(K v)
{
    const unsigned lane = threadIdx.x & 63;
    v = lp_clean<1>(v, lane & 2);
    v = lp_clean<2>(v, lane & 4);
    v = lp_clean<4>(v, lane & 8);
    v = lp_clean<8>(v, lane & 16);
    v = lp_clean<16>(v, lane & 32);
    return lp_clean<32>(v, false);
}
// both descending; the 64 largest of the 128
template <typename K> __device__ __forceinline__ K lp_merge(K list, K other)
{
    const K r = lp_reverse(other);
    return lp_clean<32>(list > r ? list : r, false);
}

// A wave's candidates: up to 64 wait in shared memory; a full buffer is sorted into `list` (lane i: the i-th largest so
// far, 0: none), after which nothing below its k-th enters.
// (pointers into shared memory say so: a plain volatile pointer is read by flat loads)
typedef __attribute__((address_space(3))) volatile unsigned long long lp_lds64;
typedef __attribute__((address_space(3))) volatile unsigned char lp_lds8;
struct LpList {
    unsigned long long list = 0, kth = 0;
    int count = 0;
    bool sorted = false;        // whether list holds anything
    lp_lds64 *buf;

    __device__ __forceinline__ void flush(int k)
    {
        const int lane = threadIdx.x & 63;
        const unsigned long long v = lp_sort64(lane < count ? buf[lane] : 0ull);
        list = sorted ? lp_merge(list, v) : v;
        sorted = true;
        kth = (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(list >> 32), k - 1) << 32 |
              (unsigned)__builtin_amdgcn_readlane((int)list, k - 1);
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
// Adds the values; gives back the largest.
template <int N, int U> __device__ __forceinline__ float lp_add_vectors(LpSums &r, const float (&v)[U][N])
{
    float high = v[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) high = fmaxf(high, v[u][i]);
    if (high > r.m) lp_move(r, high);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) lp_add(r, v[u][i]);
    return high;
}

// The turns of a scan, 16 elements a thread each, in four quarters; the last has the turn that may lack some as well.
struct LpTurns {
    int step, turns, left;      // elements of all threads' vectors; whole turns; elements behind them
    __device__ __forceinline__ LpTurns(int from, int to, int threads, int n, int u)
    {
        step = threads * n;
        turns = (to - from) / (step * u);
        left = to - from - turns * step * u;
    }
    __device__ __forceinline__ int begin(int quarter) const { return turns * quarter / 4; }
};

// Elements in front of the first cache line that begins at or behind p.
template <typename T> __device__ __forceinline__ int lp_head(const T *p, int left)
{
    const int h = (int)(-(unsigned)(unsigned long long)p & 127u) / (int)sizeof(T);
    return h < left ? h : left;
}

// What one thread does with its share of elements [from, to) of a row: one of the `first` that precede a cache line's
// beginning, then 16 at a time in vectors `threads` apart, with the next ones' loads in flight; the last turn, which may lack
// some, by itself.  TOP: high[0..3] receive the quarters' maxima (without the head's, which is given back).
template <typename T, bool TOP>
__device__ __forceinline__ LpSums lp_scan(const T *x, int from, int first, int to, int me, int threads, float &head, float (&high)[4])
{
    constexpr int N = Vec16<T>::N, U = 16 / N;
    LpSums r = {LP_LOWEST, 0.0f, 0.0f};
    head = -INFINITY;
    if (me < first) {
        head = Vec16<T>::get(x + from + me);
        if (head > r.m) lp_move(r, head);
        lp_add(r, head);
    }
    from += first;
    const LpTurns plan(from, to, threads, N, U);
    const int step = plan.step, turns = plan.turns;
    const T *at = x + from + me * N;
    u32x4 next[U];
    float v[U][N];
    int quarter = 0, until = plan.begin(1);
    high[0] = high[1] = high[2] = high[3] = -INFINITY;
    auto turn_page = [&]() __attribute__((always_inline)) {     // (three times in all: the first quarter ends in high[0])
        high[0] = high[1];
        high[1] = high[2];
        high[2] = high[3];
        high[3] = -INFINITY;
        until = plan.begin(++quarter + 1);
    };
    auto fetch = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = reinterpret_cast<const typename Vec16<T>::Raw *>(at + u * step)->v;
        at += step * U;
    };
    if (turns) fetch();
    for (int t = 0; t < turns; ++t) {
#pragma unroll
        for (int u = 0; u < U; ++u) Vec16<T>::unpack(next[u], v[u]);
        if (t + 1 < turns) fetch();
        if (TOP)
            while (quarter < 3 && t == until) turn_page();
        const float top = lp_add_vectors(r, v);
        if (TOP) high[3] = fmaxf(high[3], top);
    }
    if (TOP)
        while (quarter < 3) turn_page();
    const int c0 = from + turns * step * U + me * N;
    if (c0 < to) {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = ld16(x + c0 + u * step, to - c0 - u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Vec16<T>::unpack(next[u], v[u]);
#pragma unroll
            for (int i = 0; i < N; ++i) v[u][i] = c0 + u * step + i < to ? v[u][i] : -INFINITY;
        }
        const float top = lp_add_vectors(r, v);
        if (TOP) high[3] = fmaxf(high[3], top);
    }
    return r;
}

// A vector's entries that reach `bar`, into top, one from each lane a turn, the lowest first (left <= 0: none).
template <typename T>
__device__ __forceinline__ void lp_take(const T *x, int c, int left, unsigned bar, int k, LpList &top)
{
    constexpr int N = Vec16<T>::N;
    float v[N];
    Vec16<T>::unpack(ld16(x + c, left), v);
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) mine |= (i < left) & (lp_key32(v[i]) >= bar) ? 1u << i : 0u;
    while (__ballot(mine != 0u)) {
        const int j = __ffs(mine) - 1;          // (-1: nothing left, the selection below gives any of them)
        // element j by bit selection (written as ternaries it becomes an indexed register file)
        unsigned f[N];
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = __builtin_bit_cast(unsigned, v[i]);
#pragma unroll
        for (int half = N / 2; half > 0; half >>= 1) {
            unsigned pick = (j & half) ? ~0u : 0u;
            asm volatile("" : "+v"(pick));
#pragma unroll
            for (int i = 0; i < half; ++i) f[i] = (f[i] & ~pick) | (f[i + half] & pick);
        }
        top.offer(mine ? lp_key(__builtin_bit_cast(float, f[0]), c + j) : 0ull, k);
        mine &= mine - 1u;
    }
}

#define LP_MANY 512             // vectors
// The entries of this wave's threads that reach `bar`, into top.  high: the threads' quarters' maxima; `spoilt`: they do not
// show all there is; `best`: the largest key32 of any, if none is spoilt.  A lane takes one vector of one quarter that reaches
// the bar at a time, so that the few there are occupy the whole wave.  (Every such vector costs a cache line: by whole shares
// instead of quarters the second reading fetched 28 % of a row of 100003 bf16 classes again, k = 8.)
template <typename T>
__device__ __forceinline__ void lp_collect(const T *x, int from, int to, int first, int threads, const float (&high)[4],
                                           bool spoilt, unsigned bar, unsigned best, int k, lp_lds8 *owners, LpList &top)
{
    constexpr int N = Vec16<T>::N, U = 16 / N;
    const LpTurns plan(from, to, threads, N, U);
    const int lane = threadIdx.x & 63, step = plan.step;
    int n = 0, upto[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool some = plan.begin(j) < plan.begin(j + 1) || (j == 3 && plan.left > 0);
        const bool owner = some && (spoilt || lp_key32(high[j]) >= bar);
        const unsigned long long mask = __ballot(owner);
        const int at = n + __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
        if (owner) owners[at] = (unsigned char)(lane | j << 6);
        n += __popcll(mask);
        upto[j] = n;
    }
    const int most = (plan.turns + 3) / 4 * U + (plan.left > 0 ? U : 0);       // vectors of a quarter, at most
    if (n * most <= LP_MANY) {
        for (int q0 = 0; q0 < n * most; q0 += 64) {     // (the same number of turns for all lanes: the votes need them)
            const int q = q0 + lane, o = q / most, t = q - o * most;
            const unsigned own = q < n * most ? owners[o] : 0u;
            const int j = own >> 6, begin = plan.begin(j) * U, end = j == 3 ? begin + most : plan.begin(j + 1) * U;
            const int c = from + (begin + t) * step + (first + (int)(own & 63u)) * N;
            lp_take(x, c, q < n * most && begin + t < end && c < to ? to - c : 0, bar, k, top);
        }
        return;
    }
    // Very many: in the order of the row, until the list is full of entries that nothing behind them can pass.  (All of a row of
    // equal entries reach the bar, and a row of masked ones is such a row: with one in 61 of 2047 x 100003 bf16, k = 8, the others
    // waited for them, 184 us; 92 so.  In this order always: 64 x 50000, k = 32, 17 us, 14 in the other.)
    for (int j = 0; j < 4; ++j) {
        const int o0 = j ? upto[j - 1] : 0, count = upto[j] - o0, begin = plan.begin(j) * U;
        const int vectors = plan.begin(j + 1) * U - begin + (j == 3 && plan.left > 0 ? U : 0);
        for (int q0 = 0; q0 < count * vectors; q0 += 64) {
            const int lowest = from + (begin + q0 / count) * step + first * N;
            if (best < lp_key32(INFINITY) && ((unsigned long long)best << 32 | (unsigned)~lowest) < top.kth) return;
            const int q = q0 + lane, t = q / count;
            const bool live = q < count * vectors;
            const unsigned own = live ? owners[o0 + q - t * count] : 0u;
            const int c = from + (begin + t) * step + (first + (int)(own & 63u)) * N;
            lp_take(x, c, live && c < to ? to - c : 0, bar, k, top);
        }
    }
}

__device__ __forceinline__ LpSums lp_wave_join(LpSums r)
{
    const float m = wave_max(r.m);
    lp_move(r, m);
    r.s = wave_sum(r.s);
    r.a = wave_sum(r.a);
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
        if (d.stats) d.stats[row] = make_float2(r.m, log_s);
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
// (8 waves a SIMD: without the bound the scalar registers leave 7)
template <typename T, int GROUP, bool TOP>
__global__ __launch_bounds__(LP_BLOCK, 8) void lp_rows_kernel(const LpDesc d)
{
    __shared__ unsigned long long buf[TOP ? 4 : 1][64];
    __shared__ unsigned high[TOP ? 4 : 1][64];
    __shared__ unsigned char owners[TOP ? 4 : 1][256];
    __shared__ int counts[4];
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
    const T *x = (const T *)d.x + row * d.ld;
    float head, quarters[4];
    // Blocks stream long rows and begin at a cache line: their waves would share one at either end of every vector, and with 32 of
    // them on a compute unit it is fetched twice (4096 x 130001 bf16, top 8: 248 -> 209 us).  A wave that has a short row to
    // itself is faster without the detour (8192 x 3001: 20 and 23).
    const int first = GROUP == 256 ? lp_head(x + from, to - from) : 0;
    LpSums r = lp_scan<T, TOP>(x, from, first, to, me, GROUP, head, quarters);
    LpList top;
    if (TOP) {
        top.buf = (lp_lds64 *)buf[wave];
        // a thread's largest key, or a bound below it: the sums are NaN where it holds a NaN (which the maximum does not
        // show) or +infinity; 0 where it holds nothing
        const bool spoilt = r.s != r.s;
        const unsigned mine = me >= first && from + first + me * Vec16<T>::N >= to ? 0u : spoilt ? lp_key32(INFINITY)
                              : r.s == 0.0f ? lp_key32(-INFINITY) : lp_key32(r.m);
        unsigned best = lp_sort64(mine);
        if (GROUP == 256) {
            high[wave][lane] = best;
            __syncthreads();
            for (int w = 1; w < 4; ++w) best = lp_merge(best, high[(wave + w) & 3][lane]);
        }
        unsigned bar = (unsigned)__builtin_amdgcn_readlane((int)best, d.k - 1);
        if (bar < 1u) bar = 1u;
        if (GROUP == 256) top.offer(me < first && lp_key32(head) >= bar ? lp_key(head, from + me) : 0ull, d.k);
        lp_collect<T>(x, from + first, to, GROUP == 256 ? wave * 64 : 0, GROUP, quarters, spoilt, bar,
                      (unsigned)__builtin_amdgcn_readlane((int)best, 0), d.k, (lp_lds8 *)owners[wave], top);
    }
    r = lp_wave_join(r);
    if (GROUP == 64) {
        if (TOP) top.flush(d.k);
        lp_write_row<T>(d, row, r, top.list);
        return;
    }
    // the four waves' sums and candidates, through shared memory; the candidates are few enough for one sort as a rule
    if (lane == 0) {
        sums[wave] = r;
        if (TOP) counts[wave] = top.sorted ? 64 + 1 : top.count;
    }
    __syncthreads();
    if (TOP) {
        const int n0 = counts[0], n1 = n0 + counts[1], n2 = n1 + counts[2], n3 = n2 + counts[3];
        if (n3 <= 64) {
            if (wave == 0) {
                const int w = lane < n0 ? 0 : lane < n1 ? 1 : lane < n2 ? 2 : 3;
                const int at = lane - (w == 0 ? 0 : w == 1 ? n0 : w == 2 ? n1 : n2);
                top.list = lp_sort64(lane < n3 ? ((lp_lds64 *)buf[w])[at] : 0ull);
            }
        } else {
            top.flush(d.k);
            top.buf[lane] = top.list;
            __syncthreads();
            if (wave < 2) {
                top.list = lp_merge(top.list, ((lp_lds64 *)buf[wave + 2])[lane]);
                top.buf[lane] = top.list;
            }
            __syncthreads();
            if (wave == 0) top.list = lp_merge(top.list, ((lp_lds64 *)buf[1])[lane]);
        }
    }
    if (wave != 0) return;
    for (int w = 1; w < 4; ++w) lp_join(r, sums[w]);
    if (d.splits == 1) {
        lp_write_row<T>(d, row, r, top.list);
        return;
    }
    const long long at = row * d.splits + split;
    if (lane == 0) d.part[at] = make_float4(r.m, r.s, r.a, 0.0f);
    if (lane < d.k) d.part_keys[at * d.k + lane] = top.list;
}

// Joins the segments of a row.  WAVES = 1: a wave takes a row and merges its few lists one after the other, four rows a
// block; 16: a block takes a row, every wave merges each 16th list and four rounds join the waves'.
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? LP_BLOCK : WAVES * 64) void lp_join_kernel(const LpDesc d)
{
    __shared__ unsigned long long buf[WAVES][64];
    const int wave = WAVES == 1 ? 0 : threadIdx.x >> 6, lane = threadIdx.x & 63;
    const long long row = WAVES == 1 ? (long long)blockIdx.x * (LP_BLOCK / 64) + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= d.rows) return;                  // (WAVES = 1 alone: no barrier below there)
    unsigned long long list = 0;
    LpSums r = {LP_LOWEST, 0.0f, 0.0f};
    if (wave == 0)
        for (int s = lane; s < d.splits; s += 64) {
            const float4 p = d.part[row * d.splits + s];
            lp_join(r, LpSums{p.x, p.y, p.z});
        }
    if (d.k) {
        for (int s = wave; s < d.splits; s += WAVES)
            list = lp_merge(list, lane < d.k ? d.part_keys[(row * d.splits + s) * d.k + lane] : 0ull);
        for (int half = WAVES / 2; half > 0; half >>= 1) {
            if (wave >= half && wave < 2 * half) buf[wave][lane] = list;
            __syncthreads();
            if (wave < half) list = lp_merge(list, buf[wave + half][lane]);
        }
    }
    if (wave == 0) lp_write_row<T>(d, row, lp_wave_join(r), list);
}

// ---------------------------------------------------------------------------------- backward over rows
// One entry's gradient without what was gathered there.
__device__ __forceinline__ float lp_grad(float x, float m, float log_s, float G, float gh, float H)
{
    const float lp = x - m - log_s, p = lp_exp(lp);
    return -p * (G + gh * (fmaxf(lp, LP_FLOOR) + H));
}

// GROUP threads take a segment of a row (GROUP = 64: the whole row).  The backward kernels walk from the last row to the
// first: what forward read last is what the 256 MB cache still has (6 x 20 x 512 x 1024 fp32, forward and backward: 210 -> 203 us).
// STREAM: the gradient is written past the caches (LP_STREAM in train_ops.hip).
template <typename T, int GROUP, bool STREAM>
__global__ __launch_bounds__(LP_BLOCK) void lp_rows_bwd_kernel(const LpDesc d)
{
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 63;
    const unsigned block = gridDim.x - 1 - blockIdx.x;
    long long row;
    int me, from = 0, to = d.V;
    if (GROUP == 64) {
        row = (long long)block * 4 + (threadIdx.x >> 6);
        me = lane;
    } else {
        row = block / d.splits;
        me = threadIdx.x;
        from = (int)(block - row * d.splits) * d.seg;
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
            st16<STREAM>(dx + c, v, to - c);
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

// Many short rows: a block takes LP_SHORT_ROWS of them as one run of elements, so that all lanes work whatever V is, with
// what a row's entries need of it in shared memory.
#define LP_SHORT_ROWS 64
template <typename T>
__global__ __launch_bounds__(LP_BLOCK) void lp_short_rows_bwd_kernel(const LpDesc d)
{
    __shared__ float m[LP_SHORT_ROWS], log_s[LP_SHORT_ROWS], G[LP_SHORT_ROWS], gh[LP_SHORT_ROWS], H[LP_SHORT_ROWS], glp[LP_SHORT_ROWS];
    __shared__ int target[LP_SHORT_ROWS];
    const long long row0 = (long long)(gridDim.x - 1 - blockIdx.x) * LP_SHORT_ROWS;
    const int rows = d.rows - row0 < LP_SHORT_ROWS ? (int)(d.rows - row0) : LP_SHORT_ROWS, V = d.V, k = d.g_top ? d.k : 0;
    // four threads add up a row's upstream gradients
    const int mine = threadIdx.x >> 2, part = threadIdx.x & 3;
    {
        float g = 0.0f;
        if (mine < rows)
            for (int j = part; j < k; j += 4) g += d.g_top[(row0 + mine) * d.k + j];
        g = wave_sum(g, 4);
        if (mine < rows && part == 0) {
            const long long row = row0 + mine;
            const float2 st = d.stats[row];
            long long t = d.target[row];
            if (t == d.ignore || t < 0 || t >= V) t = -1;
            const float a = t >= 0 && d.g_lp ? d.g_lp[row] : 0.0f;
            m[mine] = st.x;
            log_s[mine] = st.y;
            G[mine] = g + a;
            gh[mine] = d.g_h ? d.g_h[row] : 0.0f;
            H[mine] = d.entropy[row];
            glp[mine] = a;
            target[mine] = (int)t;
        }
    }
    __syncthreads();
    const T *x = (const T *)d.x + row0 * d.ld;
    T *dx = (T *)d.dx + row0 * V;
    for (int e = threadIdx.x; e < rows * V; e += LP_BLOCK) {
        const int r = e / V, c = e - r * V;
        const float g = lp_grad(Vec16<T>::get(x + r * d.ld + c), m[r], log_s[r], G[r], gh[r], H[r]);
        Vec16<T>::put(dx + e, log_s[r] == -INFINITY ? 0.0f : c == target[r] ? g + glp[r] : g);
    }
    if (!k) return;
    // the alternatives' entries again, with what was gathered there (the target's among them has both)
    __syncthreads();
    for (int e = threadIdx.x; e < rows * k; e += LP_BLOCK) {
        const int r = e / k, j = e - r * k;
        if (log_s[r] == -INFINITY) continue;
        const long long at = (row0 + r) * d.k + j;
        const int c = (int)d.top_idx[at];
        if (c < 0 || c >= V) continue;          // (not one of forward's)
        const float g = lp_grad(Vec16<T>::get(x + r * d.ld + c), m[r], log_s[r], G[r], gh[r], H[r]) + d.g_top[at];
        Vec16<T>::put(dx + (long long)r * V + c, c == target[r] ? g + glp[r] : g);
    }
}

// ---------------------------------------------------------------------------------- pixels: [outer][V][inner]
// A thread takes one pixel and walks the classes; neighbouring threads take neighbouring pixels.  K >= k alternatives
// in registers.  Forward, short rows (inner = 1) are pixels too: a wave's loads then lie a row apart, but its 64 rows of a
// few classes stay in the first-level cache from one class to the next.
template <typename T, int K>
__global__ __launch_bounds__(LP_BLOCK) void lp_pixels_kernel(const LpDesc d)
{
    const long long p = (long long)blockIdx.x * LP_BLOCK + threadIdx.x;
    if (p >= d.rows) return;
    const long long n = p / d.inner, q = p - n * d.inner;
    const T *x = (const T *)d.x + n * d.group + q;
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
            v[i] = Vec16<T>::get(x + cc * d.next);
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
    if (d.stats) d.stats[p] = make_float2(r.m, log_s);
    d.entropy[p] = none ? 0.0f : log_s - r.a / r.s;
    const long long t = d.target[p];
    float lp = 0.0f;
    if (t != d.ignore && t >= 0 && t < d.V) lp = none ? -INFINITY : Vec16<T>::get(x + t * d.next) - r.m - log_s;
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

template <typename T, int K, bool STREAM>
__global__ __launch_bounds__(LP_BLOCK) void lp_pixels_bwd_kernel(const LpDesc d)
{
    const long long p = (long long)(gridDim.x - 1 - blockIdx.x) * LP_BLOCK + threadIdx.x;
    if (p >= d.rows) return;
    const long long n = p / d.inner, q = p - n * d.inner;
    const T *x = (const T *)d.x + n * d.group + q;
    T *dx = (T *)d.dx + n * d.V * d.inner + q;      // (dense, whatever the stride between rows of x)
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
        const T xi = STREAM ? __builtin_nontemporal_load(x + c * d.next) : x[c * d.next];
        float g = lp_grad(Vec16<T>::get(&xi), st.x, st.y, G, gh, H);
        if (c == (int)t) g += glp;
#pragma unroll
        for (int j = 0; j < K; ++j) g += idx[j] == c ? gt[j] : 0.0f;
        T gi;
        Vec16<T>::put(&gi, none ? 0.0f : g);
        if (STREAM) __builtin_nontemporal_store(gi, dx + (long long)c * d.inner);
        else dx[(long long)c * d.inner] = gi;
    }
}
