// liberfnet_hip.so — C ABI (include/erfnet_hip.h) over norm_kernels.h, logprob_kernels.h and adamw_kernels.h: layer norm,
// token log probabilities, AdamW.  A translation unit of its own; as in erfnet_hip.hip the host side builds descriptors and
// launches, and never allocates, copies or synchronises.
#include "../../include/erfnet_hip.h"
#include "host.h"
#include "adamw_kernels.h"
#include "logprob_kernels.h"
#include "norm_kernels.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

namespace {

#define fail host_fail
#define LAUNCHED(name)                                                                             \
    do {                                                                                           \
        if (host_launched(name)) return 1;                                                         \
    } while (0)

// HIP takes fewer than 2^32 threads in a launch: more work goes in several.
long long most_blocks(int threads) { return ((1ll << 32) - 1) / threads; }

int log2_up(int v)
{
    int b = 0;
    while ((1 << b) < v) ++b;
    return b;
}

// ================================================================================ layer norm
// A row of up to 16 elements a lane and 64 lanes stays inside a wave (no barrier, several short rows a wave);
// longer rows take a block of up to 1024 threads with 16 elements each.
struct NormPlan {
    bool wave;
    int rounds, lanes, threads;
};
template <typename T> NormPlan norm_plan(int C)
{
    const int vecs = (C + Vec16<T>::N - 1) / Vec16<T>::N, most = 16 / Vec16<T>::N;
    NormPlan p = {true, 1, 64, NORM_BLOCK};
    if (vecs <= 64 * most) {
        while (p.rounds * 64 < vecs) p.rounds *= 2;
        p.lanes = std::max(2, 1 << log2_up((vecs + p.rounds - 1) / p.rounds));      // (64 where rounds > 1)
        return p;
    }
    p.wave = false;
    p.rounds = most;
    p.threads = ((vecs + most - 1) / most + 63) / 64 * 64;
    return p;
}
template <int V> using Int = std::integral_constant<int, V>;
// launch(even, rounds, lanes) with the plan's values as compile-time constants; lanes = 0: a block per row
template <typename T, typename F> void norm_by_shape(const NormPlan &p, int C, F launch)
{
    auto with = [&](auto even) {
        constexpr int most = 16 / Vec16<T>::N;
        if (!p.wave) launch(even, Int<most>(), Int<0>());
        else if (p.rounds == most && most > 2) launch(even, Int<most>(), Int<64>());
        else if (p.rounds == 2) launch(even, Int<2>(), Int<64>());
        else if (p.lanes == 64) launch(even, Int<1>(), Int<64>());
        else if (p.lanes == 32) launch(even, Int<1>(), Int<32>());
        else if (p.lanes == 16) launch(even, Int<1>(), Int<16>());
        else if (p.lanes == 8) launch(even, Int<1>(), Int<8>());
        else if (p.lanes == 4) launch(even, Int<1>(), Int<4>());
        else launch(even, Int<1>(), Int<2>());
    };
    if (C % Vec16<T>::N == 0) with(std::true_type());
    else with(std::false_type());
}
// Blocks that walk over the rows, with `threads` threads on a compute unit in all.  Backward takes at least `turns` rows a
// thread beyond one block per unit, so that the blocks' partial sums stay a small part of its traffic.
int norm_blocks(const NormPlan &p, long long rows, int threads, int turns)
{
    const long long per = p.wave ? NORM_BLOCK / p.lanes : 1;
    const long long all = (rows + per - 1) / per, full = 256ll * std::max(1, threads / p.threads);
    return (int)std::min(std::min(all, full), std::max<long long>(256, all / turns));
}
// (us: forward with 2048 / 1024 threads a unit, 8191 x 8192 bf16 47 / 43, 49152 x 128 fp32 9.3 / 9.6; backward, a wave a row, 1024
// / 512, 20000 x 1000 fp32 54 / 50, 786432 x 16 bf16 20.6 / 19.2; a block a row, 1024 / 512 / 256, 8191 x 4096 bf16 67 / 51 / 47,
// 8191 x 8192 97 / 86 / 86, and 256 / 384, where 128 threads are three blocks instead of two and 192 two instead of one, 20000 x
// 1030 64 / 51, 20000 x 2049 102 / 81, 20000 x 2048 55 / 56)
#define NORM_FWD_BLOCKS(p, rows) norm_blocks(p, rows, 1024, 1)
#define NORM_BWD_BLOCKS(p, rows) norm_blocks(p, rows, (p).wave ? 512 : 384, 8)

// (partial sums of wide rows, us with 16 / 64 columns a block: C = 2048 12.6 / 11.8, 4096 11.9 / 8.1, 8192 13.3 / 7.3; 16 below,
// where 64 leave most compute units without a block)
#define NORM_SUM_WIDE 2048

int norm_check(const char *what, const void *x, const void *y, long long rows, int C, float eps)
{
    if (rows < 0) return fail("%s: negative row count", what);
    if (C < 1 || C > NORM_MAX_C) return fail("%s: 1..%d channels (got %d)", what, NORM_MAX_C, C);
    if (!(eps >= 0.0f)) return fail("%s: eps must not be negative", what);
    if (rows && (!x || !y)) return fail("%s: null pointer", what);
    return 0;
}

template <typename T>
int norm_forward(const void *x, const float *w, const float *b, void *y, float *mean, float *rstd, long long rows, int C,
                 float eps, hipStream_t st)
{
    if (norm_check("layer norm", x, y, rows, C, eps)) return 1;
    if (!mean != !rstd) return fail("layer norm: mean and rstd are kept together");
    if (rows == 0) return 0;
    const NormPlan p = norm_plan<T>(C);
    NormDesc d;
    memset(&d, 0, sizeof(d));
    d.x = x; d.y = y; d.w = w; d.b = b; d.mean = mean; d.rstd = rstd;
    d.rows = rows; d.safe_rows = rows - (Vec16<T>::N - 2 + C) / C; d.C = C; d.eps = eps;
    const int blocks = NORM_FWD_BLOCKS(p, rows);
    norm_by_shape<T>(p, C, [&](auto even, auto rounds, auto lanes) {
        norm_fwd_kernel<T, rounds, lanes, even><<<blocks, p.threads, 0, st>>>(d);
    });
    LAUNCHED("norm_fwd_kernel");
    return 0;
}

template <typename T> size_t norm_ws(long long rows, int C)
{
    const NormPlan p = norm_plan<T>(C);
    return (size_t)NORM_BWD_BLOCKS(p, rows) * 2 * C * sizeof(float);
}

template <typename T>
int norm_backward(const void *x, const float *w, const float *mean, const float *rstd, const void *gy, void *dx, float *dw,
                  float *db, long long rows, int C, void *ws, size_t ws_bytes, hipStream_t st)
{
    if (norm_check("layer norm backward", x, gy, rows, C, 0.0f)) return 1;
    const bool params = dw || db;
    if (rows && (!mean || !rstd)) return fail("layer norm backward: null pointer");
    if (!dx && !params) return 0;
    const NormPlan p = norm_plan<T>(C);
    const int blocks = NORM_BWD_BLOCKS(p, rows);
    NormDesc d;
    memset(&d, 0, sizeof(d));
    d.x = x; d.gy = gy; d.y = dx; d.w = w; d.mean = const_cast<float *>(mean); d.rstd = const_cast<float *>(rstd);
    d.rows = rows; d.safe_rows = rows - (Vec16<T>::N - 2 + C) / C; d.C = C;
    if (params) {
        if (blocks && (!ws || ws_bytes < norm_ws<T>(rows, C))) return fail("layer norm backward: workspace too small");
        d.partial = (float *)ws;
    }
    if (blocks) {
        const size_t lds = params && p.wave ? (size_t)8 * C * sizeof(float) : 0;
        norm_by_shape<T>(p, C, [&](auto even, auto rounds, auto lanes) {
            if constexpr (lanes > 0) norm_bwd_kernel<T, rounds, lanes, 0, even><<<blocks, NORM_BLOCK, lds, st>>>(d);
            else if (p.threads <= 512) norm_bwd_kernel<T, rounds, 0, 512, even><<<blocks, p.threads, 0, st>>>(d);
            else if constexpr (sizeof(T) == 2)
                norm_bwd_kernel<T, 2 * rounds, 0, 512, even><<<blocks, (p.threads / 2 + 63) / 64 * 64, 0, st>>>(d);
            else norm_bwd_kernel<T, rounds, 0, 1024, even><<<blocks, p.threads, 0, st>>>(d);
        });
        LAUNCHED("norm_bwd_kernel");
    }
    if (params) {
        // (no rows: zeros)
        if (C >= NORM_SUM_WIDE) norm_grad_sum_kernel<64><<<(2 * C + 63) / 64, 1024, 0, st>>>((const float *)ws, blocks, C, dw, db);
        else norm_grad_sum_kernel<16><<<(2 * C + 15) / 16, 1024, 0, st>>>((const float *)ws, blocks, C, dw, db);
        LAUNCHED("norm_grad_sum_kernel");
    }
    return 0;
}

// ================================================================================ token log probabilities
#define LP_MAX_CLASSES (1 << 30)
// Rows of up to LP_SHORT classes leave most of a wave idle, and where there are many of them that counts: forward from 64 rows
// a class on (us, a thread a row / a wave a row, fp32, top 2: 262144 x 20 10 / 249, 262144 x 100 75 / 247, 16384 x 100 16 / 20,
// 1024 x 100 15 / 5), backward from 256 (as one run of elements / a wave a row: 262144 x 20 13 / 81, 262144 x 100 42 / 85,
// 16384 x 64 7.4 / 6.7, 16384 x 200 20 / 8).
#define LP_SHORT 128
#define LP_SHORT_FORWARD 64ll
#define LP_SHORT_BACKWARD 256ll

// Forward: a thread takes a whole pixel, and a short row of many.
bool lp_by_thread(long long outer, int V, long long inner, int k)
{
    return inner > 1 || (V <= LP_SHORT && k <= ERF_LOG_PROBS_MAX_TOP_PIXELS && outer >= LP_SHORT_FORWARD * V);
}
// Forward: a wave takes a row of up to 32 KB, 16 KB where its lists are long (they are merged once a row by a wave, by four
// in a block), and of up to 4 KB where there are too few rows for the card; a block takes the others (us, a wave / a block
// a row, top 8 and 32: 8192 x 4096 bf16 25 / 41 and 28 / 42, 8192 x 8192 39 / 50 and 45 / 51, 8192 x 16384 62 / 68 and 81 / 68, 4096 x 24001
// 46 / 51 and 63 / 54; fp32 8192 x 8192 57 / 53 and 76 / 60; 512 x 6001 bf16 10.4 / 10.0 and 13.6 / 10.3).
// Backward, which has no results to join: a wave of up to 1024 classes (8192 x 1000 bf16: 8.0 and 11.6 us, 8192 x 4000: 23.1 and
// 21.8).
#define LP_WAVE_BACKWARD 1024
#define LP_BACKWARD_SEGMENT 8192

// Backward: a gradient of 48 MB or more is written past the caches, so that the logits stay in the 256 MB one until they are
// read again (pixels: that reading is their last, and goes past them too).  Forward and backward / the same with a reader of
// the gradient behind them, us, ordinary and streamed: rows of 100003 bf16, 30 MB 24.7 / 35.2 and 25.0 / 38.9, 61 MB 43.1 / 64.0
// and 41.2 / 64.2, 195 MB 123 / 187 and 109 / 179, 390 MB 236 / 363 and 212 / 356; 20 classes of fp32 pixels, 40 MB 29.6 / 43.2
// and 30.0 / 44.3, 60 MB 45.8 / 67.6 and 43.2 / 63.8, 240 MB 185 / 267 and 178 / 258.
#define LP_STREAM (48ll << 20)
template <typename F> void lp_streamed(bool stream, F launch)
{
    if (stream) launch(std::true_type());
    else launch(std::false_type());
}

// Forward: where there are few long rows, each takes several blocks of at least 4096 classes, until there are 512, and the
// join's launch after them (us, top 8, one block / 512 in all: 8 x 100003 bf16 17.9 / 12.7, 64 x 131072 21 / 17, 256 x 131072 22 / 23, 8 x 50000 12.7 /
// 12.1; more of them cost more than they bring: 1024 x 50003, 1 / 4 a row 28 / 45, 2047 x 100003 87 / 96).
#define LP_FEW_ROWS 128
#define LP_LONG_ROW 65536
struct LpPlan {
    bool wave;
    int splits, seg;
};
template <typename T> LpPlan lp_plan(long long rows, int V, int k)
{
    const long long most = rows < 1024 ? 4096 : k > 16 ? 16384 : 32768;
    LpPlan p = {V * (long long)sizeof(T) <= most, 1, V};
    if (p.wave || rows > LP_FEW_ROWS || V < LP_LONG_ROW) return p;
    p.splits = (int)std::min<long long>(512 / std::max<long long>(rows, 1), (V + 4095) / 4096);
    p.seg = ((V + p.splits - 1) / p.splits + 4095) / 4096 * 4096;
    p.splits = (V + p.seg - 1) / p.seg;
    return p;
}
// (the same for both types: rows that are split are longer than a wave takes)
size_t lp_ws(long long outer, int V, long long inner, int k)
{
    if (lp_by_thread(outer, V, inner, k)) return 0;
    const LpPlan p = lp_plan<bf16_t>(outer, V, k);
    return p.splits > 1 ? (size_t)outer * p.splits * (sizeof(float4) + (size_t)k * 8) : 0;
}

// The images or rows of d from `from` on, `n` of them.
template <typename T> LpDesc lp_part(LpDesc d, long long from, long long n)
{
    const long long rows = from * d.inner, gathered = rows * d.k, group = d.inner > 1 ? d.V * d.inner : d.ld;
    auto move = [](auto *&p, long long by) { if (p) p += by; };
    d.x = (const T *)d.x + from * group;
    d.target += rows;
    move(d.log_prob, rows);
    move(d.entropy, rows);
    move(d.stats, rows);
    move(d.top_lp, gathered);
    move(d.top_idx, gathered);
    move(d.g_lp, rows);
    move(d.g_h, rows);
    move(d.g_top, gathered);
    if (d.dx) d.dx = (T *)d.dx + rows * d.V;
    d.rows = n * d.inner;
    return d;
}
// launch(part) over `outer` images or rows, at most `most` of them at a time; backward comes to the last first, as its kernels do.
template <typename T, typename F>
int lp_launch(const char *kernel, const LpDesc &d, long long outer, long long most, bool backward, F launch)
{
    for (long long done = 0; done < outer; done += most) {
        const long long n = std::min(most, outer - done);
        launch(lp_part<T>(d, backward ? outer - done - n : done, n));
        LAUNCHED(kernel);
    }
    return 0;
}
#define LP_MOST_PIXELS (most_blocks(LP_BLOCK) * LP_BLOCK)

int lp_check(const char *what, long long outer, int V, long long inner, int k)
{
    if (outer < 0 || inner < 1) return fail("%s: negative or empty extent", what);
    if (V < 1 || V > LP_MAX_CLASSES) return fail("%s: 1..%d classes (got %d)", what, LP_MAX_CLASSES, V);
    const int most = inner > 1 ? ERF_LOG_PROBS_MAX_TOP_PIXELS : ERF_LOG_PROBS_MAX_TOP;
    if (k < 0 || k > most || k > V) return fail("%s: top_k must be in 0..%d and at most the class count (got %d)", what, most, k);
    if (outer > (1ll << 39) / inner) return fail("%s: too many rows", what);
    if (inner > LP_MOST_PIXELS) return fail("%s: more than %lld pixels an image", what, LP_MOST_PIXELS);
    return 0;
}

template <typename T>
int lp_forward(const void *x, const long long *target, float *log_prob, float *entropy, float *stats, float *top_lp,
               long long *top_idx, long long outer, int V, long long inner, long long ld, int k, long long ignore, void *ws,
               size_t ws_bytes, hipStream_t st)
{
    if (lp_check("log_probs", outer, V, inner, k)) return 1;
    if (outer == 0) return 0;
    if (!x || !target || !log_prob || !entropy || (k && (!top_lp || !top_idx))) return fail("log_probs: null pointer");
    if (inner == 1 && ld < V && outer > 1) return fail("log_probs: rows overlap (stride %lld, %d classes)", ld, V);
    LpDesc d;
    memset(&d, 0, sizeof(d));
    d.x = x; d.target = target; d.log_prob = log_prob; d.entropy = entropy; d.stats = (float2 *)stats;
    d.top_lp = top_lp; d.top_idx = top_idx; d.rows = outer * inner; d.ld = ld; d.inner = inner; d.ignore = ignore;
    d.V = V; d.k = k;
    if (lp_by_thread(outer, V, inner, k)) {
        d.group = inner > 1 ? V * inner : ld;
        d.next = inner;
        return lp_launch<T>("lp_pixels_kernel", d, outer, LP_MOST_PIXELS / inner, false, [&](const LpDesc &d) {
            const unsigned blocks = (unsigned)((d.rows + LP_BLOCK - 1) / LP_BLOCK);
            if (k == 0) lp_pixels_kernel<T, 0><<<blocks, LP_BLOCK, 0, st>>>(d);
            else if (k == 1) lp_pixels_kernel<T, 1><<<blocks, LP_BLOCK, 0, st>>>(d);
            else if (k == 2) lp_pixels_kernel<T, 2><<<blocks, LP_BLOCK, 0, st>>>(d);
            else if (k <= 4) lp_pixels_kernel<T, 4><<<blocks, LP_BLOCK, 0, st>>>(d);
            else lp_pixels_kernel<T, 8><<<blocks, LP_BLOCK, 0, st>>>(d);
        });
    }
    const LpPlan p = lp_plan<T>(outer, V, k);
    d.splits = p.splits; d.seg = p.seg;
    if (p.splits > 1) {
        if (!ws || ws_bytes < lp_ws(outer, V, inner, k)) return fail("log_probs: workspace too small");
        d.part = (float4 *)ws;
        d.part_keys = (unsigned long long *)((char *)ws + (size_t)outer * p.splits * sizeof(float4));
    }
    // (a row that is split is one of few: they go in one launch, and so does their join)
    const long long most = p.wave ? most_blocks(LP_BLOCK) * 4 : most_blocks(LP_BLOCK) / p.splits;
    const int rc = lp_launch<T>("lp_rows_kernel", d, outer, most, false, [&](const LpDesc &d) {
        if (p.wave) {
            const unsigned blocks = (unsigned)((d.rows + 3) / 4);
            if (k) lp_rows_kernel<T, 64, true><<<blocks, LP_BLOCK, 0, st>>>(d);
            else lp_rows_kernel<T, 64, false><<<blocks, LP_BLOCK, 0, st>>>(d);
        } else {
            const unsigned blocks = (unsigned)(d.rows * p.splits);
            if (k) lp_rows_kernel<T, 256, true><<<blocks, LP_BLOCK, 0, st>>>(d);
            else lp_rows_kernel<T, 256, false><<<blocks, LP_BLOCK, 0, st>>>(d);
        }
    });
    if (rc) return rc;
    if (p.splits > 1) {
        if (p.splits <= 8) lp_join_kernel<T, 1><<<(unsigned)((outer + 3) / 4), LP_BLOCK, 0, st>>>(d);
        else lp_join_kernel<T, 16><<<(unsigned)outer, 1024, 0, st>>>(d);
        LAUNCHED("lp_join_kernel");
    }
    return 0;
}

template <typename T>
int lp_backward(const void *x, const long long *target, const float *entropy, const float *stats, const long long *top_idx,
                const float *g_lp, const float *g_h, const float *g_top, void *dx, long long outer, int V, long long inner,
                long long ld, int k, long long ignore, hipStream_t st)
{
    if (lp_check("log_probs backward", outer, V, inner, k)) return 1;
    if (outer == 0) return 0;
    if (!x || !target || !entropy || !stats || !dx || (k && !top_idx)) return fail("log_probs backward: null pointer");
    LpDesc d;
    memset(&d, 0, sizeof(d));
    d.x = x; d.target = target; d.entropy = const_cast<float *>(entropy); d.stats = (float2 *)const_cast<float *>(stats);
    d.top_idx = const_cast<long long *>(top_idx); d.g_lp = g_lp; d.g_h = g_h; d.g_top = g_top; d.dx = dx;
    d.rows = outer * inner; d.ld = ld; d.inner = inner; d.ignore = ignore; d.V = V; d.k = k;
    const bool stream = d.rows * V * (long long)sizeof(T) >= LP_STREAM;
    if (inner > 1) {
        d.group = V * inner;
        d.next = inner;
        return lp_launch<T>("lp_pixels_bwd_kernel", d, outer, LP_MOST_PIXELS / inner, true, [&](const LpDesc &d) {
            const unsigned blocks = (unsigned)((d.rows + LP_BLOCK - 1) / LP_BLOCK);
            lp_streamed(stream, [&](auto stream) {
                if (!g_top || k == 0) lp_pixels_bwd_kernel<T, 0, stream><<<blocks, LP_BLOCK, 0, st>>>(d);
                else if (k <= 2) lp_pixels_bwd_kernel<T, 2, stream><<<blocks, LP_BLOCK, 0, st>>>(d);
                else lp_pixels_bwd_kernel<T, 8, stream><<<blocks, LP_BLOCK, 0, st>>>(d);
            });
        });
    }
    const bool by_elements = V <= LP_SHORT && outer >= LP_SHORT_BACKWARD * V, wave = V <= LP_WAVE_BACKWARD;
    d.seg = LP_BACKWARD_SEGMENT;
    d.splits = (V + d.seg - 1) / d.seg;
    const long long most = by_elements ? most_blocks(LP_BLOCK) * LP_SHORT_ROWS
                                       : wave ? most_blocks(LP_BLOCK) * 4 : most_blocks(LP_BLOCK) / d.splits;
    return lp_launch<T>("lp_rows_bwd_kernel", d, outer, most, true, [&](const LpDesc &d) {
        if (by_elements) {
            lp_short_rows_bwd_kernel<T><<<(unsigned)((d.rows + LP_SHORT_ROWS - 1) / LP_SHORT_ROWS), LP_BLOCK, 0, st>>>(d);
            return;
        }
        lp_streamed(stream, [&](auto stream) {
            if (wave) lp_rows_bwd_kernel<T, 64, stream><<<(unsigned)((d.rows + 3) / 4), LP_BLOCK, 0, st>>>(d);
            else lp_rows_bwd_kernel<T, 256, stream><<<(unsigned)(d.rows * d.splits), LP_BLOCK, 0, st>>>(d);
        });
    });
}

// ================================================================================ AdamW
// Tensors (parameters, gradients, moments) of this many bytes in all are read past the caches, and their moments, which nobody
// reads before the next step, are written past them.  Ordinary and streamed, us: bf16 with fp32 moments, 256 MB: steps one
// behind the other 74 and 80, behind a 400 MB write and with a reader of the parameters 117 and 102; 320 MB 101 / 141 and 99 /
// 128; 400 MB 146 / 174 and 121 / 161; 720 MB 258 / 309 and 213 / 284.  fp32 with 8-bit ones, 320 MB 97 / 156 and 96 / 149, 720 MB 232 /
// 345 and 208 / 343.
#define ADAMW_STREAM (320ll << 20)
template <typename T, int BITS>
int adamw_step(const char *what, int count, void *const *p, const void *const *g, void *const *m, float *const *ms,
               void *const *v, float *const *vs, const long long *numel, double lr, double b1, double b2, double eps,
               double wd, long long step, hipStream_t st)
{
    if (count < 0) return fail("%s: negative tensor count", what);
    if (step < 1) return fail("%s: step counts from 1 (got %lld)", what, step);
    if (!(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0)) return fail("%s: betas outside [0, 1)", what);
    if (!(eps >= 0.0) || !(lr >= 0.0) || !(wd >= 0.0)) return fail("%s: negative lr / eps / weight decay", what);
    if (count && (!p || !g || !m || !v || !numel || (BITS == 8 && (!ms || !vs)))) return fail("%s: null pointer table", what);
    AdamwDesc<BITS> d;
    memset(&d, 0, sizeof(d));
    // the scalars in double, rounded once for the kernel
    d.k.b1 = (float)b1; d.k.ob1 = (float)(1.0 - b1); d.k.b2 = (float)b2; d.k.ob2 = (float)(1.0 - b2);
    d.k.keep = (float)(1.0 - lr * wd);
    d.k.step = (float)(lr / (1.0 - pow(b1, (double)step)));
    d.k.inv_root_c2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)step)));
    // The reciprocal takes a subnormal number for zero, and an element without a gradient so far has eps alone below its line:
    // the quotient is formed 2^24 fold above and below then (roots are under 2^64, so nothing overflows).
    const double least = 1.1754943508222875e-38, fold = eps > 0.0 && eps < least ? 16777216.0 : 1.0;
    d.k.eps = fold == 1.0 ? (float)eps : (float)std::max(eps * fold, least);
    d.k.inv_root_c2 *= (float)fold;
    d.k.step *= (float)fold;
    long long elements = 0;
    for (int i = 0; i < count; ++i) {
        if (numel[i] < 0) return fail("%s: tensor %d has a negative size", what, i);
        if (numel[i] >> 48) return fail("%s: tensor %d is too large", what, i);
        elements += numel[i];
        if (numel[i] && (!p[i] || !g[i] || !m[i] || !v[i] || (BITS == 8 && (!ms[i] || !vs[i]))))
            return fail("%s: tensor %d has a null pointer", what, i);
        for (const void *a : {(const void *)p[i], g[i], (const void *)m[i], (const void *)v[i], BITS == 8 ? (const void *)ms[i] : nullptr,
                              BITS == 8 ? (const void *)vs[i] : nullptr})
            if ((unsigned long long)a >> 48) return fail("%s: tensor %d has an address of more than 48 bits", what, i);
    }
    // a replayed launch would repeat this step's bias corrections
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    if (std::any_of(numel, numel + count, [](long long n) { return n > 0; }) &&
        (hipStreamIsCapturing(st, &capture) != hipSuccess || capture != hipStreamCaptureStatusNone)) {
        (void)hipGetLastError();
        return fail("%s: the step cannot be captured into a graph", what);
    }
    const bool stream = elements >= ADAMW_STREAM / (2 * (long long)sizeof(T) + (BITS == 8 ? 2 : 8));
    const long long most = most_blocks(ADAMW_BLOCK);
    int i = 0;
    long long done = 0;             // elements of tensor i that earlier launches have taken: whole chunks, and so whole scale blocks
    while (i < count) {
        d.count = 0;
        long long chunks = 0;
        while (i < count && d.count < AdamwDesc<BITS>::MAX && chunks < most) {
            const long long n = std::min(numel[i] - done, (most - chunks) * ADAMW_CHUNK);
            if (n) {
                const int k = d.count++;
                const long long c = (n + ADAMW_CHUNK - 1) / ADAMW_CHUNK;
                auto from = [](const void *p, long long bytes) { return (const char *)p + bytes; };
                d.set(ADAMW_P, k, from(p[i], done * (long long)sizeof(T)));
                d.set(ADAMW_G, k, from(g[i], done * (long long)sizeof(T)));
                d.set(ADAMW_M, k, from(m[i], BITS == 8 ? done : done * 4));
                d.set(ADAMW_V, k, from(v[i], BITS == 8 ? done : done * 4));
                if constexpr (BITS == 8) {
                    d.set(ADAMW_MS, k, from(ms[i], done / ADAMW_SCALE_BLOCK * 4));
                    d.set(ADAMW_VS, k, from(vs[i], done / ADAMW_SCALE_BLOCK * 4));
                }
                d.last[k] = (unsigned)(n - (c - 1) * ADAMW_CHUNK);
                chunks += c;
                d.end_chunk[k] = (unsigned)chunks;
                done += n;
            }
            if (done == numel[i]) {
                ++i;
                done = 0;
            }
        }
        if (d.count == 0) break;
        if (stream) adamw_kernel<T, BITS, true><<<(unsigned)chunks, ADAMW_BLOCK, 0, st>>>(d);
        else adamw_kernel<T, BITS, false><<<(unsigned)chunks, ADAMW_BLOCK, 0, st>>>(d);
        LAUNCHED("adamw_kernel");
    }
    return 0;
}

}  // namespace

extern "C" {

size_t erf_layer_norm_workspace_bytes(long long rows, int C)
{
    return rows < 0 || C < 1 || C > NORM_MAX_C ? 0 : std::max(norm_ws<float>(rows, C), norm_ws<bf16_t>(rows, C));
}
int erf_layer_norm_forward(const float *x, const float *w, const float *b, float *y, float *mean, float *rstd, long long rows,
                           int C, float eps, void *stream)
{
    return norm_forward<float>(x, w, b, y, mean, rstd, rows, C, eps, (hipStream_t)stream);
}
int erf_layer_norm_forward_bf16(const void *x, const float *w, const float *b, void *y, float *mean, float *rstd,
                                long long rows, int C, float eps, void *stream)
{
    return norm_forward<bf16_t>(x, w, b, y, mean, rstd, rows, C, eps, (hipStream_t)stream);
}
int erf_layer_norm_backward(const float *x, const float *w, const float *mean, const float *rstd, const float *gy, float *dx,
                            float *dw, float *db, long long rows, int C, void *ws, size_t ws_bytes, void *stream)
{
    return norm_backward<float>(x, w, mean, rstd, gy, dx, dw, db, rows, C, ws, ws_bytes, (hipStream_t)stream);
}
int erf_layer_norm_backward_bf16(const void *x, const float *w, const float *mean, const float *rstd, const void *gy,
                                 void *dx, float *dw, float *db, long long rows, int C, void *ws, size_t ws_bytes,
                                 void *stream)
{
    return norm_backward<bf16_t>(x, w, mean, rstd, gy, dx, dw, db, rows, C, ws, ws_bytes, (hipStream_t)stream);
}

size_t erf_log_probs_workspace_bytes(long long outer, int V, long long inner, int top_k)
{
    return outer < 1 || V < 1 || V > LP_MAX_CLASSES || inner < 1 || top_k < 0 || top_k > LP_MAX_TOP
               ? 0 : lp_ws(outer, V, inner, top_k);
}
int erf_log_probs_forward(const float *logits, const long long *target, float *log_prob, float *entropy, float *stats,
                          float *top_log_probs, long long *top_indices, long long outer, int V, long long inner,
                          long long row_stride, int top_k, long long ignore_index, void *ws, size_t ws_bytes, void *stream)
{
    return lp_forward<float>(logits, target, log_prob, entropy, stats, top_log_probs, top_indices, outer, V, inner, row_stride,
                             top_k, ignore_index, ws, ws_bytes, (hipStream_t)stream);
}
int erf_log_probs_forward_bf16(const void *logits, const long long *target, float *log_prob, float *entropy, float *stats,
                               float *top_log_probs, long long *top_indices, long long outer, int V, long long inner,
                               long long row_stride, int top_k, long long ignore_index, void *ws, size_t ws_bytes,
                               void *stream)
{
    return lp_forward<bf16_t>(logits, target, log_prob, entropy, stats, top_log_probs, top_indices, outer, V, inner,
                              row_stride, top_k, ignore_index, ws, ws_bytes, (hipStream_t)stream);
}
int erf_log_probs_backward(const float *logits, const long long *target, const float *entropy, const float *stats,
                           const long long *top_indices, const float *g_log_prob, const float *g_entropy,
                           const float *g_top, float *dlogits, long long outer, int V, long long inner,
                           long long row_stride, int top_k, long long ignore_index, void *stream)
{
    return lp_backward<float>(logits, target, entropy, stats, top_indices, g_log_prob, g_entropy, g_top, dlogits, outer, V,
                              inner, row_stride, top_k, ignore_index, (hipStream_t)stream);
}
int erf_log_probs_backward_bf16(const void *logits, const long long *target, const float *entropy, const float *stats,
                                const long long *top_indices, const float *g_log_prob, const float *g_entropy,
                                const float *g_top, void *dlogits, long long outer, int V, long long inner,
                                long long row_stride, int top_k, long long ignore_index, void *stream)
{
    return lp_backward<bf16_t>(logits, target, entropy, stats, top_indices, g_log_prob, g_entropy, g_top, dlogits, outer, V,
                               inner, row_stride, top_k, ignore_index, (hipStream_t)stream);
}

int erf_adamw_step(int count, float *const *params, const float *const *grads, float *const *exp_avg,
                   float *const *exp_avg_sq, const long long *numel, double lr, double beta1, double beta2, double eps,
                   double weight_decay, long long step, void *stream)
{
    return adamw_step<float, 32>("adamw", count, (void *const *)params, (const void *const *)grads, (void *const *)exp_avg,
                                 nullptr, (void *const *)exp_avg_sq, nullptr, numel, lr, beta1, beta2, eps, weight_decay, step,
                                 (hipStream_t)stream);
}
int erf_adamw_step_bf16(int count, void *const *params, const void *const *grads, float *const *exp_avg,
                        float *const *exp_avg_sq, const long long *numel, double lr, double beta1, double beta2,
                        double eps, double weight_decay, long long step, void *stream)
{
    return adamw_step<bf16_t, 32>("adamw", count, params, grads, (void *const *)exp_avg, nullptr, (void *const *)exp_avg_sq,
                                  nullptr, numel, lr, beta1, beta2, eps, weight_decay, step, (hipStream_t)stream);
}
int erf_adamw8_step(int count, float *const *params, const float *const *grads, void *const *exp_avg,
                    float *const *exp_avg_scale, void *const *exp_avg_sq_root, float *const *exp_avg_sq_root_scale,
                    const long long *numel, double lr, double beta1, double beta2, double eps, double weight_decay,
                    long long step, void *stream)
{
    return adamw_step<float, 8>("adamw8", count, (void *const *)params, (const void *const *)grads, exp_avg, exp_avg_scale,
                                exp_avg_sq_root, exp_avg_sq_root_scale, numel, lr, beta1, beta2, eps, weight_decay, step,
                                (hipStream_t)stream);
}
int erf_adamw8_step_bf16(int count, void *const *params, const void *const *grads, void *const *exp_avg,
                         float *const *exp_avg_scale, void *const *exp_avg_sq_root, float *const *exp_avg_sq_root_scale,
                         const long long *numel, double lr, double beta1, double beta2, double eps, double weight_decay,
                         long long step, void *stream)
{
    return adamw_step<bf16_t, 8>("adamw8", count, params, grads, exp_avg, exp_avg_scale, exp_avg_sq_root,
                                 exp_avg_sq_root_scale, numel, lr, beta1, beta2, eps, weight_decay, step, (hipStream_t)stream);
}

}  // extern "C"
