// AdamW (decoupled weight decay) over many tensors at once:
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p (1 - lr wd) - (lr / c1) m / (sqrt(v) / sqrt(c2) + eps),
//   c1 = 1 - b1^t, c2 = 1 - b2^t.
// Parameters and gradients fp32 or bf16 (widened, rounded once on the way back), arithmetic fp32.
//
// BITS = 32 holds m and v in fp32.  BITS = 8 holds m and r = sqrt(v) as float8 (e4m3: 4 significant bits, largest 448) with
// one fp32 scale, the block's largest magnitude / 448, for each 256 consecutive elements of a tensor.  The root halves v's
// range in the exponent, so the 2^17 that e4m3 spans cover 2^35 of v, and it is what the denominator needs.  A root
// that is not zero is never stored as zero: an element whose moment outlives its rounded-off denominator would
// otherwise move by lr m / eps.  The scale is the largest magnitude itself, not a power of two above it: v
// moves by 1 - b2 a step, far below half a code, and only through the scale do the codes follow such small moves.
// NaN and infinity are stored as NaN in their own element and left out of the block's scale.
//
// Bound by memory: 28 / 22 bytes an element (fp32 / bf16 parameters) with 32-bit moments, 16 / 10 with 8-bit ones.
// A wave takes 256 consecutive elements at a time, four a lane: one 16-byte access of fp32, and exactly one scale.
#pragma once
#include "vec16.h"
#include "wave.h"

// (two rounds a wave: 4 take 105 registers with 8-bit moments and leave 4 waves a SIMD; bf16, 64 / 512 MB 24.0 / 146 us, 22.9 /
// 138 with 2; with fp32 moments within 2 %)
#define ADAMW_BLOCK 256
#define ADAMW_SCALE_BLOCK 256
#define ADAMW_ROUNDS 2
#define ADAMW_CHUNK (ADAMW_BLOCK * 4 * ADAMW_ROUNDS)
#define ADAMW_TINY 7.8886090522101181e-31f      // 2^-100: 448 / x stays finite above it; blocks below are stored as zeros

struct AdamwScalars {
    float b1, ob1, b2, ob2, keep, step, inv_root_c2, eps;       // ob = 1 - b, keep = 1 - lr wd, step = lr / c1
};
// One launch's tensors, as many as 4 KB of kernel arguments hold: 126 with 32-bit moments and 92 with 8-bit ones, by the 48 bits
// that an address has (whole pointers and sizes: 90 and 66, and the 229 tensors of a network take a launch more).
enum { ADAMW_P, ADAMW_G, ADAMW_M, ADAMW_V, ADAMW_MS, ADAMW_VS };        // 8 bits: codes of m and of the root, their scales
template <int BITS> struct AdamwDesc {
    static constexpr int POINTERS = BITS == 8 ? 6 : 4, MAX = BITS == 8 ? 92 : 126;
    AdamwScalars k;
    int count;
    unsigned end_chunk[MAX];    // running total of chunks up to and including tensor i
    unsigned last[MAX];         // elements in its last chunk
    unsigned low[POINTERS][MAX], high[POINTERS / 2][MAX];       // high: two pointers' upper 16 bits
    void set(int which, int i, const void *p)
    {
        const unsigned long long a = (unsigned long long)p;
        unsigned &h = high[which / 2][i];
        low[which][i] = (unsigned)a;
        h = which & 1 ? (h & 0xffffu) | (unsigned)(a >> 32) << 16 : (h & 0xffff0000u) | (unsigned)(a >> 32);
    }
    // (by way of global memory's own pointers, or every access would be a flat one)
    __device__ __forceinline__ char *get(int which, int t) const
    {
        const unsigned h = which & 1 ? high[which / 2][t] >> 16 : high[which / 2][t] & 0xffffu;
        return (char *)(__attribute__((address_space(1))) char *)((unsigned long long)h << 32 | low[which][t]);
    }
};
static_assert(sizeof(AdamwDesc<32>) <= 4096 && sizeof(AdamwDesc<8>) <= 4096, "kernel arguments");

// sqrt to one unit in the last place: the instruction has that, but takes subnormal numbers for zero.
__device__ __forceinline__ float adamw_root(float v)
{
    const bool small = v < 1.2621774483536189e-29f;             // 2^-96
    const float r = __builtin_amdgcn_sqrtf(v * (small ? 4294967296.0f : 1.0f));
    return r * (small ? 1.52587890625e-05f : 1.0f);             // 2^32, 2^-16
}
// b1 m + (1 - b1) g, each product rounded: a fused product would be nearer by half a unit, but a moment on the border between
// two 8-bit codes would then fall to another one than in an update written with torch's operations, and a block whose largest
// moment does so has another scale one step later (one block of 1.5 million; none with the same roundings here and in encode).
__device__ __forceinline__ float adamw_mean(const AdamwScalars &d, float m, float g)
{
#pragma clang fp contract(off)
    const float a = d.b1 * m, b = d.ob1 * g;
    return a + b;
}
// The quotient is a product with a reciprocal to one unit in the last place.  (With exact roots and quotients and a
// maximum of its own for every scale the 8-bit step took 85 vector instructions an element, and those bound it: bf16
// parameters, 720 MB, 325 us, 198 so; fp32 232 and 180; with fp32 moments memory binds either way.)
__device__ __forceinline__ float adamw_update(const AdamwScalars &d, float p, float g, float &m, float &v, float &root)
{
    m = adamw_mean(d, m, g);
    v = d.b2 * v + d.ob2 * (g * g);
    root = adamw_root(v);
    return p * d.keep - d.step * m * __builtin_amdgcn_rcpf(root * d.inv_root_c2 + d.eps);
}

// four consecutive elements, the first `left` of them there
template <typename T> struct AdamwQuad;
template <> struct AdamwQuad<float> {
    struct __attribute__((packed, aligned(4))) Raw { f32x4 v; };
    template <bool STREAM> static __device__ __forceinline__ f32x4 load(const void *p, long long i, int left)
    {
        f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
        const float *q = (const float *)p + i;
        if (left >= 4) r = ld_vec<STREAM>(reinterpret_cast<const Raw *>(q));
        else
            for (int j = 0; j < 3; ++j) if (j < left) r[j] = q[j];
        return r;
    }
    template <bool STREAM> static __device__ __forceinline__ void store(void *p, long long i, int left, f32x4 r)
    {
        float *q = (float *)p + i;
        if (left >= 4) st_vec<STREAM>(reinterpret_cast<Raw *>(q), r);
        else
            for (int j = 0; j < 3; ++j) if (j < left) q[j] = r[j];
    }
};
template <> struct AdamwQuad<bf16_t> {
    struct __attribute__((packed, aligned(2))) Raw { u32x2 v; };
    template <bool STREAM> static __device__ __forceinline__ f32x4 load(const void *p, long long i, int left)
    {
        f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
        const bf16_t *q = (const bf16_t *)p + i;
        if (left >= 4) r = unpack_bf16x4(ld_vec<STREAM>(reinterpret_cast<const Raw *>(q)));
        else
            for (int j = 0; j < 3; ++j) if (j < left) r[j] = bf16_to_f32(q[j]);
        return r;
    }
    template <bool STREAM> static __device__ __forceinline__ void store(void *p, long long i, int left, f32x4 r)
    {
        bf16_t *q = (bf16_t *)p + i;
        if (left >= 4) st_vec<STREAM>(reinterpret_cast<Raw *>(q), pack_bf16x4(r));
        else
            for (int j = 0; j < 3; ++j) if (j < left) q[j] = f32_to_bf16(r[j]);
    }
};
struct AdamwCodes {
    struct __attribute__((packed, aligned(1))) Raw { unsigned v; };
    template <bool STREAM> static __device__ __forceinline__ unsigned load(const void *p, long long i, int left)
    {
        const unsigned char *q = (const unsigned char *)p + i;
        unsigned r = 0;
        if (left >= 4) r = ld_vec<STREAM>(reinterpret_cast<const Raw *>(q));
        else
            for (int j = 0; j < 3; ++j) if (j < left) r |= (unsigned)q[j] << (8 * j);
        return r;
    }
    template <bool STREAM> static __device__ __forceinline__ void store(void *p, long long i, int left, unsigned r)
    {
        unsigned char *q = (unsigned char *)p + i;
        if (left >= 4) st_vec<STREAM>(reinterpret_cast<Raw *>(q), r);
        else
            for (int j = 0; j < 3; ++j) if (j < left) q[j] = (unsigned char)(r >> (8 * j));
    }
    static __device__ __forceinline__ f32x4 decode(unsigned r, float scale)
    {
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)r, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)r, true);
        return (f32x4){a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale};
    }
    // As bits, magnitudes have the order of the values, infinity and NaN above them all: one maximum finds the scale and
    // says whether there are any, one minimum whether a root would round to zero; only then a wave goes element by element.
    static constexpr unsigned INF = 0x7f800000u;
    static __device__ __forceinline__ unsigned bits(float x) { return __builtin_bit_cast(unsigned, x) & 0x7fffffffu; }
    static __device__ __forceinline__ unsigned most(f32x4 x, unsigned below = ~0u)      // of this lane's, below `below`
    {
        unsigned top = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = bits(x[j]) > top && bits(x[j]) < below ? bits(x[j]) : top;
        return top;
    }
    // codes of x, whose largest magnitude over the wave is `top` (all 64 lanes take part); ROOT: x >= 0 and nonzero stays nonzero
    template <bool ROOT> static __device__ __forceinline__ unsigned encode(f32x4 x, unsigned top, float &scale)
    {
        const bool odd = top >= INF;
        if (odd) top = __builtin_bit_cast(unsigned, wave_max(__builtin_bit_cast(float, most(x, INF))));
        const float high = __builtin_bit_cast(float, top);
        const bool some = high >= ADAMW_TINY;
        scale = some ? high * (1.0f / 448.0f) : 0.0f;
        // 448 (1 / high), as torch divides; the reciprocal, of high / 4 because that is never subnormal, with its remainder
        // added back
        const float q = 0.25f * high, r0 = __builtin_amdgcn_rcpf(q);
        const float inv = some ? 112.0f * __builtin_fmaf(__builtin_fmaf(-q, r0, 1.0f), r0, r0) : 0.0f;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = x[j] * inv;
        if (ROOT) {
            constexpr float code = 0.001953125f;                // 2^-9, the least above zero
            if (some && __any(fminf(fminf(y[0], y[1]), fminf(y[2], y[3])) < code)) {
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = bits(x[j]) ? fmaxf(y[j], code) : 0.0f;
            }
        }
        if (odd) {
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = bits(x[j]) >= INF ? __builtin_nanf("") : y[j];
        }
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
        return (unsigned)r;
    }
};

// A wave's `ADAMW_ROUNDS` blocks of 256 elements, the first at `base`, blocks ADAMW_BLOCK * 4 elements apart; all loads go
// out before the first result is needed.  FULL: every element is there.  STREAM: reads, and the moments' writes, past the caches
// (ADAMW_STREAM in train_ops.hip).
template <typename T, int BITS, bool FULL, bool STREAM>
__device__ __forceinline__ void adamw_chunk(const AdamwDesc<BITS> &d, int t, long long n, long long base)
{
    char *const pp = d.get(ADAMW_P, t), *const pm = d.get(ADAMW_M, t), *const pv = d.get(ADAMW_V, t);
    const char *const pg = d.get(ADAMW_G, t);
    float *pms = nullptr, *pvs = nullptr;
    if constexpr (BITS == 8) {
        pms = (float *)d.get(ADAMW_MS, t);
        pvs = (float *)d.get(ADAMW_VS, t);
    }
    const int lane = threadIdx.x & 63;
    f32x4 p[ADAMW_ROUNDS], g[ADAMW_ROUNDS], m[ADAMW_ROUNDS], v[ADAMW_ROUNDS];
    unsigned cm[ADAMW_ROUNDS], cr[ADAMW_ROUNDS];
    float ms[ADAMW_ROUNDS], rs[ADAMW_ROUNDS];
#pragma unroll
    for (int r = 0; r < ADAMW_ROUNDS; ++r) {
        const long long at = base + (long long)r * ADAMW_BLOCK * 4, i = at + lane * 4;
        const int left = FULL ? 4 : n - i >= 4 ? 4 : n - i > 0 ? (int)(n - i) : 0;
        p[r] = AdamwQuad<T>::template load<STREAM>(pp, i, left);
        g[r] = AdamwQuad<T>::template load<STREAM>(pg, i, left);
        if constexpr (BITS == 32) {
            m[r] = AdamwQuad<float>::load<STREAM>(pm, i, left);
            v[r] = AdamwQuad<float>::load<STREAM>(pv, i, left);
        } else {
            cm[r] = AdamwCodes::load<STREAM>(pm, i, left);
            cr[r] = AdamwCodes::load<STREAM>(pv, i, left);
            const bool there = FULL || at < n;
            ms[r] = there ? pms[at / ADAMW_SCALE_BLOCK] : 0.0f;
            rs[r] = there ? pvs[at / ADAMW_SCALE_BLOCK] : 0.0f;
            m[r] = v[r] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};      // (what a block behind the last one counts for below)
        }
    }
#pragma unroll
    for (int r = 0; r < ADAMW_ROUNDS; ++r) {
        const long long at = base + (long long)r * ADAMW_BLOCK * 4, i = at + lane * 4;
        const int left = FULL ? 4 : n - i >= 4 ? 4 : n - i > 0 ? (int)(n - i) : 0;
        if (!FULL && at >= n) break;            // (uniform over the wave)
        if constexpr (BITS == 8) {
            m[r] = AdamwCodes::decode(cm[r], ms[r]);
            v[r] = AdamwCodes::decode(cr[r], rs[r]);
            v[r] *= v[r];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float mj = m[r][j], vj = v[r][j], root;
            p[r][j] = adamw_update(d.k, p[r][j], g[r][j], mj, vj, root);
            m[r][j] = mj;
            v[r][j] = BITS == 8 ? root : vj;
        }
        AdamwQuad<T>::template store<false>(pp, i, left, p[r]);
        if constexpr (BITS == 32) {
            AdamwQuad<float>::store<STREAM>(pm, i, left, m[r]);
            AdamwQuad<float>::store<STREAM>(pv, i, left, v[r]);
        }
    }
    if constexpr (BITS == 8) {
        unsigned top[2 * ADAMW_ROUNDS];
#pragma unroll
        for (int r = 0; r < ADAMW_ROUNDS; ++r) {
            top[2 * r] = AdamwCodes::most(m[r]);
            top[2 * r + 1] = AdamwCodes::most(v[r]);
        }
        wave_max_all(top);
#pragma unroll
        for (int r = 0; r < ADAMW_ROUNDS; ++r) {
            const long long at = base + (long long)r * ADAMW_BLOCK * 4, i = at + lane * 4;
            const int left = FULL ? 4 : n - i >= 4 ? 4 : n - i > 0 ? (int)(n - i) : 0;
            if (!FULL && at >= n) break;
            float sm, sr;
            const unsigned nm = AdamwCodes::encode<false>(m[r], top[2 * r], sm), nr = AdamwCodes::encode<true>(v[r], top[2 * r + 1], sr);
            AdamwCodes::store<STREAM>(pm, i, left, nm);
            AdamwCodes::store<STREAM>(pv, i, left, nr);
            if (lane == 0) { pms[at / ADAMW_SCALE_BLOCK] = sm; pvs[at / ADAMW_SCALE_BLOCK] = sr; }
        }
    }
}

template <typename T, int BITS, bool STREAM>
__global__ __launch_bounds__(ADAMW_BLOCK) void adamw_kernel(const AdamwDesc<BITS> d)
{
    // the tensor of this chunk: the number of running totals that are not above it (64 lanes look at two each)
    const int lane = threadIdx.x & 63, l0 = lane < d.count ? lane : 0, l1 = lane + 64 < d.count ? lane + 64 : 0;
    const int t = __popcll(__ballot(lane < d.count && blockIdx.x >= d.end_chunk[l0])) +
                  __popcll(__ballot(lane + 64 < d.count && blockIdx.x >= d.end_chunk[l1]));
    const unsigned first = t ? d.end_chunk[t - 1] : 0u;
    const long long n = (long long)(d.end_chunk[t] - first - 1u) * ADAMW_CHUNK + d.last[t];
    const long long chunk = (long long)(blockIdx.x - first) * ADAMW_CHUNK;
    const long long base = chunk + (threadIdx.x >> 6) * ADAMW_SCALE_BLOCK;
    if (chunk + ADAMW_CHUNK <= n) adamw_chunk<T, BITS, true, STREAM>(d, t, n, base);
    else adamw_chunk<T, BITS, false, STREAM>(d, t, n, base);
}
