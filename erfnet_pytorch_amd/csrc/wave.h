// Reductions over neighbouring lanes of a wave without shared memory (data-parallel primitives and the gfx950 lane swaps).
#pragma once
#include "common.h"

template <int CTRL> __device__ __forceinline__ float wave_dpp(float v)
{
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ void wave_halves(float v, float &a, float &b)        // lanes 0..31 and 32..63, to both halves
{
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned x = r[0], y = r[1];
    a = __builtin_bit_cast(float, x);
    b = __builtin_bit_cast(float, y);
}
__device__ __forceinline__ void wave_rows(float v, float &a, float &b)          // rows of 16: each pair's first and second
{
    const unsigned u = __builtin_bit_cast(unsigned, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned x = r[0], y = r[1];
    a = __builtin_bit_cast(float, x);
    b = __builtin_bit_cast(float, y);
}

// The value of lane (own ^ O).
template <int O> __device__ __forceinline__ unsigned wave_xor(unsigned v)
{
    const int i = (int)v;
    if (O == 1) return (unsigned)__builtin_amdgcn_update_dpp(i, i, 0xb1, 0xf, 0xf, false);
    if (O == 2) return (unsigned)__builtin_amdgcn_update_dpp(i, i, 0x4e, 0xf, 0xf, false);
    if (O == 4) {       // mirror within 8 (own ^ 7), then within 4 (own ^ 3)
        const int m = __builtin_amdgcn_update_dpp(i, i, 0x141, 0xf, 0xf, false);
        return (unsigned)__builtin_amdgcn_update_dpp(m, m, 0x1b, 0xf, 0xf, false);
    }
    if (O == 8) return (unsigned)__builtin_amdgcn_update_dpp(i, i, 0x128, 0xf, 0xf, false);     // rotate a row by 8
    if (O == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        const unsigned first = r[0], second = r[1];
        return (threadIdx.x & 16) ? first : second;
    }
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const unsigned first = r[0], second = r[1];
    return (threadIdx.x & 32) ? first : second;
}
// The value of lane (63 - own): mirrored within 16, then the rows and the halves exchanged.
__device__ __forceinline__ unsigned wave_reverse(unsigned v)
{
    const int i = (int)v;
    return wave_xor<32>(wave_xor<16>((unsigned)__builtin_amdgcn_update_dpp(i, i, 0x140, 0xf, 0xf, false)));
}

// Sum (or maximum) over aligned groups of `lanes` lanes, a power of two up to 64; every lane gets its group's.  A step
// joins the two halves of a group that are each uniform already, so a mirror does for an exchange.
template <typename F> __device__ __forceinline__ float wave_reduce(float v, int lanes, F join)
{
    float a, b;
    if (lanes > 1) v = join(v, wave_dpp<0xb1>(v));          // quad_perm 1,0,3,2
    if (lanes > 2) v = join(v, wave_dpp<0x4e>(v));          // quad_perm 2,3,0,1
    if (lanes > 4) v = join(v, wave_dpp<0x141>(v));         // mirror within 8
    if (lanes > 8) v = join(v, wave_dpp<0x140>(v));         // mirror within 16
    if (lanes > 16) { wave_rows(v, a, b); v = join(a, b); }
    if (lanes > 32) { wave_halves(v, a, b); v = join(a, b); }
    return v;
}
__device__ __forceinline__ float wave_sum(float v, int lanes = 64)
{
    return wave_reduce(v, lanes, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v, int lanes = 64)
{
    return wave_reduce(v, lanes, [](float a, float b) { return fmaxf(a, b); });
}
// Maxima of N values (4 or 8) over the whole wave, as scalars.  The first two steps each join two registers into one that holds
// a half (a row of 16) of either, so that N / 4 registers take the last four: 7 steps for 4 values instead of 24.
template <int N> __device__ __forceinline__ void wave_max_all(unsigned (&v)[N])
{
    unsigned a[N / 2], b[N / 4];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {           // lanes below 32: v[2 i], the others v[2 i + 1]
        const auto r = __builtin_amdgcn_permlane32_swap(v[2 * i], v[2 * i + 1], false, false);
        const unsigned x = r[0], y = r[1];
        a[i] = x > y ? x : y;
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {           // rows: v[4 i], v[4 i + 2], v[4 i + 1], v[4 i + 3]
        const auto r = __builtin_amdgcn_permlane16_swap(a[2 * i], a[2 * i + 1], false, false);
        const unsigned x = r[0], y = r[1];
        b[i] = x > y ? x : y;
    }
    auto step = [](unsigned x, int y) { return x > (unsigned)y ? x : (unsigned)y; };
#pragma unroll
    for (int i = 0; i < N / 4; ++i) b[i] = step(b[i], __builtin_amdgcn_update_dpp((int)b[i], (int)b[i], 0xb1, 0xf, 0xf, false));
#pragma unroll
    for (int i = 0; i < N / 4; ++i) b[i] = step(b[i], __builtin_amdgcn_update_dpp((int)b[i], (int)b[i], 0x4e, 0xf, 0xf, false));
#pragma unroll
    for (int i = 0; i < N / 4; ++i) b[i] = step(b[i], __builtin_amdgcn_update_dpp((int)b[i], (int)b[i], 0x141, 0xf, 0xf, false));
#pragma unroll
    for (int i = 0; i < N / 4; ++i) b[i] = step(b[i], __builtin_amdgcn_update_dpp((int)b[i], (int)b[i], 0x140, 0xf, 0xf, false));
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[4 * i + j] = (unsigned)__builtin_amdgcn_readlane((int)b[i], 16 * ((j & 1) * 2 + (j >> 1)));
}
