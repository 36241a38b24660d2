// 16-byte accesses to rows that start at any element (gfx950 global loads and stores take any byte
// address; the packed types below tell the compiler so).  A row of an odd length keeps the wide access:
// only the lane that holds the row's last, partial vector goes element by element.
#pragma once
#include "common.h"

template <typename T> struct Vec16;
template <> struct Vec16<float> {
    static constexpr int N = 4;
    struct __attribute__((packed, aligned(4))) Raw { u32x4 v; };
    static __device__ __forceinline__ void unpack(u32x4 r, float (&f)[4])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned u = r[i];        // (a bit cast of the vector's element itself reads element 0)
            f[i] = __builtin_bit_cast(float, u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4])
    {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, f[i]);
        return r;
    }
    static __device__ __forceinline__ float get(const float *p) { return *p; }
    static __device__ __forceinline__ void put(float *p, float f) { *p = f; }
};
template <> struct Vec16<bf16_t> {
    static constexpr int N = 8;
    struct __attribute__((packed, aligned(2))) Raw { u32x4 v; };
    static __device__ __forceinline__ void unpack(u32x4 r, float (&f)[8])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __builtin_bit_cast(float, r[i] << 16);
            f[2 * i + 1] = __builtin_bit_cast(float, r[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8])
    {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){f[2 * i], f[2 * i + 1]}, bf16x2));
        return r;
    }
    static __device__ __forceinline__ float get(const bf16_t *p) { return bf16_to_f32(*p); }
    static __device__ __forceinline__ void put(bf16_t *p, float f) { *p = f32_to_bf16(f); }
};

// The first `left` elements of r, zeros behind them.
template <typename T> __device__ __forceinline__ u32x4 first16(u32x4 r, int left)
{
    constexpr int per = 4 / sizeof(T);          // elements of one 32-bit word
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int k = left - w * per;
        r[w] &= k >= per ? 0xffffffffu : per == 2 && k == 1 ? 0xffffu : 0u;
    }
    return r;
}

// `left` elements of the row begin at p; elements from `left` on read as zero.  `inside`: all 16 bytes at p lie in the
// tensor, whoever they belong to, so that a row's last, partial vector is one load as well (element by element its
// loads wait for one another: a layer norm of bf16 rows of 101 ran at 1.8 TB/s with them, 4.3 TB/s without).
template <typename T> __device__ __forceinline__ u32x4 ld16(const T *p, int left, bool inside = false)
{
    u32x4 r = {0u, 0u, 0u, 0u};
    if (left >= Vec16<T>::N || (inside && left > 0)) {
        r = reinterpret_cast<const typename Vec16<T>::Raw *>(p)->v;
    } else if (left > 0) {
        constexpr int per = 4 / sizeof(T);
#pragma unroll
        for (int i = 0; i < Vec16<T>::N - 1; ++i)
            if (i < left) {
                const unsigned bits = sizeof(T) == 4 ? __builtin_bit_cast(unsigned, (float)Vec16<T>::get(p + i))
                                                     : __builtin_bit_cast(unsigned, (float)Vec16<T>::get(p + i)) >> 16;
                r[i / per] |= bits << (i % per * 16);
            }
    }
    return r;
}
// An access that leaves the caches to others (STREAM), or an ordinary one; V is a packed struct around a vector.
template <bool STREAM, typename V> __device__ __forceinline__ auto ld_vec(const V *p)
{
    typedef decltype(V::v) Loose __attribute__((aligned(alignof(V))));      // (a pointer to the member would promise its own)
    if (STREAM) return (decltype(V::v))__builtin_nontemporal_load((const Loose *)p);
    return p->v;
}
template <bool STREAM, typename V, typename R> __device__ __forceinline__ void st_vec(V *p, R r)
{
    typedef R Loose __attribute__((aligned(alignof(V))));
    if (STREAM) __builtin_nontemporal_store((Loose)r, (Loose *)p);
    else p->v = r;
}
// The first `left` elements of f: 16 bytes, or the partial vector in pieces of 8, 4 and 2.
template <bool STREAM = false, typename T> __device__ __forceinline__ void st16(T *p, const float (&f)[Vec16<T>::N], int left)
{
    typedef typename Vec16<T>::Raw Raw;
    u32x4 r = Vec16<T>::pack(f);
    if (left >= Vec16<T>::N) {
        st_vec<STREAM>(reinterpret_cast<Raw *>(p), r);
        return;
    }
    if (left <= 0) return;
    struct __attribute__((packed, aligned(sizeof(T)))) Two { u32x2 v; };
    struct __attribute__((packed, aligned(sizeof(T)))) One { unsigned v; };
    constexpr int per = 4 / sizeof(T);
    if (left & (2 * per)) {
        reinterpret_cast<Two *>(p)->v = (u32x2){r[0], r[1]};
        p += 2 * per;
        r[0] = r[2];
        r[1] = r[3];
    }
    if (left & per) {
        reinterpret_cast<One *>(p)->v = r[0];
        p += per;
        r[0] = r[1];
    }
    if (per == 2 && (left & 1)) *reinterpret_cast<unsigned short *>(p) = (unsigned short)r[0];
}
