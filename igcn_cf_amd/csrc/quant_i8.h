// What the row quantiser and the products that quantise on their way share.
#pragma once
#include "dtypes.h"

namespace igcn {

// 16 bytes of a row: 4 or 8 values, as they came.  `left`: values of the row from here on; what is behind its end reads as zero.
template <typename T> struct Chunk {
    static constexpr int kValues = 16 / sizeof(T);
    uint32_t w[4];
    __device__ __forceinline__ void load(const T *__restrict__ p, int64_t left)
    {
        T x[kValues];
        if (left >= kValues) load_vector(x, p);
        else {
#pragma unroll
            for (int i = 0; i < kValues; ++i) x[i] = i < left ? p[i] : T(0.f);
        }
        __builtin_memcpy(w, x, 16);
    }
    __device__ __forceinline__ float value(int i) const
    {
        T x;
        if constexpr (sizeof(T) == 4) { const uint32_t u = w[i]; __builtin_memcpy(&x, &u, 4); }
        else { const uint16_t u = (uint16_t)(w[i >> 1] >> (16 * (i & 1))); __builtin_memcpy(&x, &u, 2); }
        return to_float(x);
    }
};

// The largest magnitude of some values, by bit patterns (NaN above infinity above all numbers, in every type): two at a time where they are
// of 16 bits.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <typename T> struct Largest {
    uint32_t m = 0u;
    __device__ __forceinline__ void of(const Chunk<T> &c)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) m = max(m, c.w[i] & 0x7fffffffu);
            else m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, c.w[i] & 0x7fff7fffu)));
        }
    }
    __device__ __forceinline__ uint32_t bits() const             // as a float32 pattern
    {
        if constexpr (sizeof(T) == 4) return m;
        else {
            const uint16_t u = (uint16_t)max(m & 0xffffu, m >> 16);
            T x;
            __builtin_memcpy(&x, &u, 2);
            return __float_as_uint(to_float(x)) & 0x7fffffffu;
        }
    }
};

// A row's scale and its reciprocal, from the bit pattern of its largest magnitude.
struct RowScale {
    float s, inv;
    __device__ __forceinline__ explicit RowScale(uint32_t big)
    {
        const float b = __uint_as_float(big);
        if (big >= 0x04000000u) {                                // 2^-119 and more: b / 127 correctly rounded without the long division
            constexpr float kRcp = 1.f / 127.f;
            const float q = b * kRcp;
            s = fmaf(fmaf(-127.f, q, b), kRcp, q);
            s = big < 0x7f800000u ? s : NAN;
        } else s = b / 127.f;
        inv = s > 0.f ? __builtin_amdgcn_rcpf(s) : 0.f;          // (1 ulp; a row of zeros, or one that is broken: codes 0)
    }
    // x / s to the nearest whole number, ties to even, decided exactly: q = rint(x inv) is within 1 of it, r = x - q s is exact (|r| <= s:
    // no more digits than x and s have together), and r against s / 2 says which neighbour is nearer.  A scale below 2^-120 has few
    // digits or an infinite reciprocal: 64 bits decide there.
    __device__ __forceinline__ int code(float x) const
    {
        if (s >= 0x1p-120f) {
            float q = rintf(x * inv);
            const float r = fmaf(-q, s, x), h = 0.5f * s, a = fabsf(r);
            const bool odd = ((int)q & 1) != 0;
            if (a > h || (a == h && odd)) q += r > 0.f ? 1.f : -1.f;
            return (int)__builtin_amdgcn_fmed3f(q, -127.f, 127.f);
        }
        return s > 0.f ? (int)fmin(fmax(rint((double)x / (double)s), -127.0), 127.0) : 0;
    }
};

// The codes of a piece, packed.  x inv + 1.5 2^23 in one operation leaves the nearest whole number in the low bits; off by at most
// 127 2^-23 before that rounding, it is the right one unless what was cut off is within 2^-15 of a half: a wave that meets such a
// value takes the exact way for its place in the piece (one value in 16 000; in bfloat16, where half of the largest is a likely value, most
// pieces: 50000 x 64 7.5 us when the whole piece went that way, 6.7 so).  5 instructions a value instead of 16: at 16 they took as long as the bytes.
template <typename T> __device__ __forceinline__ void pack_codes(uint32_t (&w)[Chunk<T>::kValues / 4], const Chunk<T> &c, const RowScale &s)
{
    constexpr int E = Chunk<T>::kValues;
    constexpr float kMagic = 12582912.f, kNear = 0.5f - 0x1p-15f;
    float near = 0.f;
    uint32_t b[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float x = c.value(i), m = fmaf(x, s.inv, kMagic);
        near = fmaxf(near, fabsf(fmaf(x, s.inv, kMagic - m)));
        b[i] = __float_as_uint(m);
    }
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {                            // the low bytes of four words
        const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x04000c0cu);
        w[i] = s.inv > 0.f ? lo | hi : 0u;                       // (a row of zeros, or one that is broken)
    }
    if (__any((near >= kNear || s.s < 0x1p-120f) && s.inv > 0.f)) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float x = c.value(i), m = fmaf(x, s.inv, kMagic);
            if (__any((fabsf(fmaf(x, s.inv, kMagic - m)) >= kNear || s.s < 0x1p-120f) && s.inv > 0.f)) {
                const int shift = 8 * (i & 3);
                w[i >> 2] = (w[i >> 2] & ~(0xffu << shift)) | (uint32_t)(s.code(x) & 0xff) << shift;
            }
        }
    }
}

template <typename T> __device__ __forceinline__ void store_codes(int8_t *__restrict__ q, int64_t left, const Chunk<T> &c, const RowScale &s)
{
    constexpr int E = Chunk<T>::kValues;
    uint32_t w[E / 4];
    pack_codes<T>(w, c, s);
    if (left >= E) __builtin_memcpy(q, w, E);
    else {
#pragma unroll
        for (int i = 0; i < E; ++i) if (i < left) q[i] = (int8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
}

}  // namespace igcn
