// What the row quantiser and the products that quantise on their way share.
#pragma once
#include "dtypes.h"

namespace igcn {

// 16 bytes of a row: 4 or 8 values.  `left`: values of the row from here on; what is behind its end reads as zero.
template <typename T> struct Chunk {
    static constexpr int kValues = 16 / sizeof(T);
    float v[kValues];
    __device__ __forceinline__ void load(const T *__restrict__ p, int64_t left)
    {
        if (left >= kValues) {
            T x[kValues];
            load_vector(x, p);
#pragma unroll
            for (int i = 0; i < kValues; ++i) v[i] = to_float(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kValues; ++i) v[i] = i < left ? to_float(p[i]) : 0.f;
        }
    }
    __device__ __forceinline__ uint32_t largest(uint32_t m) const        // bit patterns of magnitudes: NaN above infinity above all numbers
    {
#pragma unroll
        for (int i = 0; i < kValues; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        return m;
    }
};

// A row's scale and its reciprocal, from the bit pattern of its largest magnitude.
struct RowScale {
    float s, inv;
    __device__ __forceinline__ explicit RowScale(uint32_t big)
    {
        s = big < 0x7f800000u ? __uint_as_float(big) / 127.f : NAN;
        inv = s > 0.f ? 1.f / s : 0.f;                           // (a row of zeros, or one that is broken: codes 0)
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
// 127 2^-24 before that rounding, it is the right one unless what was cut off is within 2^-16 of a half: a wave that meets such a
// value (one in 30 000) takes the exact way for the piece.  5 instructions a value instead of 16: at 16 they took as long as the bytes.
template <typename T> __device__ __forceinline__ void pack_codes(uint32_t (&w)[Chunk<T>::kValues / 4], const Chunk<T> &c, const RowScale &s)
{
    constexpr int E = Chunk<T>::kValues;
    constexpr float kMagic = 12582912.f, kNear = 0.5f - 0x1p-16f;
    float near = 0.f;
    uint32_t b[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float m = fmaf(c.v[i], s.inv, kMagic);
        near = fmaxf(near, fabsf(fmaf(c.v[i], s.inv, kMagic - m)));
        b[i] = __float_as_uint(m);
    }
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {                            // the low bytes of four words
        const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x04000c0cu);
        w[i] = s.inv > 0.f ? lo | hi : 0u;                       // (a row of zeros, or one that is broken)
    }
    if (__any((near >= kNear || s.s < 0x1p-120f) && s.inv > 0.f)) {
#pragma unroll
        for (int i = 0; i < E / 4; ++i) w[i] = 0u;
#pragma unroll
        for (int i = 0; i < E; ++i) w[i >> 2] |= (uint32_t)(s.code(c.v[i]) & 0xff) << (8 * (i & 3));
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
