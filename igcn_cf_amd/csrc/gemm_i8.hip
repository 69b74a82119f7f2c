// Rows held in 8-bit integers with one scale each, and the product of two sets of such rows.
//
//   s[r] = max_k |x[r, k]| / 127 (float32),  q[r, k] = x[r, k] / s[r] to the nearest whole number, ties to the even one
//   y[m, n] = (sum_k a[m, k] b[n, k]) sa[m] sb[n] (+ bias[n])
//
// The sum is exact (int32: K <= 131 071); the scales are applied once, in float32, before the one rounding to the output's type.
#include "dtypes.h"

namespace igcn {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// x / s to the nearest whole number, ties to even, decided exactly: q is within 1 of it, r = x - q s is exact (|r| <= s: no more
// digits than x and s have), and r against s / 2 says which neighbour is nearer.
__device__ __forceinline__ int nearest(float x, float s, float inv)
{
    float q = rintf(x * inv);
    const float r = fmaf(-q, s, x), h = 0.5f * s, a = fabsf(r);
    const bool odd = ((int)q & 1) != 0;
    if (a > h || (a == h && odd)) q += r > 0.f ? 1.f : -1.f;
    return (int)fminf(fmaxf(q, -127.f), 127.f);
}

template <typename T>
__global__ __launch_bounds__(kBlock) void quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, int64_t rows, int64_t k, int8_t *__restrict__ q,
                                                               int64_t ldq, float *__restrict__ scale)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t r = (int64_t)blockIdx.x * (kBlock / kWave) + (threadIdx.x >> 6);
    if (r >= rows) return;
    const T *row = x + r * ldx;
    uint32_t big = 0u;                                           // bit patterns of magnitudes: NaN above infinity above all numbers
    for (int64_t i = lane; i < k; i += kWave) big = max(big, __float_as_uint(to_float(row[i])) & 0x7fffffffu);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, off));
    const bool finite = big < 0x7f800000u;
    const float s = finite ? __uint_as_float(big) / 127.f : NAN;
    if (lane == 0) scale[r] = s;
    for (int64_t i = lane; i < k; i += kWave) {
        int c = 0;
        if (finite && s > 0.f) c = s >= 0x1p-120f ? nearest(to_float(row[i]), s, 1.f / s) : (int)fmin(fmax(rint((double)to_float(row[i]) / (double)s), -127.0), 127.0);
        q[r * ldq + i] = (int8_t)c;
    }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void dequantize_rows_kernel(const int8_t *__restrict__ q, int64_t ldq, const float *__restrict__ scale, int64_t rows,
                                                                 int64_t k, T *__restrict__ y, int64_t ldy)
{
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t r = (int64_t)blockIdx.x * (kBlock / kWave) + (threadIdx.x >> 6);
    if (r >= rows) return;
    const float s = scale[r];
    for (int64_t i = lane; i < k; i += kWave) y[r * ldy + i] = from_float<T>((float)q[r * ldq + i] * s);
}

struct GemmArgs {
    const int8_t *a, *b;
    const float *sa, *sb, *bias;
    void *y;
    int64_t lda, ldb, ldy, m, n, k;
    int out;
};

__device__ __forceinline__ void store_out(const GemmArgs &G, int64_t r, int64_t c, int acc)
{
    float v = (float)acc * G.sa[r] * G.sb[c];
    if (G.bias) v += G.bias[c];
    if (G.out == IGCN_DTYPE_F32) static_cast<float *>(G.y)[r * G.ldy + c] = v;
    else if (G.out == IGCN_DTYPE_BF16) static_cast<__hip_bfloat16 *>(G.y)[r * G.ldy + c] = from_float<__hip_bfloat16>(v);
    else static_cast<__half *>(G.y)[r * G.ldy + c] = from_float<__half>(v);
}

// 16 codes of a row from k on, zeros behind its end
__device__ __forceinline__ i32x4 load16(const int8_t *__restrict__ row, int64_t k, int64_t n)
{
    i32x4 v = {0, 0, 0, 0};
    if (k + 16 <= n && (reinterpret_cast<uintptr_t>(row + k) & 15) == 0) return *reinterpret_cast<const i32x4 *>(row + k);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k + i < n) v[i >> 2] |= (int)(uint8_t)row[k + i] << (8 * (i & 3));
    return v;
}

constexpr int kTile = 64, kDepth = 64;
// One workgroup = 64 x 64 of y, a wave 32 x 32 of it
__global__ __launch_bounds__(kBlock) void gemm_i8_kernel(const GemmArgs G)
{
    __shared__ i32x4 as[kTile * kDepth / 16], bs[kTile * kDepth / 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
    const int row = threadIdx.x >> 2, piece = threadIdx.x & 3;
    i32x16 acc = {};
    for (int64_t k0 = 0; k0 < G.k; k0 += kDepth) {
        i32x4 zero = {0, 0, 0, 0};
        as[row * 4 + piece] = m0 + row < G.m ? load16(G.a + (m0 + row) * G.lda, k0 + 16 * piece, G.k) : zero;
        bs[row * 4 + piece] = n0 + row < G.n ? load16(G.b + (n0 + row) * G.ldb, k0 + 16 * piece, G.k) : zero;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const i32x4 av = as[((wave >> 1) * 32 + (lane & 31)) * 4 + 2 * s + (lane >> 5)];
            const i32x4 bv = bs[((wave & 1) * 32 + (lane & 31)) * 4 + 2 * s + (lane >> 5)];
            acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(av, bv, acc, 0, 0, 0);
        }
        __syncthreads();
    }
    const int64_t c = n0 + (wave & 1) * 32 + (lane & 31);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t r = m0 + (wave >> 1) * 32 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        if (r < G.m && c < G.n) store_out(G, r, c, acc[i]);
    }
}

}  // namespace igcn

using namespace igcn;

extern "C" int igcn_quantize_rows_i8(const void *x, int32_t dtype, int64_t ldx, int64_t rows, int64_t k, int8_t *q, int64_t ldq, float *scale, void *stream)
{
    if (!dtype_ok(dtype)) return IGCN_E_RANGE;
    if (rows < 0 || k < 0 || rows > 0x1fffffffcll || ldx < k || ldq < k) return IGCN_E_SHAPE;
    if (rows == 0) return IGCN_OK;
    if (!scale || (k > 0 && (!x || !q))) return IGCN_E_NULL;
    if (misaligned(x, dtype) || (reinterpret_cast<uintptr_t>(scale) & 3)) return IGCN_E_ALIGN;
    const dim3 grid((unsigned)((rows + 3) / 4));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == IGCN_DTYPE_F32) hipLaunchKernelGGL(quantize_rows_kernel<float>, grid, dim3(kBlock), 0, st, static_cast<const float *>(x), ldx, rows, k, q, ldq, scale);
    else if (dtype == IGCN_DTYPE_BF16) hipLaunchKernelGGL(quantize_rows_kernel<__hip_bfloat16>, grid, dim3(kBlock), 0, st, static_cast<const __hip_bfloat16 *>(x), ldx, rows, k, q, ldq, scale);
    else hipLaunchKernelGGL(quantize_rows_kernel<__half>, grid, dim3(kBlock), 0, st, static_cast<const __half *>(x), ldx, rows, k, q, ldq, scale);
    return launch_status();
}

extern "C" int igcn_dequantize_rows_i8(const int8_t *q, int64_t ldq, const float *scale, int64_t rows, int64_t k, void *y, int32_t dtype, int64_t ldy, void *stream)
{
    if (!dtype_ok(dtype)) return IGCN_E_RANGE;
    if (rows < 0 || k < 0 || rows > 0x1fffffffcll || ldy < k || ldq < k) return IGCN_E_SHAPE;
    if (rows == 0 || k == 0) return IGCN_OK;
    if (!q || !scale || !y) return IGCN_E_NULL;
    if (misaligned(y, dtype) || (reinterpret_cast<uintptr_t>(scale) & 3)) return IGCN_E_ALIGN;
    const dim3 grid((unsigned)((rows + 3) / 4));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == IGCN_DTYPE_F32) hipLaunchKernelGGL(dequantize_rows_kernel<float>, grid, dim3(kBlock), 0, st, q, ldq, scale, rows, k, static_cast<float *>(y), ldy);
    else if (dtype == IGCN_DTYPE_BF16) hipLaunchKernelGGL(dequantize_rows_kernel<__hip_bfloat16>, grid, dim3(kBlock), 0, st, q, ldq, scale, rows, k, static_cast<__hip_bfloat16 *>(y), ldy);
    else hipLaunchKernelGGL(dequantize_rows_kernel<__half>, grid, dim3(kBlock), 0, st, q, ldq, scale, rows, k, static_cast<__half *>(y), ldy);
    return launch_status();
}

extern "C" int igcn_matmul_i8(const int8_t *a, int64_t lda, const float *sa, const int8_t *b, int64_t ldb, const float *sb, const float *bias,
                              int64_t m, int64_t n, int64_t k, void *y, int32_t dtype, int64_t ldy, void *stream)
{
    if (!dtype_ok(dtype)) return IGCN_E_RANGE;
    if (m < 0 || n < 0 || k < 0 || lda < k || ldb < k || ldy < n) return IGCN_E_SHAPE;
    if (k > IGCN_MAX_I8_DEPTH) return IGCN_E_RANGE;
    if (m == 0 || n == 0) return IGCN_OK;
    if (!sa || !sb || !y || (k > 0 && (!a || !b))) return IGCN_E_NULL;
    if (misaligned(y, dtype) || ((reinterpret_cast<uintptr_t>(sa) | reinterpret_cast<uintptr_t>(sb) | reinterpret_cast<uintptr_t>(bias)) & 3)) return IGCN_E_ALIGN;
    const int64_t gx = (n + kTile - 1) / kTile, gy = (m + kTile - 1) / kTile;
    if (gx > 0x7fffffff || gy > 65535) return IGCN_E_SHAPE;
    GemmArgs G = {a, b, sa, sb, bias, y, lda, ldb, ldy, m, n, k, dtype};
    hipLaunchKernelGGL(gemm_i8_kernel, dim3((unsigned)gx, (unsigned)gy), dim3(kBlock), 0, static_cast<hipStream_t>(stream), G);
    return launch_status();
}
