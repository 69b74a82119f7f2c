// Rows as 8-bit integers with one scale each, and back.
//
//   s[r] = max_k |x[r, k]| / 127 (float32),  q[r, k] = x[r, k] / s[r] to the nearest whole number, ties to the even one
//
// Bound by the bytes: x read once, q written once.  A row's values stay in registers between its maximum and its codes: L lanes hold a
// row in I pieces of 16 bytes each (adjacent lanes, adjacent pieces: every load and store of a wave covers whole lines), L the smallest
// power of two that makes I one, up to a wave; from 129 pieces on more waves share the row, at most two pieces a lane until it is long
// (2048 rows of 8192 bfloat16: two pieces on 512 lanes 13.7 us, four on 256 16.7).  Short rows: each lane group takes R rows at once, R loads
// in flight before the first maximum.  Rows over kHeldPieces do not fit: they are read a second time (from L2).
// Measured: 206151 x 64 float32 12.7 us = 5.3 TB/s (and back 11.8 = 5.7), 2048 x 8191 bfloat16, rows at any multiple of 2, 14.3 us = 3.5
// (back to float32 16).
#include "quant_i8.h"

namespace igcn {

constexpr int kHeldPieces = 8 * kBlock;                          // 32 KiB: the longest row that a workgroup keeps in registers

template <int L> __device__ __forceinline__ uint32_t group_max(uint32_t m, uint32_t *lds)
{
#pragma unroll
    for (int off = (L < kWave ? L : kWave) / 2; off > 0; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off));
    if constexpr (L > kWave) {
        if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x >> 6] = m;
        __syncthreads();
        m = lds[0];
#pragma unroll
        for (int i = 1; i < L / kWave; ++i) m = max(m, lds[i]);
    }
    return m;
}

template <typename T, int L, int I, int R>
__global__ __launch_bounds__(L > kWave ? L : kBlock) void quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, int64_t rows, int64_t k, int8_t *__restrict__ q,
                                                               int64_t ldq, float *__restrict__ scale)
{
    constexpr int E = Chunk<T>::kValues, kThreads = L > kWave ? L : kBlock;
    __shared__ uint32_t lds[kThreads / kWave];
    const int lane = threadIdx.x & (L - 1);
    const int64_t r0 = ((int64_t)blockIdx.x * (kThreads / L) + threadIdx.x / L) * R;
    Chunk<T> c[R][I];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int64_t at = (int64_t)(lane + L * i) * E;
            c[r][i].load(x + (r0 + r) * ldx + at, r0 + r < rows ? k - at : 0);
        }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        Largest<T> big;
#pragma unroll
        for (int i = 0; i < I; ++i) big.of(c[r][i]);
        const RowScale s(group_max<L>(big.bits(), lds));
        if (r0 + r >= rows) return;                              // (L > a wave: R is 1, the whole workgroup leaves)
        if (lane == 0) scale[r0 + r] = s.s;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int64_t at = (int64_t)(lane + L * i) * E;
            if (at < k) store_codes(q + (r0 + r) * ldq + at, k - at, c[r][i], s);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kBlock) void quantize_long_rows_kernel(const T *__restrict__ x, int64_t ldx, int64_t k, int8_t *__restrict__ q, int64_t ldq,
                                                                    float *__restrict__ scale)
{
    constexpr int E = Chunk<T>::kValues;
    __shared__ uint32_t lds[kBlock / kWave];
    const T *row = x + blockIdx.x * ldx;
    Largest<T> big;
    for (int64_t at = (int64_t)threadIdx.x * E; at < k; at += kBlock * E) {
        Chunk<T> c;
        c.load(row + at, k - at);
        big.of(c);
    }
    const RowScale s(group_max<kBlock>(big.bits(), lds));
    if (threadIdx.x == 0) scale[blockIdx.x] = s.s;
    for (int64_t at = (int64_t)threadIdx.x * E; at < k; at += kBlock * E) {
        Chunk<T> c;
        c.load(row + at, k - at);
        store_codes(q + blockIdx.x * ldq + at, k - at, c, s);
    }
}

// 16 bytes of y a lane; a row's pieces on adjacent lanes of L
template <typename T, int L, int R>
__global__ __launch_bounds__(kBlock) void dequantize_rows_kernel(const int8_t *__restrict__ q, int64_t ldq, const float *__restrict__ scale, int64_t rows,
                                                                 int64_t k, T *__restrict__ y, int64_t ldy)
{
    constexpr int E = Chunk<T>::kValues;
    const int64_t at = ((int64_t)blockIdx.y * L + (threadIdx.x & (L - 1))) * E;
    const int64_t r0 = ((int64_t)blockIdx.x * (kBlock / L) + threadIdx.x / L) * R;
    const int64_t left = k - at;
    if (left <= 0) return;
    uint32_t w[R][E / 4] = {};
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r0 + r >= rows) break;
        s[r] = scale[r0 + r];
        const int8_t *p = q + (r0 + r) * ldq + at;
        if (left >= E) __builtin_memcpy(w[r], p, E);
        else {
#pragma unroll
            for (int i = 0; i < E; ++i) if (i < left) w[r][i >> 2] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r0 + r >= rows) break;
        T v[E];
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = from_float<T>((float)(int8_t)(w[r][i >> 2] >> (8 * (i & 3))) * s[r]);
        T *p = y + (r0 + r) * ldy + at;
        if (left >= E) store_vector(p, v);
        else {
#pragma unroll
            for (int i = 0; i < E; ++i) if (i < left) p[i] = v[i];
        }
    }
}

template <typename T, int L, int I, int R>
static int quantize_launch(const T *x, int64_t ldx, int64_t rows, int64_t k, int8_t *q, int64_t ldq, float *scale, hipStream_t st)
{
    constexpr int kThreads = L > kWave ? L : kBlock;
    const int64_t per = (int64_t)(kThreads / L) * R;
    hipLaunchKernelGGL((quantize_rows_kernel<T, L, I, R>), dim3((unsigned)((rows + per - 1) / per)), dim3(kThreads), 0, st, x, ldx, rows, k, q, ldq, scale);
    return launch_status();
}

template <typename T> static int quantize(const T *x, int64_t ldx, int64_t rows, int64_t k, int8_t *q, int64_t ldq, float *scale, hipStream_t st)
{
    const int64_t pieces = (k + Chunk<T>::kValues - 1) / Chunk<T>::kValues;
    if (pieces <= 4) return quantize_launch<T, 4, 1, 4>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces <= 8) return quantize_launch<T, 8, 1, 4>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces <= 16) return quantize_launch<T, 16, 1, 2>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces <= 32) return quantize_launch<T, 32, 1, 2>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces <= 64) return quantize_launch<T, 64, 1, 2>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces <= 128) return quantize_launch<T, 64, 2, 1>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces <= 256) return quantize_launch<T, 128, 2, 1>(x, ldx, rows, k, q, ldq, scale, st);
    // no more rows than CUs: a row's own time is what counts, so 1 024 lanes share it (4 rows of 8192 bfloat16: 5.0 us; 512 lanes 7.4)
    if (pieces > 256 && rows <= 256 && pieces <= 1024) return quantize_launch<T, 1024, 1, 1>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces > 256 && rows <= 256 && pieces <= 2048) return quantize_launch<T, 1024, 2, 1>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces <= 512) return quantize_launch<T, kBlock, 2, 1>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces <= 1024) return quantize_launch<T, 2 * kBlock, 2, 1>(x, ldx, rows, k, q, ldq, scale, st);
    if (pieces <= kHeldPieces) return quantize_launch<T, kBlock, 8, 1>(x, ldx, rows, k, q, ldq, scale, st);
    hipLaunchKernelGGL(quantize_long_rows_kernel<T>, dim3((unsigned)rows), dim3(kBlock), 0, st, x, ldx, k, q, ldq, scale);
    return launch_status();
}

template <typename T, int L, int R>
static int dequantize_launch(const int8_t *q, int64_t ldq, const float *scale, int64_t rows, int64_t k, int64_t pieces, T *y, int64_t ldy, hipStream_t st)
{
    const int64_t per = (int64_t)(kBlock / L) * R, gy = (pieces + L - 1) / L;
    hipLaunchKernelGGL((dequantize_rows_kernel<T, L, R>), dim3((unsigned)((rows + per - 1) / per), (unsigned)gy), dim3(kBlock), 0, st, q, ldq, scale, rows, k, y, ldy);
    return launch_status();
}

template <typename T> static int dequantize(const int8_t *q, int64_t ldq, const float *scale, int64_t rows, int64_t k, T *y, int64_t ldy, hipStream_t st)
{
    const int64_t pieces = (k + Chunk<T>::kValues - 1) / Chunk<T>::kValues;
    if (pieces <= 4) return dequantize_launch<T, 4, 4>(q, ldq, scale, rows, k, pieces, y, ldy, st);
    if (pieces <= 8) return dequantize_launch<T, 8, 4>(q, ldq, scale, rows, k, pieces, y, ldy, st);
    if (pieces <= 16) return dequantize_launch<T, 16, 4>(q, ldq, scale, rows, k, pieces, y, ldy, st);
    if (pieces <= 32) return dequantize_launch<T, 32, 4>(q, ldq, scale, rows, k, pieces, y, ldy, st);
    return dequantize_launch<T, 64, 4>(q, ldq, scale, rows, k, pieces, y, ldy, st);
}

}  // namespace igcn

using namespace igcn;

constexpr int64_t kMostRows = 0x7fffffff;
// A launch has fewer than 2^32 threads and 65536 x 64 pieces of a row: larger arrays go in slabs, a gigabyte each and more
constexpr int64_t kSlabRows = 1 << 22, kSlabColumns = 1 << 23;

extern "C" int igcn_quantize_rows_i8(const void *x, int32_t dtype, int64_t ldx, int64_t rows, int64_t k, int8_t *q, int64_t ldq, float *scale, void *stream)
{
    if (!dtype_ok(dtype)) return IGCN_E_RANGE;
    if (rows < 0 || k < 0 || rows > kMostRows || ldx < k || ldq < k) return IGCN_E_SHAPE;
    if (rows == 0) return IGCN_OK;
    if (!scale || (k > 0 && (!x || !q))) return IGCN_E_NULL;
    if (misaligned(x, dtype) || (reinterpret_cast<uintptr_t>(scale) & 3)) return IGCN_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = IGCN_OK;
    for (int64_t r = 0; r < rows && rc == IGCN_OK; r += kSlabRows) {
        const int64_t n = rows - r < kSlabRows ? rows - r : kSlabRows;
        if (dtype == IGCN_DTYPE_F32) rc = quantize(static_cast<const float *>(x) + r * ldx, ldx, n, k, q + r * ldq, ldq, scale + r, st);
        else if (dtype == IGCN_DTYPE_BF16) rc = quantize(static_cast<const __hip_bfloat16 *>(x) + r * ldx, ldx, n, k, q + r * ldq, ldq, scale + r, st);
        else rc = quantize(static_cast<const __half *>(x) + r * ldx, ldx, n, k, q + r * ldq, ldq, scale + r, st);
    }
    return rc;
}

extern "C" int igcn_dequantize_rows_i8(const int8_t *q, int64_t ldq, const float *scale, int64_t rows, int64_t k, void *y, int32_t dtype, int64_t ldy, void *stream)
{
    if (!dtype_ok(dtype)) return IGCN_E_RANGE;
    if (rows < 0 || k < 0 || rows > kMostRows || ldy < k || ldq < k) return IGCN_E_SHAPE;
    if (rows == 0 || k == 0) return IGCN_OK;
    if (!q || !scale || !y) return IGCN_E_NULL;
    if (misaligned(y, dtype) || (reinterpret_cast<uintptr_t>(scale) & 3)) return IGCN_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    int rc = IGCN_OK;
    for (int64_t r = 0; r < rows; r += kSlabRows)
        for (int64_t c = 0; c < k && rc == IGCN_OK; c += kSlabColumns) {
            const int64_t n = rows - r < kSlabRows ? rows - r : kSlabRows, w = k - c < kSlabColumns ? k - c : kSlabColumns, at = r * ldy + c;
            const int8_t *from = q + r * ldq + c;
            if (dtype == IGCN_DTYPE_F32) rc = dequantize(from, ldq, scale + r, n, w, static_cast<float *>(y) + at, ldy, st);
            else if (dtype == IGCN_DTYPE_BF16) rc = dequantize(from, ldq, scale + r, n, w, static_cast<__hip_bfloat16 *>(y) + at, ldy, st);
            else rc = dequantize(from, ldq, scale + r, n, w, static_cast<__half *>(y) + at, ldy, st);
        }
    return rc;
}
