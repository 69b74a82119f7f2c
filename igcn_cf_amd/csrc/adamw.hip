// AdamW over many tensors in one call, moments in float32 or in 8 bits, with the gradient norm over all tensors and clipping by it.
//
//   g' = c g,  c = min(1, max_norm / (|g| + 1e-6)) or 1;   m = b1 m + (1 - b1) g';   v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// Nothing is used twice: the step is bound by the bytes of p, g, m, v (28 a float32 element, 16.1 with 8-bit moments), a small call by
// its launches.  So: one launch for up to kTensors tensors, their pointers in the launch arguments (nothing is copied to the device,
// a captured step replays with the addresses it was captured with), and one small launch before it that counts the steps, forms the
// bias corrections once per tensor in 64 bits and adds the norm's partial sums up in a fixed order.  Measured (a large copy moves 4.9
// TB/s): 13.2 M float32 elements 70 us = 5.3 TB/s, with 8-bit moments 37 us = 5.7, 128 M of those 366 us = 5.6; 15 bfloat16 tensors, 23 M
// elements, 85 us = 5.9; the norm of 13.2 M float32 gradients 13 us = 4.0, of 23 M in bfloat16 18 us.
//
// 8-bit moments: blocks of 128 consecutive elements share s_m = max |m| / 448 and s_v = max v / 57344 (float32); m / s_m is held as
// e4m3, v / s_v as e5m2.  An average that moves by 0.1 % a step would stand still under a code step of 12-25 % rounded to nearest, so
// the codes are rounded stochastically: code = floor(x + u), u of 16 bits from a hash of (seed, tensor, step, element) — right in the
// mean, the same on every replay and every machine (the float32 step count ends at 2^24: from there on every step draws the same u).
// v > 0 is not held as 0 (m / sqrt(0)) unless it is under 2^-165 of its block's largest.  The averages and codes are formed in
// float32 with every operation rounded once, in the order written (no fused multiply-add): elementary float32 operations in any other
// program give the same codes, bit for bit.
#include "dtypes.h"
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

namespace igcn {

constexpr int kTensors = 56;             // of one launch: 64 bytes each in at most 4 KiB of launch arguments
constexpr int kPer = 8;                  // elements of a thread: 16 lanes (a DPP row) hold a block of 128
constexpr int kChunk = kBlock * kPer;    // elements of a workgroup
constexpr int kNormBlocks = 2048;        // partial sums of a norm launch
constexpr int64_t kMostChunks = (1 << 24) - 1;      // of a launch: 2^32 threads at most
static_assert(IGCN_ADAMW_BLOCK == 16 * kPer, "a block of the 8-bit moments is a DPP row's elements");

struct TensorTable {
    igcn_adamw_tensor t[kTensors];
    int first[kTensors + 1];             // first chunk of each tensor; [n] = all chunks of the launch
    int n;
};
// what the small launch leaves for the others, per tensor of the call
struct Prepared { float factor, step_size, inv_sqrt_c2, keep; uint32_t key, pad[3]; };      // keep = 1 - lr wd

struct Hyper {
    double beta1, beta2, log_beta1, log_beta2, lr, weight_decay, max_norm;
    const float *lr_dev;
    float eps;
    uint32_t seed_lo, seed_hi;
};

// 8 consecutive values of src at element i; `whole`: all 8 are there (at any address: the hardware loads and stores 16 bytes anywhere)
template <typename T> __device__ __forceinline__ void load8(const T *__restrict__ src, int64_t i, int64_t n, bool whole, T (&x)[kPer])
{
    if (whole) {
        load_vector(x, src + i);
    } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k) x[k] = i + k < n ? src[i + k] : T(0.f);
    }
}
template <typename T> __device__ __forceinline__ void store8(T *__restrict__ dst, int64_t i, int64_t n, bool whole, const T (&x)[kPer])
{
    if (whole) {
        store_vector(dst + i, x);
    } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k) if (i + k < n) dst[i + k] = x[k];
    }
}

__device__ __forceinline__ int tensor_of_chunk(const TensorTable &T, int chunk)
{
    int lo = 0, hi = T.n - 1;                                   // the last tensor whose first chunk is not behind this one
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (T.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// ---- the norm ------------------------------------------------------------------------------------------------------------------
template <typename G> __device__ __forceinline__ double chunk_squares(const G *__restrict__ g, int64_t i, int64_t n)
{
    if (i >= n) return 0.0;
    G x[kPer];
    load8(g, i, n, i + kPer <= n, x);
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) { const double y = to_float(x[k]); s = fma(y, y, s); }
    return s;
}

// squares of elements 8 `thread` ... + 7 of a chunk
__device__ __forceinline__ double grad_chunk(const TensorTable &T, int chunk, int thread)
{
    const int k = tensor_of_chunk(T, chunk);
    const igcn_adamw_tensor &t = T.t[k];
    const int64_t i = (int64_t)(chunk - T.first[k]) * kChunk + thread * kPer;
    if (t.grad_dtype == IGCN_DTYPE_F32) return chunk_squares(static_cast<const float *>(t.grad), i, t.n);
    if (t.grad_dtype == IGCN_DTYPE_BF16) return chunk_squares(static_cast<const __hip_bfloat16 *>(t.grad), i, t.n);
    return chunk_squares(static_cast<const __half *>(t.grad), i, t.n);
}

template <int THREADS = kBlock> __device__ __forceinline__ double block_sum(double s, double *lds)
{
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    s = lds[0];
#pragma unroll
    for (int i = 1; i < THREADS / kWave; ++i) s += lds[i];
    __syncthreads();
    return s;
}

// squares of elements i, i + kChunk, ... below `end`: four loads under way before the first sum
template <typename G> __device__ __forceinline__ double run_squares(const G *__restrict__ g, int64_t i, int64_t end)
{
    constexpr int kDeep = 4;
    double s = 0.0;
    for (; i + (kDeep - 1) * kChunk + kPer <= end; i += kDeep * kChunk) {
        G x[kDeep][kPer];
#pragma unroll
        for (int d = 0; d < kDeep; ++d) load_vector(x[d], g + i + d * kChunk);
#pragma unroll
        for (int d = 0; d < kDeep; ++d)
#pragma unroll
            for (int k = 0; k < kPer; ++k) { const double y = to_float(x[d][k]); s = fma(y, y, s); }
    }
    for (; i < end; i += kChunk) s += chunk_squares(g, i, end);
    return s;
}

// partial[blockIdx.x] = squares of the chunks per blockIdx.x ... + per - 1: sums in float64, in an order that depends on the sizes alone
__global__ __launch_bounds__(kBlock) void grad_squares_kernel(const TensorTable T, int per, double *__restrict__ partial)
{
    __shared__ double lds[kBlock / kWave];
    double s = 0.0;
    const int to = min((int)(blockIdx.x + 1) * per, T.first[T.n]);
    for (int chunk = blockIdx.x * per; chunk < to;) {            // from tensor to tensor
        const int k = tensor_of_chunk(T, chunk), stop = min(to, T.first[k + 1]);
        const igcn_adamw_tensor &t = T.t[k];
        const int64_t i = (int64_t)(chunk - T.first[k]) * kChunk + threadIdx.x * kPer, end = min(t.n, (int64_t)(stop - T.first[k]) * kChunk);
        if (t.grad_dtype == IGCN_DTYPE_F32) s += run_squares(static_cast<const float *>(t.grad), i, end);
        else if (t.grad_dtype == IGCN_DTYPE_BF16) s += run_squares(static_cast<const __hip_bfloat16 *>(t.grad), i, end);
        else s += run_squares(static_cast<const __half *>(t.grad), i, end);
        chunk = stop;
    }
    s = block_sum(s, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double norm_of(const double *__restrict__ partial, int n, double *lds)
{
    constexpr int kEach = kNormBlocks / kBlock;                  // (all of one launch's at once)
    double s = 0.0;
    for (int i0 = threadIdx.x; i0 < n; i0 += kNormBlocks) {
        double x[kEach];
#pragma unroll
        for (int d = 0; d < kEach; ++d) x[d] = i0 + d * kBlock < n ? partial[i0 + d * kBlock] : 0.0;
#pragma unroll
        for (int d = 0; d < kEach; ++d) s += x[d];
    }
    return sqrt(block_sum(s, lds));
}

__global__ __launch_bounds__(kBlock) void grad_norm_kernel(const double *__restrict__ partial, int n, float *__restrict__ out)
{
    __shared__ double lds[kBlock / kWave];
    const double norm = norm_of(partial, n, lds);
    if (threadIdx.x == 0) *out = (float)norm;
}

__device__ __forceinline__ double clip_factor(const Hyper &H, double norm)
{
    const double f = H.max_norm / (norm + 1e-6);
    return f > 1.0 ? 1.0 : f;                                    // (a NaN norm stays one: the parameters show it)
}
// One thread per tensor: its step counted, what the elements need of it formed in 64 bits.
__device__ __forceinline__ Prepared count_step(const igcn_adamw_tensor &t, int index, const Hyper &H, double factor)
{
    const float step = *t.step + 1.f;
    *t.step = step;
    const double lr = H.lr_dev ? (double)*H.lr_dev : H.lr;
    Prepared q;
    q.factor = (float)factor;
    q.step_size = (float)(lr / -expm1((double)step * H.log_beta1));          // 1 - b^t without cancellation
    q.inv_sqrt_c2 = (float)(1.0 / sqrt(-expm1((double)step * H.log_beta2)));
    q.key = mix32(mix32((uint32_t)(int64_t)step ^ H.seed_lo) ^ (H.seed_hi + (uint32_t)index * 0x9e3779b9u));
    q.keep = (float)(1.0 - lr * H.weight_decay);
    q.pad[0] = q.pad[1] = q.pad[2] = 0u;
    return q;
}

// ---- before the step: steps counted, bias corrections, the clipping factor ------------------------------------------------------
__global__ __launch_bounds__(kBlock) void adamw_prepare_kernel(const TensorTable T, int index0, const Hyper H, const double *__restrict__ partial,
                                                               int n_partial, const float *norm_in, float *norm_out, Prepared *__restrict__ prep)
{
    __shared__ double lds[kBlock / kWave];
    double factor = 1.0;
    if (H.max_norm > 0.0) {
        const double norm = norm_in ? (double)*norm_in : norm_of(partial, n_partial, lds);
        if (!norm_in && norm_out && index0 == 0 && threadIdx.x == 0) *norm_out = (float)norm;
        factor = clip_factor(H, norm);
    }
    if ((int)threadIdx.x < T.n) prep[index0 + threadIdx.x] = count_step(T.t[threadIdx.x], index0 + threadIdx.x, H, factor);
}

// ---- the step --------------------------------------------------------------------------------------------------------------------
// The hardware's square root and reciprocal (1 ulp each: the update is far below the parameter) know no numbers below 2^-126.  SMALL: what is
// that small goes through them scaled by a power of two, which is exact.  Only an eps in whose company such a root counts asks for it
// (small_eps): in every call, 8-bit moments of bfloat16 parameters, bound by their arithmetic, took 288 us for 270 (134 M elements).
template <bool SMALL> __device__ __forceinline__ float stepped(float p, float m, float v, const Prepared &q, float eps)
{
    float up = 1.f, back = 1.f, scale = 1.f;
    if constexpr (SMALL) { const bool low = v < 0x1p-100f; up = low ? 0x1p64f : 1.f; back = low ? 0x1p-32f : 1.f; }
    const float denom = fmaf(__builtin_amdgcn_sqrtf(v * up) * back, q.inv_sqrt_c2, eps);
    if constexpr (SMALL) scale = denom < 0x1p-100f ? 0x1p100f : 1.f;
    return fmaf(-q.step_size, m * __builtin_amdgcn_rcpf(denom * scale) * scale, p * q.keep);
}

template <bool SMALL, typename P, typename G>
__device__ __forceinline__ void step32(const igcn_adamw_tensor &t, int64_t i, const Hyper &H, const Prepared &q)
{
    const bool ok = i + kPer <= t.n;
    P p[kPer]; G g[kPer]; float m[kPer], v[kPer];
    load8(static_cast<const G *>(t.grad), i, t.n, ok, g);
    load8(static_cast<const float *>(t.exp_avg), i, t.n, ok, m);
    load8(static_cast<const float *>(t.exp_avg_sq), i, t.n, ok, v);
    load8(static_cast<const P *>(t.param), i, t.n, ok, p);
    // m + a (x - m) has no error from beta's own rounding, which a long average with beta near 1 would add up; but what it cuts off is a
    // part of the old average's size, so a short one (beta under a half), which keeps little of that, is formed term by term.
    const float factor = q.factor, b1 = (float)H.beta1, b2 = (float)H.beta2, a1 = (float)(1.0 - H.beta1), a2 = (float)(1.0 - H.beta2);
    const bool long_m = H.beta1 >= 0.5, long_v = H.beta2 >= 0.5;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const float x = to_float(g[k]) * factor;
        m[k] = long_m ? fmaf(a1, x - m[k], m[k]) : fmaf(b1, m[k], a1 * x);
        // (a x first: x^2 passes float32 where a x^2 does not; and an infinite v stays one)
        v[k] = fmaf(a2 * x, x, long_v && v[k] < INFINITY ? fmaf(-a2, v[k], v[k]) : b2 * v[k]);
        p[k] = from_float<P>(stepped<SMALL>(to_float(p[k]), m[k], v[k], q, H.eps));
    }
    store8(static_cast<float *>(t.exp_avg), i, t.n, ok, m);
    store8(static_cast<float *>(t.exp_avg_sq), i, t.n, ok, v);
    store8(static_cast<P *>(t.param), i, t.n, ok, p);
}

template <int ROR> __device__ __forceinline__ float row_ror(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x120 | ROR, 0xf, 0xf, true));
}
__device__ __forceinline__ float row_max(float x)               // the largest of 16 lanes, in all of them
{
    x = fmaxf(x, row_ror<8>(x)); x = fmaxf(x, row_ror<4>(x)); x = fmaxf(x, row_ror<2>(x)); return fmaxf(x, row_ror<1>(x));
}

// t >= 0 as an 8-bit floating code of MANT binary digits, smallest normal 2^EMIN, rounded up where its cut-off part and
// u = (r16 + 0.5) / 2^16 make one
template <int MANT, int EMIN> __device__ __forceinline__ uint32_t code_of(float t, uint32_t r16)
{
    const int e = max(__float_as_int(t) >> 23, 127 + EMIN);
    const float u = ((float)r16 + 0.5f) * 0x1p-16f;
    return ((uint32_t)(e - (127 + EMIN)) << MANT) + (uint32_t)(__builtin_amdgcn_ldexpf(t, MANT + 127 - e) + u);
}

template <bool SMALL, typename P, typename G>
__device__ __forceinline__ void step8(const igcn_adamw_tensor &t, int64_t i, const Hyper &H, const Prepared &q)
{
#pragma clang fp contract(off)
    const bool ok = i + kPer <= t.n;
    P p[kPer]; G g[kPer]; uint8_t mc[kPer], vc[kPer];
    load8(static_cast<const G *>(t.grad), i, t.n, ok, g);
    load8(static_cast<const uint8_t *>(t.exp_avg), i, t.n, ok, mc);
    load8(static_cast<const uint8_t *>(t.exp_avg_sq), i, t.n, ok, vc);
    load8(static_cast<const P *>(t.param), i, t.n, ok, p);
    const int64_t block = i / IGCN_ADAMW_BLOCK;
    const bool there = i < t.n;                                  // (lanes behind the end stay for their row's maximum)
    const float sm = there ? t.scales[2 * block] : 0.f, sv = there ? t.scales[2 * block + 1] : 0.f;
    const float b1 = (float)H.beta1, b2 = (float)H.beta2, a1 = (float)(1.0 - H.beta1), a2 = (float)(1.0 - H.beta2);
    float m[kPer], v[kPer], big_m = 0.f, big_v = 0.f;
    float all = fabsf(sm) + fabsf(sv);                           // finite where every input of these averages is
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const float x = to_float(g[k]) * q.factor;
        all += fabsf(x);
        m[k] = b1 * (__builtin_amdgcn_cvt_f32_fp8(mc[k], 0) * sm) + a1 * x;
        v[k] = b2 * (__builtin_amdgcn_cvt_f32_bf8(vc[k], 0) * sv) + a2 * x * x;
        big_m = fmaxf(big_m, fabsf(m[k]));
        big_v = fmaxf(big_v, v[k]);
        p[k] = from_float<P>(stepped<SMALL>(to_float(p[k]), m[k], v[k], q, H.eps));
    }
    const bool bad = !(all < INFINITY);
    if (bad) big_m = big_v = INFINITY;
    big_m = row_max(big_m);
    big_v = row_max(big_v);
    constexpr float kSmallest = 0x1p-100f;                       // below: held as zero (the reciprocal stays finite)
    const float inv_m = big_m >= kSmallest && big_m < INFINITY ? 1.f / big_m * 448.f : 0.f;
    const float inv_v = big_v >= kSmallest && big_v < INFINITY ? 1.f / big_v * 57344.f : 0.f;
    const uint32_t base = mix32(q.key ^ (uint32_t)((uint64_t)i >> 32));
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const uint32_t h = mix32((uint32_t)(i + k) ^ base);
        const float tm = fabsf(m[k]) * inv_m, tv = v[k] * inv_v;
        uint32_t cm = bad ? 0u : code_of<3, -6>(tm, h & 0xffffu), cv = bad ? 0u : code_of<2, -14>(tv, h >> 16);
        cv = max(cv, tv > 0.f ? 1u : 0u);
        cm |= cm && m[k] < 0.f ? 0x80u : 0u;
        mc[k] = (uint8_t)cm;
        vc[k] = (uint8_t)cv;
    }
    if (!there) return;
    store8(static_cast<uint8_t *>(t.exp_avg), i, t.n, ok, mc);
    store8(static_cast<uint8_t *>(t.exp_avg_sq), i, t.n, ok, vc);
    store8(static_cast<P *>(t.param), i, t.n, ok, p);
    if ((threadIdx.x & 15) == 0) {
        t.scales[2 * block] = big_m < INFINITY ? (inv_m == 0.f ? 0.f : big_m * (1.f / 448.f)) : NAN;
        t.scales[2 * block + 1] = big_v < INFINITY ? (inv_v == 0.f ? 0.f : big_v * (1.f / 57344.f)) : NAN;
    }
}

template <int BITS, bool SMALL, typename P, typename G>
__device__ __forceinline__ void step_any(const igcn_adamw_tensor &t, int64_t i, const Hyper &H, const Prepared &q)
{
    if constexpr (BITS == 8) step8<SMALL, P, G>(t, i, H, q);
    else if (i < t.n) step32<SMALL, P, G>(t, i, H, q);
}

// elements 8 `thread` ... + 7 of a tensor's chunk
template <int BITS, bool SMALL>
__device__ __forceinline__ void step_chunk(const igcn_adamw_tensor &t, int chunk, int thread, const Hyper &H, const Prepared &q)
{
    const int64_t i = (int64_t)chunk * kChunk + thread * kPer;
    if (t.dtype == IGCN_DTYPE_F32) step_any<BITS, SMALL, float, float>(t, i, H, q);
    else if (t.dtype == IGCN_DTYPE_BF16) {
        if (t.grad_dtype == IGCN_DTYPE_F32) step_any<BITS, SMALL, __hip_bfloat16, float>(t, i, H, q);
        else step_any<BITS, SMALL, __hip_bfloat16, __hip_bfloat16>(t, i, H, q);
    } else {
        if (t.grad_dtype == IGCN_DTYPE_F32) step_any<BITS, SMALL, __half, float>(t, i, H, q);
        else step_any<BITS, SMALL, __half, __half>(t, i, H, q);
    }
}

template <int BITS, bool SMALL>
__global__ __launch_bounds__(kBlock) void adamw_step_kernel(const TensorTable T, const Hyper H, const Prepared *__restrict__ prep)
{
    const int k = tensor_of_chunk(T, blockIdx.x);
    const Prepared q = prep[k];
    step_chunk<BITS, SMALL>(T.t[k], blockIdx.x - T.first[k], threadIdx.x, H, q);
}

// A call of small tensors is its launches: here one does all of it.  A workgroup of kSmallBlock threads per tensor, so that nobody else
// reads the step it counts; the norm over all tensors, where there is one, every workgroup adds up for itself, in the same order.
// us of a captured call, one launch / two: a tensor of 4 chunks 4.4 / 4.3 (8-bit moments 6.7 / 6.2); of 12 chunks, three rounds of the workgroup,
// one launch would take 9.3 (15.4).  From the host a launch less is 2.5 us less.
constexpr int kSmallBlock = 1024;
constexpr int64_t kSmallChunks = kSmallBlock / kBlock;           // of a tensor
constexpr int64_t kSmallNormChunks = 16;                         // of the call, where every workgroup reads all gradients
template <int BITS, bool SMALL>
__global__ __launch_bounds__(kSmallBlock) void adamw_small_kernel(const TensorTable T, const Hyper H, const float *norm_in, float *norm_out)
{
    constexpr int kParts = kSmallBlock / kBlock;
    __shared__ Prepared prep;
    __shared__ double lds[kSmallBlock / kWave];
    const int part = __builtin_amdgcn_readfirstlane(threadIdx.x / kBlock), thread = threadIdx.x % kBlock;
    double factor = 1.0;
    if (H.max_norm > 0.0) {
        double norm;
        if (norm_in) norm = (double)*norm_in;
        else {
            double s = 0.0;
            for (int chunk = part; chunk < T.first[T.n]; chunk += kParts) s += grad_chunk(T, chunk, thread);
            norm = sqrt(block_sum<kSmallBlock>(s, lds));
            if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
        }
        factor = clip_factor(H, norm);
    }
    const igcn_adamw_tensor &t = T.t[blockIdx.x];
    if (threadIdx.x == 0) prep = count_step(t, blockIdx.x, H, factor);
    __syncthreads();
    if (part < T.first[blockIdx.x + 1] - T.first[blockIdx.x]) step_chunk<BITS, SMALL>(t, part, thread, H, prep);        // (a quarter of the workgroup a chunk)
}

// Whether sqrt(v / (1 - b2^t)) with v below 2^-126, 2^-63 / sqrt(1 - b2) at most, is more than 2^-27 of eps: less is lost in the sum's rounding.
// (From there on eps, and so the denominator, is above 2^-36.)
static bool small_eps(const Hyper &H) { return H.eps < 0x1p-36 / std::sqrt(1.0 - H.beta2); }

// ---- host side -------------------------------------------------------------------------------------------------------------------
static int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// Calls fn(table, index of its first tensor) for every launch the tensors need; empty tensors keep their place (no chunk of their own).
template <typename F> static int for_tables(const igcn_adamw_tensor *tensors, int64_t n, F fn)
{
    for (int64_t at = 0; at < n;) {
        TensorTable T;
        T.n = 0;
        int64_t chunks = 0;
        const int64_t from = at;
        for (; at < n && T.n < kTensors; ++at) {
            const int64_t c = chunks_of(tensors[at].n);
            if (chunks + c > kMostChunks) break;                // (one tensor alone is at most that: check_tensors)
            T.t[T.n] = tensors[at];
            T.first[T.n++] = (int)chunks;
            chunks += c;
        }
        for (int i = T.n; i <= kTensors; ++i) T.first[i] = (int)chunks;
        const int rc = fn(T, (int)from);
        if (rc != IGCN_OK) return rc;
    }
    return IGCN_OK;
}

static int grad_squares(const igcn_adamw_tensor *tensors, int64_t n, double *partial, int *n_partial, hipStream_t st)
{
    *n_partial = 0;
    return for_tables(tensors, n, [&](const TensorTable &T, int) {
        const int chunks = T.first[T.n];
        if (chunks == 0) return (int)IGCN_OK;
        const int least = (chunks + kNormBlocks - 1) / kNormBlocks, per = least == 1 ? 1 : (least + 3) / 4 * 4, blocks = (chunks + per - 1) / per;
        hipLaunchKernelGGL(grad_squares_kernel, dim3((unsigned)blocks), dim3(kBlock), 0, st, T, per, partial + *n_partial);
        *n_partial += blocks;
        return launch_status();
    });
}

// Whether memory that the step writes is shared between two of its tensors, or with a gradient or a number that it reads (those may share theirs).
static int check_overlap(const igcn_adamw_tensor *tensors, int64_t n, bool eight, const float *lr_dev, const float *norm_in, const float *norm_out)
{
    struct Stretch { uintptr_t begin, end; bool written; };
    const std::unique_ptr<Stretch[]> all(new (std::nothrow) Stretch[6 * n + 2]);
    if (!all) return (int)hipErrorOutOfMemory;
    int64_t count = 0;
    auto add = [&](const void *p, int64_t bytes, bool written) {
        if (bytes) all[count++] = Stretch{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes, written};
    };
    for (int64_t i = 0; i < n; ++i) {
        const igcn_adamw_tensor &t = tensors[i];
        add(t.param, t.n * (t.dtype == IGCN_DTYPE_F32 ? 4 : 2), true);
        add(t.exp_avg, t.n * (eight ? 1 : 4), true);
        add(t.exp_avg_sq, t.n * (eight ? 1 : 4), true);
        if (eight) add(t.scales, (t.n + IGCN_ADAMW_BLOCK - 1) / IGCN_ADAMW_BLOCK * 8, true);
        add(t.step, 4, true);
        add(t.grad, t.n * (t.grad_dtype == IGCN_DTYPE_F32 ? 4 : 2), false);
    }
    add(lr_dev, lr_dev ? 4 : 0, false);
    add(norm_in ? norm_in : norm_out, norm_in || norm_out ? 4 : 0, !norm_in);
    std::sort(all.get(), all.get() + count, [](const Stretch &a, const Stretch &b) { return a.begin < b.begin; });
    uintptr_t any = 0, written = 0;                              // the furthest end so far
    for (int64_t i = 0; i < count; ++i) {
        if (all[i].begin < (all[i].written ? any : written)) return IGCN_E_OVERLAP;
        any = std::max(any, all[i].end);
        if (all[i].written) written = std::max(written, all[i].end);
    }
    return IGCN_OK;
}

// moment_bits 0: only the gradients are looked at
static int check_tensors(const igcn_adamw_tensor *tensors, int64_t n, int moment_bits, const float *lr_dev = nullptr, const float *norm_in = nullptr,
                         const float *norm_out = nullptr)
{
    if (n < 0 || n > 0x7fffffff) return IGCN_E_SHAPE;
    if (n > 0 && !tensors) return IGCN_E_NULL;
    const bool eight = moment_bits == 8;
    for (int64_t i = 0; i < n; ++i) {
        const igcn_adamw_tensor &t = tensors[i];
        if (t.n < 0 || t.n > kMostChunks * kChunk) return IGCN_E_SHAPE;
        if (!dtype_ok(t.grad_dtype)) return IGCN_E_RANGE;
        if (t.n > 0 && !t.grad) return IGCN_E_NULL;
        if (misaligned(t.grad, t.grad_dtype)) return IGCN_E_ALIGN;
        if (moment_bits == 0) continue;
        if (!dtype_ok(t.dtype) || (t.grad_dtype != t.dtype && t.grad_dtype != IGCN_DTYPE_F32)) return IGCN_E_RANGE;
        if (!t.step || (t.n > 0 && (!t.param || !t.exp_avg || !t.exp_avg_sq))) return IGCN_E_NULL;
        if (eight && t.n > 0 && !t.scales) return IGCN_E_NULL;
        if (misaligned(t.param, t.dtype)) return IGCN_E_ALIGN;
        if (!eight && ((reinterpret_cast<uintptr_t>(t.exp_avg) | reinterpret_cast<uintptr_t>(t.exp_avg_sq)) & 3)) return IGCN_E_ALIGN;
        if ((reinterpret_cast<uintptr_t>(t.scales) | reinterpret_cast<uintptr_t>(t.step)) & 3) return IGCN_E_ALIGN;
    }
    return moment_bits ? check_overlap(tensors, n, eight, lr_dev, norm_in, norm_out) : (int)IGCN_OK;
}

}  // namespace igcn

using namespace igcn;

extern "C" int64_t igcn_adamw_workspace_bytes(const igcn_adamw_tensor *tensors_host, int64_t n_tensors)
{
    if (check_tensors(tensors_host, n_tensors, 0) != IGCN_OK) return -1;
    int64_t partials = 0;
    const int rc = for_tables(tensors_host, n_tensors, [&](const TensorTable &T, int) {
        partials += std::min(T.first[T.n], kNormBlocks);
        return (int)IGCN_OK;
    });
    if (rc != IGCN_OK) return -1;
    return n_tensors * (int64_t)sizeof(Prepared) + partials * 8 + 16;
}

extern "C" int igcn_grad_norm(const igcn_adamw_tensor *tensors_host, int64_t n_tensors, float *norm, void *workspace, void *stream)
{
    const int rc = check_tensors(tensors_host, n_tensors, 0);
    if (rc != IGCN_OK) return rc;
    if (!norm || !workspace) return IGCN_E_NULL;
    if ((reinterpret_cast<uintptr_t>(norm) & 3) || (reinterpret_cast<uintptr_t>(workspace) & 15)) return IGCN_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    double *partial = static_cast<double *>(workspace);
    int n_partial = 0;
    const int rs = grad_squares(tensors_host, n_tensors, partial, &n_partial, st);
    if (rs != IGCN_OK) return rs;
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kBlock), 0, st, partial, n_partial, norm);
    return launch_status();
}

extern "C" int igcn_adamw_step(const igcn_adamw_tensor *tensors_host, int64_t n_tensors, int32_t moment_bits, double lr, const float *lr_dev,
                               double beta1, double beta2, double eps, double weight_decay, double max_norm, const float *norm_in,
                               float *norm_out, uint64_t seed, void *workspace, void *stream)
{
    if (moment_bits != 8 && moment_bits != 32) return IGCN_E_RANGE;
    const bool clipped = max_norm > 0.0;
    const int rc = check_tensors(tensors_host, n_tensors, moment_bits, lr_dev, clipped ? norm_in : nullptr, clipped ? norm_out : nullptr);
    if (rc != IGCN_OK) return rc;
    if (!(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return IGCN_E_RANGE;
    if (!(eps >= 0.0) || !(weight_decay >= 0.0) || !(max_norm >= 0.0)) return IGCN_E_RANGE;
    if (n_tensors > 0 && !workspace) return IGCN_E_NULL;
    if (max_norm > 0.0 && !norm_in && !norm_out) return IGCN_E_NULL;
    const uintptr_t numbers = reinterpret_cast<uintptr_t>(norm_in) | reinterpret_cast<uintptr_t>(norm_out) | reinterpret_cast<uintptr_t>(lr_dev);
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) || (numbers & 3)) return IGCN_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    Prepared *prep = static_cast<Prepared *>(workspace);
    double *partial = reinterpret_cast<double *>(prep + n_tensors);
    int n_partial = 0;
    Hyper H;
    H.beta1 = beta1; H.beta2 = beta2; H.log_beta1 = std::log(beta1); H.log_beta2 = std::log(beta2);
    H.lr = lr; H.lr_dev = lr_dev;
    H.weight_decay = weight_decay; H.max_norm = max_norm; H.eps = (float)eps;
    H.seed_lo = (uint32_t)seed; H.seed_hi = (uint32_t)(seed >> 32);
    const bool small = small_eps(H);
    if (n_tensors > 0 && n_tensors <= kTensors) {
        int64_t all = 0, most = 0;
        for (int64_t i = 0; i < n_tensors; ++i) {
            const int64_t c = chunks_of(tensors_host[i].n);
            all += c;
            most = c > most ? c : most;
        }
        if (most <= kSmallChunks && (all <= kSmallNormChunks || max_norm == 0.0 || norm_in))
            return for_tables(tensors_host, n_tensors, [&](const TensorTable &T, int) {
                auto launch = [&](auto *kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)T.n), dim3(kSmallBlock), 0, st, T, H, norm_in, norm_out); };
                if (moment_bits == 8) small ? launch(adamw_small_kernel<8, true>) : launch(adamw_small_kernel<8, false>);
                else small ? launch(adamw_small_kernel<32, true>) : launch(adamw_small_kernel<32, false>);
                return launch_status();
            });
    }
    if (max_norm > 0.0 && !norm_in) {
        const int rs = grad_squares(tensors_host, n_tensors, partial, &n_partial, st);
        if (rs != IGCN_OK) return rs;
        if (n_tensors == 0) {
            hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kBlock), 0, st, partial, 0, norm_out);
            return launch_status();
        }
    }
    return for_tables(tensors_host, n_tensors, [&](const TensorTable &T, int index0) {
        hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(kBlock), 0, st, T, index0, H, partial, n_partial, norm_in, norm_out, prep);
        int rs = launch_status();
        if (rs != IGCN_OK || T.first[T.n] == 0) return rs;
        auto launch = [&](auto *kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)T.first[T.n]), dim3(kBlock), 0, st, T, H, prep + index0); };
        if (moment_bits == 8) small ? launch(adamw_step_kernel<8, true>) : launch(adamw_step_kernel<8, false>);
        else small ? launch(adamw_step_kernel<32, true>) : launch(adamw_step_kernel<32, false>);
        return launch_status();
    });
}
