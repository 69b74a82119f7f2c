// The product of two sets of rows held in 8-bit integers with one scale each.
//
//   y[m, n] = (sum_k a[m, k] b[n, k]) sa[m] sb[n] (+ bias[n])
//
// The sum is exact (int32: K <= 131 071); the scales are applied once, in float32, before the one rounding to the output's type.
#include "quant_i8.h"
#include <type_traits>

namespace igcn {

typedef int i32x16 __attribute__((ext_vector_type(16)));

struct GemmArgs {
    const int8_t *a, *b;
    const float *sa, *sb, *bias;
    void *y;
    int64_t lda, ldb, ldy, m, n, k;
    int out;
};

// The sum's way to y, the same in every kernel: each operation rounded once in float32, no fused multiply-add.
__device__ __forceinline__ float scaled(int acc, float sa, float sb, const float *bias, int64_t c)
{
#pragma clang fp contract(off)
    const float v = (float)acc * sa * sb;
    return bias ? v + bias[c] : v;
}
__device__ __forceinline__ void store_out(const GemmArgs &G, int64_t r, int64_t c, float v)
{
    if (G.out == IGCN_DTYPE_F32) static_cast<float *>(G.y)[r * G.ldy + c] = v;
    else if (G.out == IGCN_DTYPE_BF16) static_cast<__hip_bfloat16 *>(G.y)[r * G.ldy + c] = from_float<__hip_bfloat16>(v);
    else static_cast<__half *>(G.y)[r * G.ldy + c] = from_float<__half>(v);
}

// 16 codes of a row from k on, zeros behind its end
__device__ __forceinline__ i32x4 load16(const int8_t *__restrict__ row, int64_t k, int64_t n)
{
    i32x4 v = {0, 0, 0, 0};
    if (k + 16 <= n) return *reinterpret_cast<const i32x4_any *>(row + k);
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
        if (r < G.m && c < G.n) store_out(G, r, c, scaled(acc[i], G.sa[r], G.sb[c], G.bias, c));
    }
}


// ---- few rows of a --------------------------------------------------------------------------------------------------------------------
// Bound by the bytes of b, each used once: no tile of b is worth staging.  A wave takes 16 rows of b as the matrix instruction's first
// operand straight from memory (16x16x64: lane l holds row l % 16, 16 bytes at 16 (l / 16)) and the rows of a, the second operand, from
// LDS, where a workgroup lays them out once in the order the lanes read them: [64 codes of depth][16 of them][row][16 bytes].  Rows of a are rounded up to a
// power of two there (lanes past it read another row's bytes; what they compute is not stored).  SHARE: with a long depth the four waves
// of a workgroup take a quarter of it each and add their sums up in LDS (whole numbers: in any order), which fills the card four
// times as well where b has few rows; with a short one every wave has tiles of its own.  KEEP loads are in flight before the first use.
// x in floating point (X is not int8_t): every workgroup makes it 8-bit on the way, with the quantiser's own steps — no launch, no
// buffer; worth it while that is less work than a launch (kFusedValues).
constexpr int kStep = 64;                                        // codes of depth a matrix instruction takes
constexpr int kFewRows = 64;                                     // rows of a: 16 GROUPS
constexpr int kPanelBytes = 32768;                               // of LDS: five workgroups on a CU
constexpr int64_t kFusedValues = 8192;

struct FewArgs {
    GemmArgs g;
    const void *x;                                               // the rows of a in floating point (ldx apart), or NULL
    int64_t ldx;
    int shift, panel;                                            // 2^shift rows of a in LDS; steps of depth that fit there
    int64_t jobs;                                                // of a workgroup at most: tile groups it walks
};

template <int GROUPS, int TILES, int KEEP, bool SHARE, typename X>
__global__ __launch_bounds__(kBlock) void few_rows_i8_kernel(const FewArgs F)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ float sx[kFewRows];
    const GemmArgs &G = F.g;
    i32x4 *const xs = reinterpret_cast<i32x4 *>(smem);           // [step][quarter][row] x 16 bytes
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = lane >> 4;
    const int rows2 = 1 << F.shift, m = (int)G.m;
    int *const sums = reinterpret_cast<int *>(smem + (int64_t)F.panel * kStep * rows2);       // SHARE: [tile, group, wave][row of a][17]
    const int64_t steps = (G.k + kStep - 1) / kStep, tiles = (G.n + 15) / 16;
    const int64_t group0 = (int64_t)blockIdx.x * F.jobs * (SHARE ? 1 : 4) + (SHARE ? 0 : wave);
    constexpr bool kFloat = !std::is_same<X, int8_t>::value;

    if constexpr (kFloat) {                                      // (one panel: the whole depth)
        constexpr int E = Chunk<X>::kValues;
        for (int r = wave; r < m; r += 4) {
            const X *row = static_cast<const X *>(F.x) + r * F.ldx;
            uint32_t big = 0u;
            for (int64_t at = lane * E; at < G.k; at += 64 * E) { Chunk<X> c; c.load(row + at, G.k - at); big = c.largest(big); }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, off));
            const RowScale s(big);
            if (lane == 0) sx[r] = s.s;
            for (int64_t at = lane * E; at < steps * kStep; at += 64 * E) {
                Chunk<X> c;
                c.load(row + at, G.k - at);
                uint32_t w[E / 4] = {};
#pragma unroll
                for (int i = 0; i < E; ++i) w[i >> 2] |= (uint32_t)(s.code(c.v[i]) & 0xff) << (8 * (i & 3));
                __builtin_memcpy(smem + ((at >> 4) * rows2 + r) * 16 + (at & 15), w, E);
            }
        }
    } else if (threadIdx.x < m) sx[threadIdx.x] = G.sa[threadIdx.x];
    __syncthreads();

    i32x4 acc[TILES][GROUPS];
    for (int64_t job = 0; job < F.jobs; ++job) {
        const int64_t tile0 = (group0 + job * (SHARE ? 1 : 4)) * TILES;
        if (SHARE ? tile0 >= tiles : tile0 - (int64_t)wave * TILES >= tiles) break;          // (the same for the whole workgroup)
        const int8_t *row[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int64_t r = (tile0 + t) * 16 + (lane & 15);
            row[t] = G.b + (r < G.n ? r : G.n - 1) * G.ldb + 16 * quarter;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) acc[t][g] = i32x4{0, 0, 0, 0};
        }
        for (int64_t p0 = 0; p0 < steps; p0 += F.panel) {
            const int64_t p1 = p0 + F.panel < steps ? p0 + F.panel : steps;
            if constexpr (!kFloat) if (job == 0 || F.panel < steps) {
                __syncthreads();
                for (int64_t i = threadIdx.x; i < (p1 - p0) * 4 * rows2; i += kBlock) {
                    const int64_t r = i & (rows2 - 1), piece = i >> F.shift;
                    xs[i] = r < m ? load16(G.a + r * G.lda, (p0 * 4 + piece) * 16, G.k) : i32x4{0, 0, 0, 0};
                }
                __syncthreads();
            }
            const int64_t from = SHARE ? p0 + (p1 - p0) * wave / 4 : p0, to = SHARE ? p0 + (p1 - p0) * (wave + 1) / 4 : p1;
            auto multiply = [&](const i32x4 (&v)[TILES], int64_t s) {
                const i32x4 *x = xs + ((s - p0) * 4 + quarter) * rows2;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const i32x4 xv = x[(g * 16 + (lane & 15)) & (rows2 - 1)];
#pragma unroll
                    for (int t = 0; t < TILES; ++t) acc[t][g] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[t], xv, acc[t][g], 0, 0, 0);
                }
            };
            const int64_t whole = G.k / kStep < to ? G.k / kStep : to;
            int64_t s = from;
            for (; s + KEEP <= whole; s += KEEP) {
                i32x4 v[KEEP][TILES];
#pragma unroll
                for (int u = 0; u < KEEP; ++u)
#pragma unroll
                    for (int t = 0; t < TILES; ++t) v[u][t] = *reinterpret_cast<const i32x4_any *>(row[t] + (s + u) * kStep);
#pragma unroll
                for (int u = 0; u < KEEP; ++u) multiply(v[u], s + u);
            }
            for (; s < to; ++s) {
                i32x4 v[TILES];
#pragma unroll
                for (int t = 0; t < TILES; ++t) v[t] = load16(row[t] - 16 * quarter, s * kStep + 16 * quarter, G.k);
                multiply(v, s);
            }
        }
        if constexpr (SHARE) {                                   // lane l holds rows of b 4 (l / 16) + i, row l % 16 of a
            __syncthreads();                                     // (everyone is through with the last job's sums)
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const int at = (t * GROUPS + g) * 4 + wave;
#pragma unroll
                    for (int i = 0; i < 4; ++i) sums[(at * 16 + (lane & 15)) * 17 + 4 * quarter + i] = acc[t][g][i];
                }
            __syncthreads();
            const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const int64_t n = (tile0 + t) * 16 + c;
                    const int mm = g * 16 + r;
                    if (n < G.n && mm < m) {
                        int sum = 0;
#pragma unroll
                        for (int w = 0; w < 4; ++w) sum += sums[(((t * GROUPS + g) * 4 + w) * 16 + r) * 17 + c];
                        store_out(G, mm, n, scaled(sum, sx[mm], G.sb[n], G.bias, n));
                    }
                }
        } else {
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    const int mm = g * 16 + (lane & 15);
                    const int64_t n0 = (tile0 + t) * 16 + 4 * quarter;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (mm < m && n0 + i < G.n) store_out(G, mm, n0 + i, scaled(acc[t][g][i], sx[mm], G.sb[n0 + i], G.bias, n0 + i));
                }
        }
    }
}

template <int GROUPS, typename X> static int few_rows_launch(FewArgs F, hipStream_t st)
{
    const int64_t steps = (F.g.k + kStep - 1) / kStep, tiles = (F.g.n + 15) / 16;
    F.shift = 0;
    while ((1 << F.shift) < F.g.m) ++F.shift;
    const int64_t fits = kPanelBytes / (kStep << F.shift);
    F.panel = (int)(steps < fits ? (steps ? steps : 1) : fits);
    const bool share = steps >= 16;                              // a quarter of the depth is a batch of loads at least
    const bool one_panel = F.panel >= steps;
    constexpr int kTilesOwn = GROUPS == 1 ? 4 : GROUPS == 2 ? 2 : 1;
    const int64_t per = share ? 1 : 4 * kTilesOwn, groups = (tiles + per - 1) / per;
    // a workgroup that lays the rows of a out once and walks several tiles with them: as many as keep 2 048 workgroups busy
    F.jobs = one_panel ? (groups + 2047) / 2048 : 1;
    const int64_t blocks = (groups + F.jobs - 1) / F.jobs;
    if (blocks > 0x7fffffff) return IGCN_E_SHAPE;
    const size_t lds = ((size_t)F.panel * kStep << F.shift) + (share ? (size_t)GROUPS * 4 * 16 * 17 * 4 : 0);
    const dim3 grid((unsigned)blocks);
    if (share) hipLaunchKernelGGL((few_rows_i8_kernel<GROUPS, 1, 4, true, X>), grid, dim3(kBlock), lds, st, F);
    else hipLaunchKernelGGL((few_rows_i8_kernel<GROUPS, kTilesOwn, 1, false, X>), grid, dim3(kBlock), lds, st, F);
    return launch_status();
}

template <typename X> static int few_rows(const FewArgs &F, hipStream_t st)
{
    return F.g.m <= 16 ? few_rows_launch<1, X>(F, st) : F.g.m <= 32 ? few_rows_launch<2, X>(F, st) : few_rows_launch<4, X>(F, st);
}

static int product(const GemmArgs &G, hipStream_t st)
{
    if (G.m <= kFewRows) {
        FewArgs F = {};
        F.g = G;
        return few_rows<int8_t>(F, st);
    }
    const int64_t gx = (G.n + kTile - 1) / kTile, gy = (G.m + kTile - 1) / kTile;
    if (gx > 0x7fffffff || gy > 65535) return IGCN_E_SHAPE;
    hipLaunchKernelGGL(gemm_i8_kernel, dim3((unsigned)gx, (unsigned)gy), dim3(kBlock), 0, st, G);
    return launch_status();
}

static int check_product(const float *sa, const int8_t *b, int64_t ldb, const float *sb, const float *bias, int64_t m, int64_t n, int64_t k, const void *y,
                         int32_t dtype, int64_t ldy)
{
    if (!dtype_ok(dtype)) return IGCN_E_RANGE;
    if (m < 0 || n < 0 || k < 0 || ldb < k || ldy < n) return IGCN_E_SHAPE;
    if (k > IGCN_MAX_I8_DEPTH) return IGCN_E_RANGE;
    if (m == 0 || n == 0) return IGCN_OK;
    if (!sb || !y || (k > 0 && !b)) return IGCN_E_NULL;
    if (misaligned(y, dtype) || ((reinterpret_cast<uintptr_t>(sa) | reinterpret_cast<uintptr_t>(sb) | reinterpret_cast<uintptr_t>(bias)) & 3)) return IGCN_E_ALIGN;
    return IGCN_OK;
}

static bool quantises_on_the_way(int64_t m, int64_t k) { return m <= kFewRows && m * k <= kFusedValues && m * ((k + kStep - 1) / kStep) * kStep <= kPanelBytes / 2; }
static int64_t up16(int64_t x) { return (x + 15) / 16 * 16; }

}  // namespace igcn

using namespace igcn;

extern "C" int igcn_matmul_i8(const int8_t *a, int64_t lda, const float *sa, const int8_t *b, int64_t ldb, const float *sb, const float *bias,
                              int64_t m, int64_t n, int64_t k, void *y, int32_t dtype, int64_t ldy, void *stream)
{
    const int rc = check_product(sa, b, ldb, sb, bias, m, n, k, y, dtype, ldy);
    if (rc != IGCN_OK) return rc;
    if (lda < k) return IGCN_E_SHAPE;
    if (m == 0 || n == 0) return IGCN_OK;
    if (!sa || (k > 0 && !a)) return IGCN_E_NULL;
    const GemmArgs G = {a, b, sa, sb, bias, y, lda, ldb, ldy, m, n, k, dtype};
    return product(G, static_cast<hipStream_t>(stream));
}

extern "C" int64_t igcn_linear_i8_workspace_bytes(int64_t m, int64_t k)
{
    if (m < 0 || k < 0 || k > IGCN_MAX_I8_DEPTH || m > 0x7fffffff) return -1;
    return quantises_on_the_way(m, k) ? 0 : up16(m * up16(k)) + 4 * m;
}

extern "C" int igcn_linear_i8(const void *x, int32_t x_dtype, int64_t ldx, const int8_t *b, int64_t ldb, const float *sb, const float *bias,
                              int64_t m, int64_t n, int64_t k, void *y, int32_t dtype, int64_t ldy, void *workspace, void *stream)
{
    const int rc = check_product(nullptr, b, ldb, sb, bias, m, n, k, y, dtype, ldy);
    if (rc != IGCN_OK) return rc;
    if (!dtype_ok(x_dtype)) return IGCN_E_RANGE;
    if (ldx < k || m > 0x7fffffff) return IGCN_E_SHAPE;
    if (m == 0 || n == 0) return IGCN_OK;
    if (k > 0 && !x) return IGCN_E_NULL;
    if (misaligned(x, x_dtype)) return IGCN_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    GemmArgs G = {nullptr, b, nullptr, sb, bias, y, 0, ldb, ldy, m, n, k, dtype};
    if (quantises_on_the_way(m, k)) {
        FewArgs F = {};
        F.g = G;
        F.x = x;
        F.ldx = ldx;
        if (x_dtype == IGCN_DTYPE_F32) return few_rows<float>(F, st);
        if (x_dtype == IGCN_DTYPE_BF16) return few_rows<__hip_bfloat16>(F, st);
        return few_rows<__half>(F, st);
    }
    if (!workspace) return IGCN_E_NULL;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return IGCN_E_ALIGN;
    int8_t *codes = static_cast<int8_t *>(workspace);            // rows 16 bytes apart or a multiple: the product's loads stay aligned
    float *scale = reinterpret_cast<float *>(codes + up16(m * up16(k)));
    const int rq = igcn_quantize_rows_i8(x, x_dtype, ldx, m, k, codes, up16(k), scale, stream);
    if (rq != IGCN_OK) return rq;
    G.a = codes;
    G.lda = up16(k);
    G.sa = scale;
    return product(G, st);
}
