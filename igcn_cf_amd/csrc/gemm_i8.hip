// The product of two sets of rows held in 8-bit integers with one scale each.
//
//   y[m, n] = (sum_k a[m, k] b[n, k]) sa[m] sb[n] (+ bias[n])
//
// The sum is exact (int32: K <= 131 071); the scales are applied once, in float32, before the one rounding to the output's type.
//
// Measured: 8192 x 8192 x 4096 to bfloat16 262 us = 2.1 POP/s (a library's bare int8 product: 306 us; matrix pipes busy 52 % of the cycles, LDS
// 1.6 M conflict cycles of 30 M), 512 x 96421 x 64 to float32 46-54 us = 3.7-4.3 TB/s of y (the same stores alone 45), 4 x 16384 x 8192 28 us =
// 4.8 TB/s of b, 16 x 4096 x 4096 7 us, 1 x 96421 x 64 from float32 7.1 us.
#include "gemm_i8_rule.h"
#include "quant_i8.h"
#include <type_traits>

namespace igcn {

typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef int int_any __attribute__((aligned(1)));

struct GemmArgs {
    const int8_t *a, *b;
    const float *sa, *sb, *bias;
    void *y;
    int64_t lda, ldb, ldy, m, n, k;
    int out;
};

// The sum's way to y, the same in every kernel: each operation rounded once in float32, no fused multiply-add.
__device__ __forceinline__ float scaled(int acc, float sa, float sb, bool biased, float bias)
{
#pragma clang fp contract(off)
    const float v = (float)acc * sa * sb;
    return biased ? v + bias : v;
}
__device__ __forceinline__ void store_out(const GemmArgs &G, int64_t r, int64_t c, float v)
{
    if (G.out == IGCN_DTYPE_F32) static_cast<float *>(G.y)[r * G.ldy + c] = v;
    else if (G.out == IGCN_DTYPE_BF16) static_cast<__hip_bfloat16 *>(G.y)[r * G.ldy + c] = from_float<__hip_bfloat16>(v);
    else static_cast<__half *>(G.y)[r * G.ldy + c] = from_float<__half>(v);
}

// 16 codes without their first `by` (16 and more: zeros)
__device__ __forceinline__ i32x4 behind(i32x4 v, int by)
{
    const uint64_t lo = (uint32_t)v[0] | (uint64_t)(uint32_t)v[1] << 32, hi = (uint32_t)v[2] | (uint64_t)(uint32_t)v[3] << 32;
    const int bits = 8 * (by & 7);
    const uint64_t a = by >= 16 ? 0 : by >= 8 ? hi : lo, b = by >= 8 ? 0 : hi, c = a >> bits | (b << 1) << (63 - bits), d = b >> bits;
    return i32x4{(int)c, (int)(c >> 32), (int)d, (int)(d >> 32)};
}
// 16 codes of which the first `keep` stay (0 and less: none)
__device__ __forceinline__ i32x4 first(i32x4 v, int keep)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = min(max(keep - 4 * i, 0), 4);
        v[i] &= (int)(((uint64_t)1 << 8 * n) - 1);
    }
    return v;
}
__device__ __forceinline__ i32x4 load16(const int8_t *__restrict__ p) { return *reinterpret_cast<const i32x4_any *>(p); }
// 16 codes of a row of n from k on, zeros behind its end: the last 16 of the row hold what is there of them
__device__ __forceinline__ i32x4 load16(const int8_t *__restrict__ row, int k, int n)
{
    if (n >= 16) {
        const int at = min(k, n - 16);
        return behind(load16(row + at), k - at);
    }
    i32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i)
        if (k + i < n) v[i >> 2] |= (int)(uint8_t)row[k + i] << (8 * (i & 3));
    return v;
}

// ---- many rows of a -------------------------------------------------------------------------------------------------------------------
// Bound by the matrix cores (deep sums) or by writing y (shallow ones).  A workgroup makes a TM x TN tile of y, a wave TM / WM x TN / WN of it in
// 32 x 32 pieces (v_mfma_i32_32x32x32_i8: lane l holds row l % 32, 16 bytes of depth at 16 (l / 32)).  128 codes of depth of either side
// go to LDS per stage, two stages in turn: the next one is on its way from memory while this one is multiplied, one barrier a stage.
// DIRECT (rows 16-byte aligned, depth a multiple of 16): memory to LDS without registers (global_load_lds, 1 KiB a wave and instruction,
// lane after lane); else through registers, one stage under way there (300 x 700 x 333 4.9 us, 300 x 700 x 2051 10.6, 512 x 8192 x 4095 37.1;
// with up to three under way 5.5, 11.2, 36.4).  A row's eight 16-byte pieces stand in LDS at piece ^ (row / 2 % 8): 16 lanes that read the
// same piece of 16 neighbouring rows hit 64 different banks; memory-to-LDS writes linearly, so it is the lane's source that is permuted.
// Depth past the end reads a block of zeros, rows past the end the last row (not stored).
// BY_DEPTH (a 64 x 64 tile of four waves): a wave takes a quarter of the stage's depth for the whole tile instead of all of it for its own piece,
// and they exchange sums in the end: LDS is read half as often and no product waits for the one before it.
// Workgroups go to the eight XCDs in turn: each XCD takes a run of tiles, 4 tiles of a deep at a time, so that the tiles under way there
// share their rows in its L2 (512 x 96421 x 64, whose rows of y end inside a line, without: 47 -> 74 us).
__device__ const i32x4 g_zeros = {0, 0, 0, 0};

typedef __attribute__((address_space(3))) void lds_void;

// memory -> LDS, 16 bytes a lane, lane after lane from byte `lds` on, without the compiler's knowledge: it would wait for it before any
// later LDS read, the other stage's among them.  The kernel waits itself (wait_for_lds) before the barrier behind which it is read.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"                  // (m0 is a reserved register: saying that it is written is the point)
__device__ __forceinline__ void to_lds(const void *base, unsigned offset, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void to_lds(const void *p, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(p), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop
// all but the last LEFT are there
template <int LEFT> __device__ __forceinline__ void wait_for_lds() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(LEFT) : "memory"); }

struct TileArgs { GemmArgs g; int64_t tiles_m, tiles_n, per_xcd; bool asks_ahead; };

constexpr size_t kExchanged = 3 * 4 * 4096;                      // of LDS: three waves' sums of four pieces

template <int TM, int TN, int WM, int WN, int STAGES, bool DIRECT, bool BY_DEPTH>
__global__ __launch_bounds__(64 * WM * WN, 1) void tiles_i8_kernel(const TileArgs T)
{
    constexpr int kWaves = WM * WN, RT = TM / WM / 32, CT = TN / WN / 32, NA = TM / 8 / kWaves, NB = TN / 8 / kWaves;
    constexpr int kStage = (TM + TN) * kDepth;
    static_assert(!BY_DEPTH || (RT == 1 && CT == 1 && kWaves == kDepth / 32), "a quarter of the depth for each of four waves");
    constexpr int AR = BY_DEPTH ? WM : RT, AC = BY_DEPTH ? WN : CT;       // pieces whose sums a wave holds
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    unsigned char *const ring = smem + (TM + 2 * TN) * 4;       // the stages; behind them, the strips of the way out
    const GemmArgs &G = T.g;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = (int64_t)(blockIdx.x & 7) * T.per_xcd + (blockIdx.x >> 3);
    if ((int64_t)(blockIdx.x >> 3) >= T.per_xcd || t >= T.tiles_m * T.tiles_n) return;
    // runs of 4 tile rows, column after column
    constexpr int bd = 4;
    const int64_t band = t / (bd * T.tiles_n), in = t - band * bd * T.tiles_n, high = T.tiles_m - bd * band < bd ? T.tiles_m - bd * band : bd;
    const int64_t m0 = (bd * band + in % high) * TM, n0 = in / high * TN;

    // this lane's pieces: rows 8 (wave NA + i) + lane / 8 of the tile, piece (lane % 8) ^ (row / 2 % 8); offsets from the tile's first row fit
    // 32 bits
    auto piece = [&](int i) { return ((lane & 7) ^ ((4 * i + (lane >> 4)) & 7)) * 16; };       // ... of rows 8 i ... 8 i + 7
    const int8_t *const base_a = G.a + m0 * G.lda, *const base_b = G.b + n0 * G.ldb;
    const int last_a = (int)(G.m - m0 < TM ? G.m - m0 : TM) - 1, last_b = (int)(G.n - n0 < TN ? G.n - n0 : TN) - 1;
    unsigned oa[NA], ob[NB];
#pragma unroll
    for (int i = 0; i < NA; ++i) oa[i] = (unsigned)min(8 * (wave * NA + i) + (lane >> 3), last_a) * (unsigned)G.lda + piece(wave * NA + i);
#pragma unroll
    for (int i = 0; i < NB; ++i) ob[i] = (unsigned)min(8 * (wave * NB + i) + (lane >> 3), last_b) * (unsigned)G.ldb + piece(wave * NB + i);
    const int64_t stages = (G.k + kDepth - 1) / kDepth;
    i32x4 held[DIRECT ? 1 : NA + NB];                            // the stage on its way in registers, where it goes that way
    const unsigned lds0 = (unsigned)(uintptr_t)(lds_void *)ring;

    const int k = (int)G.k;
    auto fetch = [&](int64_t s) {                                // stage s of both sides: on its way to LDS, or to registers
        const int k0 = (int)s * kDepth;
        if constexpr (DIRECT) {
            const unsigned at = lds0 + (unsigned)(s % STAGES) * kStage + wave * NA * 1024, bt = at + TM * kDepth + wave * (NB - NA) * 1024;
            if (k0 + kDepth <= k) {
#pragma unroll
                for (int i = 0; i < NA; ++i) to_lds(base_a + k0, oa[i], at + 1024 * i);
#pragma unroll
                for (int i = 0; i < NB; ++i) to_lds(base_b + k0, ob[i], bt + 1024 * i);
            } else {                                             // (pieces are whole: the depth is a multiple of 16)
                const void *const zeros = &g_zeros;
#pragma unroll
                for (int i = 0; i < NA; ++i) to_lds(k0 + piece(wave * NA + i) < k ? (const void *)(base_a + k0 + oa[i]) : zeros, at + 1024 * i);
#pragma unroll
                for (int i = 0; i < NB; ++i) to_lds(k0 + piece(wave * NB + i) < k ? (const void *)(base_b + k0 + ob[i]) : zeros, bt + 1024 * i);
            }
        } else {                                                 // (past the end: the row's last 16 codes, put in place by land())
#pragma unroll
            for (int i = 0; i < NA; ++i) held[i] = load16(base_a + (oa[i] - piece(wave * NA + i)) + min(k0 + piece(wave * NA + i), k - 16));
#pragma unroll
            for (int i = 0; i < NB; ++i) held[NA + i] = load16(base_b + (ob[i] - piece(wave * NB + i)) + min(k0 + piece(wave * NB + i), k - 16));
        }
    };
    auto land = [&](int64_t s) {                                 // registers to LDS
        i32x4 *at = reinterpret_cast<i32x4 *>(ring + (s % STAGES) * kStage);
        const int k0 = (int)s * kDepth;
        if (k0 + kDepth > k && k >= 16) {
#pragma unroll
            for (int i = 0; i < NA; ++i) held[i] = behind(held[i], max(k0 + piece(wave * NA + i) - (k - 16), 0));
#pragma unroll
            for (int i = 0; i < NB; ++i) held[NA + i] = behind(held[NA + i], max(k0 + piece(wave * NB + i) - (k - 16), 0));
        }
#pragma unroll
        for (int i = 0; i < NA; ++i) at[(wave * NA + i) * 64 + lane] = held[i];
#pragma unroll
        for (int i = 0; i < NB; ++i) at[TM * kDepth / 16 + (wave * NB + i) * 64 + lane] = held[NA + i];
    };

    // Where every tile starts with reads that queue behind the writes of y (i8_asks_ahead): the first row of tiles of a band asks for the rows
    // of b of kSoon tiles on, twice what an XCD has under way, so that those find them in a cache.
    constexpr int kSoon = 64;
    i32x4 soon = {0, 0, 0, 0};
    if constexpr (DIRECT && !BY_DEPTH && TM < 256) {
        static_assert(64 * kWaves == 4 * TN, "four lanes a row");
        const int64_t r = n0 + kSoon * TN + threadIdx.x / 4;
        if (T.asks_ahead && in % high == 0 && r < G.n) soon = load16(G.b + r * G.ldb + ((threadIdx.x & 3) * k / 4 & ~15));
    }
    i32x16 acc[AR][AC] = {};
    const int wm = wave / WN, wn = wave % WN;
    const int half = lane >> 5, turn = (lane >> 1) & 7;
    const int ra = (BY_DEPTH ? 0 : wm * (TM / WM)) + (lane & 31), rb = (BY_DEPTH ? 0 : wn * (TN / WN)) + (lane & 31);
    float *const fa = reinterpret_cast<float *>(smem), *const fb = fa + TM, *const fc = fb + TN;       // the tile's scales and bias, for the way out
    for (int i = threadIdx.x; i < TM; i += 64 * kWaves) fa[i] = i <= last_a ? G.sa[m0 + i] : 0.f;
    for (int i = threadIdx.x; i < TN; i += 64 * kWaves) {
        fb[i] = i <= last_b ? G.sb[n0 + i] : 0.f;
        fc[i] = G.bias && i <= last_b ? G.bias[n0 + i] : 0.f;
    }
    if constexpr (DIRECT) {
        for (int64_t s = 0; s < STAGES - 1 && s < stages; ++s) fetch(s);
    } else if (k >= 16) {
        fetch(0);
        land(0);
        if (1 < stages) fetch(1);
    } else if (k > 0) {
#pragma unroll
        for (int i = 0; i < NA; ++i) held[i] = load16(base_a + (oa[i] - piece(wave * NA + i)), piece(wave * NA + i), k);
#pragma unroll
        for (int i = 0; i < NB; ++i) held[NA + i] = load16(base_b + (ob[i] - piece(wave * NB + i)), piece(wave * NB + i), k);
        land(0);
    }
    auto stage = [&](int64_t s) {
        if constexpr (DIRECT) {                                  // stage s is there: all but the STAGES - 2 behind it
            if (s + STAGES - 2 < stages) wait_for_lds<(STAGES - 2) * (NA + NB)>(); else wait_for_lds<0>();
        }
        __syncthreads();                                         // ... for everyone, and everyone is through with the stage before it
        const unsigned char *sa = ring + (s % STAGES) * kStage + ra * kDepth, *sb = ring + (s % STAGES) * kStage + TM * kDepth + rb * kDepth;
        i32x4 av[AR], bv[AC];
        auto read = [&](int j) {
            const int at = ((2 * j + half) ^ turn) * 16;
#pragma unroll
            for (int r = 0; r < AR; ++r) av[r] = *reinterpret_cast<const i32x4 *>(sa + r * 32 * kDepth + at);
#pragma unroll
            for (int c = 0; c < AC; ++c) bv[c] = *reinterpret_cast<const i32x4 *>(sb + c * 32 * kDepth + at);
        };
        read(BY_DEPTH ? wave : 0);                               // (before the next stage is sent for: its addresses take a while)
        if constexpr (DIRECT) if (s + STAGES - 1 < stages) fetch(s + STAGES - 1);
#pragma unroll
        for (int j = 0; j < (BY_DEPTH ? 1 : kDepth / 32); ++j) {
            if (j) read(j);
#pragma unroll
            for (int r = 0; r < AR; ++r)
#pragma unroll
                for (int c = 0; c < AC; ++c) acc[r][c] = __builtin_amdgcn_mfma_i32_32x32x32_i8(bv[c], av[r], acc[r][c], 0, 0, 0);
        }
        if constexpr (!DIRECT) if (s + 1 < stages) {
            land(s + 1);
            if (s + 2 < stages) fetch(s + 2);
        }
    };
    for (int64_t s = 0; s < stages; ++s) stage(s);
    __syncthreads();
    if constexpr (BY_DEPTH) {                                    // piece q of the tile goes to wave q: [piece][three other waves][quarter][lane], 4 sums each
        i32x4 *const sums = reinterpret_cast<i32x4 *>(ring);
#pragma unroll
        for (int q = 0; q < kWaves; ++q)
            if (q != wave) {
                i32x4 *to = sums + ((q * 3 + (wave - (wave > q))) * 4) * 64 + lane;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const i32x16 &part = acc[q / WN][q % WN];
                    to[64 * i] = i32x4{part[4 * i], part[4 * i + 1], part[4 * i + 2], part[4 * i + 3]};
                }
            }
        __syncthreads();
        i32x16 all = acc[0][0];
#pragma unroll
        for (int q = 1; q < kWaves; ++q)
            if (q == wave) all = acc[q / WN][q % WN];
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const i32x4 x = sums[((wave * 3 + k) * 4 + i) * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) all[4 * i + e] += x[e];
            }
        acc[0][0] = all;
        __syncthreads();                                         // (the strips stand where the sums stood)
    }

    // The way out.  b is the matrix instruction's first operand: lane l holds row l % 32 of a and columns 8 (i / 4) + 4 (l / 32) + i % 4, four
    // neighbours of a row of y at a time.  They cross a strip of LDS of the wave's own (32 rows, its columns) so that a store takes whole
    // lines: 16 bytes a lane, neighbouring lanes along the row.
    auto put = [&](auto *y) {
        using Y = std::remove_pointer_t<decltype(y)>;
        constexpr int kE = 16 / sizeof(Y), kCols = CT * 32, kLanes = kCols / kE, kRows = 64 / kLanes;
        constexpr int kRow = kCols * sizeof(Y) + 16;             // (16 bytes more a row: other banks)
        unsigned char *const strip = ring + wave * 32 * (kCols * 4 + 16);
        const bool biased = G.bias != nullptr;
        const int n1 = wn * (TN / WN) + lane % kLanes * kE;      // of the tile: this lane's columns on the way out
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const float s = fa[wm * (TM / WM) + r * 32 + (lane & 31)];
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int at = c * 32 + 8 * q + 4 * half;
                    const float4 sb4 = *reinterpret_cast<const float4 *>(fb + wn * (TN / WN) + at);
                    const float4 bi4 = *reinterpret_cast<const float4 *>(fc + wn * (TN / WN) + at);
                    auto out = [&](int e, float sb, float bias) { return from_float<Y>(scaled(acc[r][c][4 * q + e], s, sb, biased, bias)); };
                    Y v[4] = {out(0, sb4.x, bi4.x), out(1, sb4.y, bi4.y), out(2, sb4.z, bi4.z), out(3, sb4.w, bi4.w)};
                    __builtin_memcpy(__builtin_assume_aligned(strip + (lane & 31) * kRow + at * sizeof(Y), 8), v, sizeof(v));
                }
            const int m1 = wm * (TM / WM) + r * 32 + lane / kLanes;
            Y *p = y + (m0 + m1) * G.ldy + n0 + n1;
#pragma unroll
            for (int i = 0; i < 32 / kRows; ++i) {
                const i32x4 w = *reinterpret_cast<const i32x4 *>(strip + (lane / kLanes + i * kRows) * kRow + lane % kLanes * 16);
                if (m1 + i * kRows <= last_a) {
                    if (n1 + kE - 1 <= last_b) *reinterpret_cast<i32x4_any *>(p) = w;
                    else {
                        Y v[kE];
                        __builtin_memcpy(v, &w, 16);
#pragma unroll
                        for (int e = 0; e < kE; ++e) if (n1 + e <= last_b) p[e] = v[e];
                    }
                }
                p += kRows * G.ldy;
            }
        }
    };
    if (G.out == IGCN_DTYPE_F32) put(static_cast<float *>(G.y));
    else if (G.out == IGCN_DTYPE_BF16) put(static_cast<__hip_bfloat16 *>(G.y));
    else put(static_cast<__half *>(G.y));
    asm volatile("" : : "v"(soon));                           // (or the load would not be made)
}

template <int TM, int TN, int WM, int WN, int STAGES, bool BY_DEPTH = false> static int tiles_launch(const GemmArgs &G, hipStream_t st)
{
    TileArgs T;
    T.g = G;
    T.tiles_m = (G.m + TM - 1) / TM;
    T.tiles_n = (G.n + TN - 1) / TN;
    constexpr int64_t kMostTiles = ((int64_t)1 << 32) / (64 * WM * WN) - 8;      // a launch has fewer than 2^32 threads
    if (T.tiles_m > kMostTiles / T.tiles_n) return IGCN_E_SHAPE;
    T.per_xcd = (T.tiles_m * T.tiles_n + 7) / 8;
    T.asks_ahead = i8_asks_ahead(G.m, G.n, G.k, G.out == IGCN_DTYPE_F32);
    const bool direct = i8_direct(reinterpret_cast<uintptr_t>(G.a), reinterpret_cast<uintptr_t>(G.b), G.lda, G.ldb, G.k);
    auto launch = [&](auto *kernel, int most) {
        int64_t stages = (G.k + kDepth - 1) / kDepth;
        stages = stages < most ? stages : most;
        size_t ring = (size_t)stages * (TM + TN) * kDepth;
        const size_t strips = WM * WN * 32 * (TN / WN * 4 + 16);
        if (ring < strips) ring = strips;
        if (BY_DEPTH && ring < kExchanged) ring = kExchanged;
        const size_t lds = (TM + 2 * TN) * 4 + ring;
        if (lds > 65536) {                                       // (once would do; it is a host call of well under a microsecond)
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
            if (e != hipSuccess) return (int)e;
        }
        hipLaunchKernelGGL(kernel, dim3((unsigned)(8 * T.per_xcd)), dim3(64 * WM * WN), lds, st, T);
        return launch_status();
    };
    return direct ? launch(tiles_i8_kernel<TM, TN, WM, WN, STAGES, true, BY_DEPTH>, STAGES)
                  : launch(tiles_i8_kernel<TM, TN, WM, WN, 2, false, BY_DEPTH>, 2);
}

// ---- a few rows of a ------------------------------------------------------------------------------------------------------------------
// Bound by the bytes of b, each used once, or by the way through the depth where neither side has many: no tile is worth staging.  A wave
// takes 16 rows of b as the matrix instruction's first operand straight from memory (v_mfma_i32_16x16x64_i8: lane l holds row l % 16, 16 bytes
// of depth at 16 (l / 16)) and up to 16 rows of a, which stay in L2, as the second.  KEEP steps' loads are under way while the ones before are
// multiplied.

// A lane's row of either side.  BYTES: rows at any byte.  The memory system takes 16 bytes from a multiple of 4 at full speed, from
// elsewhere at half of it (1 row against 16384 x 4095: 31 us, this way 15): a lane loads the five words around its 16 bytes and shifts them
// into place; the first and the last row of b, whose words may reach over its ends, are loaded as they are.  What is behind a row's end
// meets zeros of a.
template <bool BYTES> struct Row {
    const int8_t *p;
    int off, last, more;                                         // of the row behind a multiple of 4; the last piece's place; to the fifth word
    struct Piece { i32x4 v; int fifth; };
    __device__ __forceinline__ void at_row(const int8_t *side, int64_t ld, int64_t r, int64_t rows, int k)      // (rows past the end: the last one)
    {
        r = min(r, rows - 1);
        const bool inner = BYTES && r > 0 && r < rows - 1;
        p = side + r * ld;
        off = inner ? (int)(reinterpret_cast<uintptr_t>(p) & 3) : 0;
        last = inner ? (k + 3) / 4 * 4 - 16 : k - 16;
        more = inner ? 16 : 0;
        p -= off;
    }
    __device__ __forceinline__ Piece load(int at) const          // depth `at` on; behind the row's end its last 16 codes (a row of 16 and more)
    {
        const int8_t *q = p + min(at, last);
        Piece c;
        c.v = load16(q);
        if constexpr (BYTES) c.fifth = *reinterpret_cast<const int_any *>(q + more);
        return c;
    }
    __device__ __forceinline__ i32x4 codes(const Piece &c) const
    {
        i32x4 w = c.v;
        if constexpr (BYTES) {
            const int five[5] = {c.v[0], c.v[1], c.v[2], c.v[3], c.fifth};
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (int)__builtin_amdgcn_alignbyte((uint32_t)five[i + 1], (uint32_t)five[i], (uint32_t)off);
        }
        return w;
    }
    __device__ __forceinline__ i32x4 in_place(i32x4 w, int at) const { return behind(w, max(at - last, 0)); }      // of the last, broken step
    __device__ __forceinline__ i32x4 short_row(int at, int k) const { return load16(p + off, at, k); }             // a row of fewer than 16
};

// 16 MG rows of a, TILES x 16 rows of b a workgroup.  Its four waves take a quarter of the depth each and add their sums up in LDS (whole
// numbers: in any order), which fills the card where b has few rows and a wave's loads where they are long.  Rows of a come from L2 like
// those of b from memory, no barrier until the end: laid out in LDS first, 8 rows against 4096 x 8192 took 17.4 us, this way 9.5.
template <int MG, int TILES, bool BYTES>
__global__ __launch_bounds__(kBlock) void stream_i8_kernel(const GemmArgs G)
{
    constexpr int KEEP = 4;
    __shared__ int sums[MG * TILES * 4 * 16 * 17];               // [group of a, tile, wave][row of a][17]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at_lane = 16 * (lane >> 4), k = (int)G.k;
    const int steps = (k + kStep - 1) / kStep, whole = k / kStep, from = steps * wave / 4, to = steps * (wave + 1) / 4;
    const int64_t tile0 = (int64_t)blockIdx.x * TILES, row0 = (int64_t)blockIdx.y * 16 * MG;
    Row<BYTES> row[TILES];
    Row<BYTES> row_a[MG];
#pragma unroll
    for (int t = 0; t < TILES; ++t) row[t].at_row(G.b, G.ldb, (tile0 + t) * 16 + (lane & 15), G.n, k);
#pragma unroll
    for (int g = 0; g < MG; ++g) row_a[g].at_row(G.a, G.lda, row0 + 16 * g + (lane & 15), G.m, k);
    typename Row<BYTES>::Piece v[KEEP][TILES], x[KEEP][MG];
    i32x4 acc[MG][TILES];
#pragma unroll
    for (int g = 0; g < MG; ++g)
#pragma unroll
        for (int t = 0; t < TILES; ++t) acc[g][t] = i32x4{0, 0, 0, 0};
    auto load = [&](int s) {                                     // steps s ... s + KEEP - 1; behind the wave's last one that one again
#pragma unroll
        for (int u = 0; u < KEEP; ++u) {
            const int at = min(s + u, to - 1) * kStep + at_lane;
#pragma unroll
            for (int t = 0; t < TILES; ++t) v[u][t] = row[t].load(at);
#pragma unroll
            for (int g = 0; g < MG; ++g) x[u][g] = row_a[g].load(at);
        }
    };
    auto multiply = [&](const i32x4 (&w)[TILES], const i32x4 (&y)[MG]) {
#pragma unroll
        for (int g = 0; g < MG; ++g)
#pragma unroll
            for (int t = 0; t < TILES; ++t) acc[g][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t], y[g], acc[g][t], 0, 0, 0);
    };
    if (k >= 16) {
        if (from < to) load(from);
        for (int s = from; s < to; s += KEEP) {
            i32x4 w[KEEP][TILES], y[KEEP][MG];
#pragma unroll
            for (int u = 0; u < KEEP; ++u) {
#pragma unroll
                for (int t = 0; t < TILES; ++t) w[u][t] = row[t].codes(v[u][t]);
#pragma unroll
                for (int g = 0; g < MG; ++g) y[u][g] = row_a[g].codes(x[u][g]);
            }
            if (s + KEEP < to) load(s + KEEP);                   // the next ones while these are multiplied
#pragma unroll
            for (int u = 0; u < KEEP; ++u)
                if (s + u < to) {
                    if (s + u >= whole) {
                        const int at = (s + u) * kStep + at_lane;
#pragma unroll
                        for (int t = 0; t < TILES; ++t) w[u][t] = row[t].in_place(w[u][t], at);
#pragma unroll
                        for (int g = 0; g < MG; ++g) y[u][g] = first(row_a[g].in_place(y[u][g], at), k - at);
                    }
                    multiply(w[u], y[u]);
                }
        }
    } else if (from < to) {
        i32x4 w[TILES], y[MG];
#pragma unroll
        for (int t = 0; t < TILES; ++t) w[t] = row[t].short_row(at_lane, k);
#pragma unroll
        for (int g = 0; g < MG; ++g) y[g] = row_a[g].short_row(at_lane, k);
        multiply(w, y);
    }
    const int mine = lane & 15, quarter = lane >> 4;             // lane l holds rows of b 4 (l / 16) + i, row l % 16 of a
#pragma unroll
    for (int g = 0; g < MG; ++g)
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[(((g * TILES + t) * 4 + wave) * 16 + mine) * 17 + 4 * quarter + i] = acc[g][t][i];
    __syncthreads();
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
#pragma unroll
    for (int g = 0; g < MG; ++g)
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const int64_t n = (tile0 + t) * 16 + c;
            const int64_t at = row0 + 16 * g + r;
            if (n < G.n && at < G.m) {
                int sum = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) sum += sums[(((g * TILES + t) * 4 + w) * 16 + r) * 17 + c];
                store_out(G, at, n, scaled(sum, G.sa[at], G.sb[n], G.bias != nullptr, G.bias ? G.bias[n] : 0.f));
            }
        }
}

static bool any_byte(const void *p, int64_t ld) { return i8_any_byte(reinterpret_cast<uintptr_t>(p), ld); }
static bool fits_launch(int64_t blocks) { return blocks < ((int64_t)1 << 32) / kBlock; }       // of kBlock threads: 2^32 in all

template <int MG, int TILES> static int stream(const GemmArgs &G, hipStream_t st)
{
    const int64_t blocks = (G.n + 16 * TILES - 1) / (16 * TILES), groups = (G.m + 16 * MG - 1) / (16 * MG);
    if (!fits_launch(blocks) || groups > 65535) return IGCN_E_SHAPE;
    auto launch = [&](auto *kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)groups), dim3(kBlock), 0, st, G); };
    any_byte(G.a, G.lda) || any_byte(G.b, G.ldb) ? launch(stream_i8_kernel<MG, TILES, true>) : launch(stream_i8_kernel<MG, TILES, false>);
    return launch_status();
}

// The same for a few short rows in floating point (i8_quantises_on_the_way): every workgroup makes them 8-bit on the way, with the quantiser's own
// steps, and lays them out in LDS in the order the lanes read them: [16 codes of depth][row][16 bytes], rows rounded up to a power of two (lanes past
// them read another row's bytes; what they compute is not stored).  No launch, no buffer.  SHARE: as above, else every wave has TILES of its own.
struct FewArgs {
    GemmArgs g;
    const void *x;                                               // the rows of a in floating point, ldx apart
    int64_t ldx;
    int shift;                                                   // 2^shift rows of a in LDS
    int64_t jobs;                                                // of a workgroup at most: tile groups it walks (SHARE: one)
};

template <int TILES, int KEEP, bool SHARE, bool BYTES, typename X>
__global__ __launch_bounds__(kBlock) void few_rows_i8_kernel(const FewArgs F)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ float sx[kFewRows];
    const GemmArgs &G = F.g;
    const i32x4 *const xs = reinterpret_cast<const i32x4 *>(smem);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = lane >> 4, rows2 = 1 << F.shift, m = (int)G.m, k = (int)G.k;
    const int steps = (k + kStep - 1) / kStep, whole = k / kStep, from = SHARE ? steps * wave / 4 : 0, to = SHARE ? steps * (wave + 1) / 4 : steps;
    int *const sums = reinterpret_cast<int *>(smem + (int64_t)steps * kStep * rows2);         // SHARE: [wave][row of a][17]
    const int64_t tiles = (G.n + 15) / 16, group0 = (int64_t)blockIdx.x * F.jobs * (SHARE ? 1 : 4) + (SHARE ? 0 : wave);
    static_assert(!SHARE || TILES == 1, "one tile's sums");

    Row<BYTES> row[TILES];
    typename Row<BYTES>::Piece v[KEEP][TILES];
    i32x4 acc[TILES];
    auto rows_of = [&](int64_t tile0) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) row[t].at_row(G.b, G.ldb, (tile0 + t) * 16 + (lane & 15), G.n, k);
    };
    auto load = [&](int s) {
#pragma unroll
        for (int u = 0; u < KEEP; ++u)
#pragma unroll
            for (int t = 0; t < TILES; ++t) v[u][t] = row[t].load(min(s + u, to - 1) * kStep + 16 * quarter);
    };
    rows_of(group0 * TILES);
    bool loaded = k >= 16 && from < to && group0 * TILES < tiles;
    if (loaded) load(from);                                      // the first loads, before anything else

    constexpr int E = Chunk<X>::kValues;
    for (int r = wave; r < m; r += 4) {
        const X *from_x = static_cast<const X *>(F.x) + r * F.ldx;
        Largest<X> most;
        for (int at = lane * E; at < k; at += 64 * E) { Chunk<X> c; c.load(from_x + at, k - at); most.of(c); }
        uint32_t big = most.bits();
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, off));
        const RowScale s(big);
        if (lane == 0) sx[r] = s.s;
        for (int at = lane * E; at < steps * kStep; at += 64 * E) {
            Chunk<X> c;
            uint32_t w[E / 4];
            c.load(from_x + at, k - at);
            pack_codes<X>(w, c, s);
            __builtin_memcpy(smem + ((at >> 4) * rows2 + r) * 16 + (at & 15), w, E);
        }
    }
    __syncthreads();

    for (int64_t job = 0; job < F.jobs; ++job) {
        const int64_t tile0 = (group0 + job * (SHARE ? 1 : 4)) * TILES;
        if (SHARE ? tile0 >= tiles : tile0 - (int64_t)wave * TILES >= tiles) break;          // (the same for the whole workgroup)
        if (job) rows_of(tile0);
#pragma unroll
        for (int t = 0; t < TILES; ++t) acc[t] = i32x4{0, 0, 0, 0};
        auto multiply = [&](const i32x4 (&w)[TILES], int s) {
            const i32x4 xv = xs[(s * 4 + quarter) * rows2 + (lane & 15 & (rows2 - 1))];
#pragma unroll
            for (int t = 0; t < TILES; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[t], xv, acc[t], 0, 0, 0);
        };
        if (k >= 16) {
            if (from < to && !loaded) load(from);
            loaded = false;
            for (int s = from; s < to; s += KEEP) {
                i32x4 w[KEEP][TILES];
#pragma unroll
                for (int u = 0; u < KEEP; ++u)
#pragma unroll
                    for (int t = 0; t < TILES; ++t) w[u][t] = row[t].codes(v[u][t]);
                if (s + KEEP < to) load(s + KEEP);
#pragma unroll
                for (int u = 0; u < KEEP; ++u)
                    if (s + u < to) {
                        if (s + u >= whole) {
#pragma unroll
                            for (int t = 0; t < TILES; ++t) w[u][t] = row[t].in_place(w[u][t], (s + u) * kStep + 16 * quarter);
                        }
                        multiply(w[u], s + u);
                    }
            }
        } else if (from < to) {
            i32x4 w[TILES];
#pragma unroll
            for (int t = 0; t < TILES; ++t) w[t] = row[t].short_row(16 * quarter, k);
            multiply(w, from);
        }
        if constexpr (SHARE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[(wave * 16 + (lane & 15)) * 17 + 4 * quarter + i] = acc[0][i];
            __syncthreads();
            const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
            const int64_t n = tile0 * 16 + c;
            if (n < G.n && r < m) {
                int sum = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) sum += sums[(w * 16 + r) * 17 + c];
                store_out(G, r, n, scaled(sum, sx[r], G.sb[n], G.bias != nullptr, G.bias ? G.bias[n] : 0.f));
            }
        } else {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const int r = lane & 15;
                const int64_t n0 = (tile0 + t) * 16 + 4 * quarter;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (r < m && n0 + i < G.n)
                        store_out(G, r, n0 + i, scaled(acc[t][i], sx[r], G.sb[n0 + i], G.bias != nullptr, G.bias ? G.bias[n0 + i] : 0.f));
            }
        }
    }
}

template <typename X> static int few_rows(FewArgs F, hipStream_t st)
{
    const int64_t steps = (F.g.k + kStep - 1) / kStep, tiles = (F.g.n + 15) / 16;
    F.shift = 0;
    while ((1 << F.shift) < F.g.m) ++F.shift;
    const bool share = i8_shares_depth(F.g.n);
    constexpr int kOwn = 4;
    const int64_t per = share ? 1 : 4 * kOwn, groups = (tiles + per - 1) / per;
    // a workgroup that lays the rows of a out once and walks several groups with them: as many as keep 2 048 workgroups busy
    F.jobs = (groups + 2047) / 2048;
    const int64_t blocks = (groups + F.jobs - 1) / F.jobs;
    const size_t lds = ((size_t)steps * kStep << F.shift) + (share ? 4 * 16 * 17 * 4 : 0);    // (kFusedValues, rounded up twice: well under 64 KiB)
    const bool bytes = any_byte(F.g.b, F.g.ldb);
    auto launch = [&](auto *kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kBlock), lds, st, F); };
    if (share) bytes ? launch(few_rows_i8_kernel<1, 4, true, true, X>) : launch(few_rows_i8_kernel<1, 4, true, false, X>);
    else bytes ? launch(few_rows_i8_kernel<kOwn, 1, false, true, X>) : launch(few_rows_i8_kernel<kOwn, 1, false, false, X>);
    return launch_status();
}

static int product(const GemmArgs &G, hipStream_t st)
{
    switch (i8_way(G.m, G.n, G.k, G.lda, G.ldb, G.out == IGCN_DTYPE_F32)) {
    case I8Way::kStream: return stream<1, 1>(G, st);
    case I8Way::kStreamTwoTiles: return stream<1, 2>(G, st);
    case I8Way::kStreamTwoGroups: return stream<2, 1>(G, st);
    case I8Way::kTiles64x128: return tiles_launch<64, 128, 2, 4, 2>(G, st);
    case I8Way::kTiles256: return tiles_launch<256, 256, 2, 4, 2>(G, st);
    case I8Way::kTiles128Deep: return tiles_launch<128, 128, 2, 4, 3>(G, st);
    case I8Way::kTiles128: return tiles_launch<128, 128, 2, 4, 2>(G, st);
    case I8Way::kTiles64ByDepth: return tiles_launch<64, 64, 2, 2, 4, true>(G, st);
    case I8Way::kTiles64: return tiles_launch<64, 64, 2, 2, 4>(G, st);
    case I8Way::kApart: break;
    }
    constexpr int64_t kMost = 65535 * 32;                        // rows of a in a launch
    const int64_t size = G.out == IGCN_DTYPE_F32 ? 4 : 2;
    for (int64_t at = 0; at < G.m; at += kMost) {
        GemmArgs Q = G;
        Q.a += at * G.lda;
        Q.sa += at;
        Q.y = static_cast<char *>(G.y) + at * G.ldy * size;
        Q.m = G.m - at < kMost ? G.m - at : kMost;
        const int rc = stream<2, 1>(Q, st);
        if (rc != IGCN_OK) return rc;
    }
    return IGCN_OK;
}

static int check_product(const float *sa, const int8_t *b, int64_t ldb, const float *sb, const float *bias, int64_t m, int64_t n, int64_t k,
                         const void *y, int32_t dtype, int64_t ldy)
{
    if (!dtype_ok(dtype)) return IGCN_E_RANGE;
    if (m < 0 || n < 0 || k < 0 || ldb < k || ldy < n) return IGCN_E_SHAPE;
    if (k > IGCN_MAX_I8_DEPTH) return IGCN_E_RANGE;
    if (m == 0 || n == 0) return IGCN_OK;
    if (!sb || !y || (k > 0 && !b)) return IGCN_E_NULL;
    const uintptr_t vectors = reinterpret_cast<uintptr_t>(sa) | reinterpret_cast<uintptr_t>(sb) | reinterpret_cast<uintptr_t>(bias);
    if (misaligned(y, dtype) || (vectors & 3)) return IGCN_E_ALIGN;
    return IGCN_OK;
}

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
    return i8_quantises_on_the_way(m, INT64_MAX, k) ? 0 : up16(m * up16(k)) + 4 * m;
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
    if (i8_quantises_on_the_way(m, n, k)) {
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
