// Which kernel a product of 8-bit rows goes to: a rule on sizes, leading dimensions, alignment and the output's size alone.
// Plain C++, so that a test can ask it without a GPU.  Both sides of every threshold were measured: "m x n x k  the way chosen / the other", us a launch.
#pragma once
#include <cstdint>

namespace igcn {

constexpr int kDepth = 128;                                      // codes of depth in a stage of the tile kernel
constexpr int kStep = 64;                                        // codes of depth a matrix instruction of the streaming kernels takes
constexpr int64_t kMostApart = 1 << 23;                          // bytes between rows of a tile: 256 of them fit 31 bits
constexpr int kFewRows = 8;
constexpr int64_t kFusedValues = 4096, kFusedDepth = 512, kFusedShort = 16384;

enum class I8Way {
    kStream, kStreamTwoTiles, kStreamTwoGroups, kApart,          // stream<1, 1>, <1, 2>, <2, 1>; rows megabytes apart: <2, 1> in pieces
    kTiles64x128, kTiles256, kTiles128Deep, kTiles128, kTiles64ByDepth, kTiles64
};

inline int64_t pieces(int64_t n, int64_t by) { return (n + by - 1) / by; }

// Where rows stream and are not put together to tiles (streamed / in tiles).
// Up to 8 rows of a, unless b has many short ones:
//   8 x 16384 x 512  5.3 / 5.2     8 x 28672 x 512  8.0 / 7.0     8 x 65536 x 64  5.8 / 5.0     8 x 65536 x 1024  14.7 / 16.3
//   8 x 16384 x 8192  27 / 32
// More where one workgroup for each of 256 CUs does, which 64 x 64 tiles would not fill:
//   16 x 4096 x 4096  7.0 / 11.0   16 x 8192 x 8192  15.0 / 18.1  16 x 11008 x 8192  26.6 / 21.6
//   32 x 4096 x 4096  9.1 / 11.2   32 x 8192 x 4096  14.2 / 11.5  189 x 48 x 5391  9.1 / 20.9
//   256 x 512 x 8192  13.5 / 18.3  512 x 512 x 8192  24.3 / 17.7
inline bool i8_streams(int64_t m, int64_t n, int64_t k)
{
    if (m <= 8) return k > 11 * kStep || n <= 24576;
    if (m <= 16) return n <= 8192;
    return pieces(m, 32) * pieces(n, 16) <= 256;
}

inline I8Way i8_way(int64_t m, int64_t n, int64_t k, int64_t lda, int64_t ldb, bool out_f32)
{
    if (i8_streams(m, n, k)) {
        // 32 rows of a a workgroup where 16 would need more than one a CU: 64 x 2048 x 4096  8.3 / 10.0; not so: 33 x 1000 x 8192  10.4 / 13.7
        if (m > 16) return pieces(m, 16) * pieces(n, 16) <= 256 ? I8Way::kStream : I8Way::kStreamTwoGroups;
        // Two tiles a workgroup halve the reads of a where there is a workgroup for every CU all the same:
        //   16 x 8192 x 8192  15.0 / 17.2     not so: 16 x 4096 x 8192  10.7 / 14.1     1 x 28672 x 8192  41 / 46
        return m > 4 && n > 4096 && k >= 2048 ? I8Way::kStreamTwoTiles : I8Way::kStream;
    }
    if (lda > kMostApart || ldb > kMostApart) return I8Way::kApart;
    if (m > 64) {
        // One stage of depth: writing y is all there is, and many small waves hide it best.
        //   512 x 96421 x 64 to float32: 48, 128 x 128 tiles 57, 256 x 256 55; to bfloat16 128 x 128 tiles 30, 64 x 128 38
        if (k <= kDepth && out_f32) return I8Way::kTiles64x128;
        // The largest tile that still makes nearly a workgroup for each of 256 CUs: 256 x 256 reads each code half as often as 128 x 128.
        //   8192 x 8192 x 4096  258 / 298     64 such tiles, one CU of four: 512 x 8192 x 8192  90, 128 x 128 47, 64 x 64 57
        if (k > kDepth && pieces(m, 256) * pieces(n, 256) >= 200) return I8Way::kTiles256;
        // Eight waves, two to a SIMD, one reading LDS while the other multiplies (four waves: 512 x 8192 x 512  6.9 / 8.1, x 4096  27 / 28); a third
        // stage where a CU has one workgroup anyway and the depth pays for it:
        //   256 x 16384 x 8192  56 / 68     not so: 256 x 16384 x 1024  10.3 / 10.4     3000 x 3000 x 4096  58 / 69
        const int64_t middle = pieces(m, 128) * pieces(n, 128);
        if (middle >= 200) return middle <= 256 && k >= 2048 ? I8Way::kTiles128Deep : I8Way::kTiles128;
    }
    // Waves that share the depth of a 64 x 64 tile pay where a CU has one workgroup, which waits for its own products, and the depth is
    // worth the exchange:
    //   300 x 700 x 2048  7.7 / 8.5      300 x 700 x 4096  11.2 / 13.5    180 x 3000 x 2048  7.9 / 8.6    180 x 3000 x 8192  18.7 / 23.3
    //   b not in a cache: 64 x 12000 x 2048  10.6 / 10.2                  64 x 12000 x 8192  26.2 / 26.7
    // not so:
    //   300 x 700 x 512  4.8 / 5.2       300 x 700 x 1024  6.1 / 6.1      64 x 16384 x 4096  14.7 / 14.9  40 x 30000 x 2048  13.6 / 14.0
    return k >= 2048 && pieces(m, 64) * pieces(n, 64) <= 200 ? I8Way::kTiles64ByDepth : I8Way::kTiles64;
}

// One stage of depth and 32 MB of y and more, more than the L2s hold: a tile's reads of b then queue behind the writes of y, and the first
// row of tiles asks for later rows of b ahead.  asked / not, with b not in a cache, and with b there:
//   to float32:   128 x 96421 x 64 (49 MB of y)  14.4 / 16.9, 13.1 / 12.6     512 x 96421 x 64  46 / 53, 38 / 36     2048 x 96421 x 64  191 / 211, 191 / 214
//   to bfloat16:  200 x 96421 x 64 (39 MB)  15.5 / 17.2, 14.5 / 14.0          512 x 96421 x 64  30 / 33, 27 / 27
//   smaller y:    64 x 96421 x 128 to float32 (25 MB)  10.9 / 11.0, 9.2 / 9.1   to bfloat16  9.5 / 8.4, 7.9 / 7.4     9 x 20956 x 128  4.8 / 4.0, 4.1 / 4.1
inline bool i8_asks_ahead(int64_t m, int64_t n, int64_t k, bool out_f32) { return k > 0 && k <= kDepth && m * n >= (out_f32 ? 1 << 23 : 1 << 24); }

// Rows that start at, and are apart by, multiples of 16 bytes, a depth of whole 16-byte pieces: memory to LDS without registers
inline bool i8_direct(uintptr_t a, uintptr_t b, int64_t lda, int64_t ldb, int64_t k)
{
    return ((a | b | (uintptr_t)lda | (uintptr_t)ldb | (uintptr_t)k) & 15) == 0;
}
inline bool i8_any_byte(uintptr_t p, int64_t ld) { return ((p | (uintptr_t)ld) & 3) != 0; }

// A few short rows in floating point are made 8-bit inside the product while that is less work than a launch (and from the host it is one less):
//   1 x 96421 x 64  6.7 / 8.8     1 x 96421 x 512  16.8 / 20.2    1 x 4000 x 1024  5.1 / 7.1     8 x 4000 x 512  6.5 / 7.5
//   not so: 1 x 96421 x 1024  21.4 / 26.8     1 x 16384 x 1024 (the limit)  8.8 / 8.0     8 x 4000 x 1024  7.4 / 8.7
inline bool i8_quantises_on_the_way(int64_t m, int64_t n, int64_t k)
{
    return m <= kFewRows && m * k <= kFusedValues && k <= (n <= kFusedShort ? 2 * kFusedDepth : kFusedDepth);
}
// ... there: whether a workgroup's waves share a tile's depth, or have tiles of their own, which starts fewer workgroups where b has many short rows
// (more than 2048 tiles have at most 8 steps):
//   8 x 16384 x 512  5.8 / 10.2     own: 8 x 50000 x 256  9.1 / 12.4     8 x 96421 x 64  7.4 / 10.0
inline bool i8_shares_depth(int64_t n) { return pieces(n, 16) <= 2048; }

}  // namespace igcn
