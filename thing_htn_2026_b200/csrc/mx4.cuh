// Matrices in microscaled 4-bit floating point, as the kernels of this library hold them.
//
// A row is cut into blocks of 32 entries.  A block has a scale 2^(b - 127), held as the byte b (255: the block is not a
// number), and its entries are 4-bit floats: a sign, two bits of exponent, one of mantissa, the magnitudes
// 0, 1/2, 1, 3/2, 2, 3, 4, 6 for the codes 0 to 7.
//
//   codes   [rows][padded / 2] bytes, two entries a byte, the first in the low half; padded = columns rounded up to 128
//   scales  [ceil(rows / 128)][padded / 128][512] bytes: what 128 rows need for 128 columns, in the order in which tensor memory
//           takes it: byte (row % 32) * 16 + (row % 128 / 32) * 4 + (column % 128 / 32)
//
// Behind the last column both are zero (0 * 2^-127).  Scales of rows behind the last one are whatever they were: every result
// row depends on its own row's scales alone.
#pragma once

#include "common.cuh"

constexpr int kMx4Block = 32;       // entries of a scale
constexpr int kMx4Atom = 128;       // columns (and rows) of a piece of scales
constexpr int kMx4AtomBytes = 512;

__host__ __device__ __forceinline__ long long mx4_padded(long long columns) { return (columns + kMx4Atom - 1) / kMx4Atom * kMx4Atom; }

// where the four scale bytes of `row` for columns [128 atom, 128 atom + 128) begin; atoms = padded / 128
__host__ __device__ __forceinline__ long long mx4_scale_at(long long row, long long atom, long long atoms) {
    const long long r = row & 127;
    return ((row >> 7) * atoms + atom) * kMx4AtomBytes + (r & 31) * 16 + (r >> 5) * 4;
}

// 2^(b - 127) as a float32; NaN for 255
__device__ __forceinline__ float mx4_scale(uint32_t b) {
    return __uint_as_float(b == 0 ? 0x00400000u : b == 255 ? 0x7fffffffu : b << 23);
}

// The magnitude and sign of a code as a float32: its three low bits are the exponent and mantissa of a float32 that is 2^126 times too small.
__device__ __forceinline__ float mx4_value(uint32_t code) {
    return __uint_as_float((code & 7) << 22 | (code & 8) << 28) * 8.507059173023462e37f;      // 2^126
}

// Division of numbers below 2^31 by a divisor that the host knows: n / d = (hi(n m) + n) >> l with 2^(l-1) < d <= 2^l and
// m = floor(2^32 (2^l - d) / d) + 1.
struct Mx4Divisor {
    uint32_t d, m, l;
    explicit Mx4Divisor(uint32_t divisor) : d(divisor), l(0) {
        while ((1ull << l) < d) ++l;
        m = (uint32_t)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
    }
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return (__umulhi(n, m) + n) >> l; }
};

// Row and piece of a unit, so many neighbouring entries, and of those STEP further on.
template <uint32_t STEP>
struct Mx4Place {
    uint32_t row, piece;
    __device__ __forceinline__ Mx4Place(uint32_t unit, const Mx4Divisor& pieces) : row(pieces.of(unit)), piece(unit - row * pieces.d) {}
    __device__ __forceinline__ void step(const Mx4Divisor& pieces) {
        piece += STEP;
        if (pieces.d >= STEP) {
            if (piece >= pieces.d) {
                piece -= pieces.d;
                ++row;
            }
        } else {
            const uint32_t more = pieces.of(piece);
            row += more;
            piece -= more * pieces.d;
        }
    }
};
