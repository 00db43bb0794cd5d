// Block scales: the format of operands with one power-of-two scale per 128 consecutive elements of the contracted axis.
//
// An operand [rows, K] is stored as float8 (e4m3) rows of round_up(K, 128) bytes, zero past K, and one exponent byte per
// row and block of 128: the value of an element is q * 2^(byte - 127) (E8M0, what the scaled MFMAs of gfx950 take as it is).
// With 128 elements a block is one step of v_mfma_scale_f32_16x16x128_f8f6f4: the scales cost no arithmetic.
//
// The bytes lie in the order in which the MFMAs read them: block by block of K, in each round_up(rows, 128) bytes, in which
// the byte of row r is at 128 (r / 128) + 8 (r % 16) + r % 128 / 16.  A lane of an MFMA supplies the byte of row lane % 16
// of its 16-row tile, and a register's four bytes can serve four tiles: lane l finds those of the eight tiles of 128 rows in
// eight consecutive bytes.  (128 x 128 blocks of a weight repeat their byte for 128 rows: 0.8 % of the weight's bytes.)
#pragma once
#include "mi8_common.h"

namespace mi8 {
namespace block {

__host__ __device__ inline int64_t padded(int64_t n) { return (n + 127) / 128 * 128; }
// where in a group of 128 rows the byte of row r is
__device__ __forceinline__ int scale_at(int r) { return 8 * (r & 15) + (r >> 4); }

// Exponent k of the scale 2^k for a block whose largest magnitude has these bits: the largest k with amax 2^k <= 448, at most
// 120 (blocks of zeros, and of less than 2^-112).  448 is 1.75 2^8.  A block that holds an infinity or a NaN becomes NaN throughout: k is
// 0 and the factor NaN.
__device__ __forceinline__ void scale_of(uint32_t amax_bits, float& factor, uint8_t& byte)
{
    const int e = (int)(amax_bits >> 23);
    int k = 8 + 127 - e - ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    k = k < 120 ? k : 120;
    const bool finite = e < 255;
    k = finite ? k : 0;
    factor = finite ? bits_to_f32((uint32_t)(127 + k) << 23) : bits_to_f32(0x7FC00000u);
    byte = (uint8_t)(127 - k);
}

}  // namespace block
}  // namespace mi8
