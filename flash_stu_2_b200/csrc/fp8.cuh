// Rows of 8-bit values with a power-of-two scale for each 128 of a row: what the kernels that write and read them share.
//
// Values are e4m3 (largest 448, one NaN, no infinity), rows padded with zeros to whole blocks of 128.  A block's scale is 2^e with the smallest
// whole e >= -127 for which its largest finite magnitude is at most 448 * 2^e, held as the byte e + 127 (E8M0).  A power of two makes every
// scaling exact and is what the tensor core applies by itself (kind::mxf8f6f4).  Scales of 128 rows x 4 blocks are 512 bytes in the
// order that the copy into tensor memory takes: byte (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4.  Rows and blocks that fill up such a
// piece have byte 0.
#pragma once
#include "common.cuh"

namespace fp8 {

constexpr int BLOCK = 128;    // values of a row that share a scale
constexpr int PIECE = 512;    // bytes of a piece of scales, and columns that its four blocks cover

__host__ __device__ __forceinline__ int blocks_of(int cols) { return (cols + BLOCK - 1) / BLOCK; }
__host__ __device__ __forceinline__ int groups_of(int cols) { return (cols + PIECE - 1) / PIECE; }

// Offset of the four scales of `row` in group g (block 4 g first).
__device__ __forceinline__ size_t scale_word(int row, int g, int groups) {
  return ((size_t)(row >> 7) * groups + g) * PIECE + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

constexpr uint32_t INF_BITS = 0x7f800000u;

// Scale byte of a block from the bits of its largest finite magnitude m * 2^(E-127), 1 <= m < 2: 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const int b = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b > 0 ? b : 0;
}
// 2^-e of a scale byte
__device__ __forceinline__ float inverse_scale(uint32_t b) { return __uint_as_float((254u - b) << 23); }

// Four values to e4m3, nearest even, the first in the lowest byte.
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// Infinity has no e4m3 value (the conversion would saturate): it becomes NaN, as NaN does.
__device__ __forceinline__ float nan_unless_finite(float v) { return magnitude(v) < INF_BITS ? v : __uint_as_float(0x7fffffffu); }

// gelu_tanh(x) = x / (1 + exp(-t)), t = 2 k0 (x + k1 x^3).  Relative error below (5 + 4.2 |t|) 2^-23 where t is negative (an exponential takes its argument's error
// as it is: 3 |t| of that are the roundings of t, 1.2 |t| the hardware exponential's own), 5 * 2^-23 where it is positive.  The form with tanh in fp32 cancels where x is
// negative and is off by more from x = -1 on.  Gates of -6 to -2 whose sums are exact: none of 16.8 million 8-bit results is another than in 64 bits, 9 % with tanh.  The
// 2^-11 of the hardware tanh, which the bf16 epilogues take, would move one in 60 of the 8-bit results to its neighbour.
__device__ __forceinline__ float gelu(float x) {
  const float t = 1.5957691216057308f * x * fmaf(0.044715f * x, x, 1.0f);
  return __fdividef(x, 1.0f + __expf(-t));
}

}  // namespace fp8
