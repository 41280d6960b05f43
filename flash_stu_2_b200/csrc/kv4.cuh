// The ring cache in 4 bits: its layout, and how a number gets into it.
//
// A ring of one tensor (keys or values) is [B][Hk] runs of bytes: slots rows of width / 2 bytes, and behind them slots x pieces scales of 4
// bytes.  width is the head dimension rounded up to 32, 64 or 128; a row of more than 64 dimensions is two pieces, the first 64 and the rest.
// A word of a row holds 8 numbers, the first in the lowest bits: word i of a row of one piece dimensions 8 i .. 8 i + 7, word 2 i + p of a row of
// two those of piece p.  (So the words that one lane of the attention kernel takes from both pieces lie side by side.)  A scale is two bf16, the piece's lowest value and
// above it the step: n stands for lowest + n step, which is exact but for one rounding.
//
// lowest is the minimum rounded down and step (maximum - lowest) / 15 rounded up, so that all values lie between 0 and 15 steps and none is off by
// more than half of one (and its rounding in fp32).  Both in bf16: 4 bytes for each 64 values, 4.5 bits a value; the rounding costs at most 2^-7 of the step and
// 2^-8 of the lowest value / 15.  A piece that holds an infinity or a NaN, or whose range passes fp32's, stands for NaN.
#pragma once
#include "common.cuh"

namespace kv4 {

__host__ __device__ __forceinline__ int width_of(int hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : 128; }
__host__ __device__ __forceinline__ int pieces_of(int hd) { return hd > 64 ? 2 : 1; }
__host__ __device__ __forceinline__ long long head_bytes(int hd, int slots) { return (long long)slots * (width_of(hd) / 2 + 4 * pieces_of(hd)); }

__device__ __forceinline__ uint32_t bf16_down(float x) {   // the bits of the nearest bf16 that is not above x, as an fp32's
  const uint32_t u = __float_as_uint(x), cut = u & 0xffff0000u;
  return u != cut && (int)u < 0 ? cut + 0x10000u : cut;
}
__device__ __forceinline__ uint32_t bf16_up(float x) {
  const uint32_t u = __float_as_uint(x), cut = u & 0xffff0000u;
  return u != cut && (int)u >= 0 ? cut + 0x10000u : cut;
}

__device__ __forceinline__ float min_nan(float a, float b) {   // NaN where one is
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Eight lanes hold a piece, x[0 .. 7] each (`there`: whether the head has these dimensions): the word of this lane's and the piece's scale.
// Called by whole warps.  Every operation is one rounding to fp32, none contracted with another.  Adding 1.5 2^23 rounds to the nearest whole number,
// ties to even, and leaves it in the lowest bits; none is below 0 or above 15, since lowest is rounded down and the step up.
__device__ __forceinline__ void quantize(const float* x, bool there, uint32_t& word, uint32_t& scale) {
  float lo = there ? x[0] : INFINITY, hi = there ? x[0] : -INFINITY;
#pragma unroll
  for (int e = 1; e < 8; e++) {
    lo = there ? min_nan(lo, x[e]) : lo;
    hi = there ? max_nan(hi, x[e]) : hi;
  }
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const float low = __uint_as_float(bf16_down(lo + 0.f));   // (+ 0: zeros without a sign)
  const float spread = (hi - low) + 0.f;
  float step = __uint_as_float(bf16_up(spread * (1.f / 15.f)));
  if (step > 0.f) step = fmaxf(step, 1.17549435e-38f);      // 2^-126: its reciprocal is finite
  const bool bad = !(fabsf(low) < INFINITY) || !(spread < INFINITY) || !(step < INFINITY);
  const float inv = step > 0.f ? 1.f / step : 0.f;
  word = 0;
#pragma unroll
  for (int e = 7; e >= 0; e--) word = (word << 4) + __float_as_uint(__fadd_rn(__fmul_rn(x[e] - low, inv), 12582912.f));   // 0x4b400000 + n
  word -= 0x3f400000u;   // the sum of 0x4b400000 << 4 e
  if (!there || bad) word = 0;
  scale = bad ? 0x7fc0u : __float_as_uint(low) >> 16 | (__float_as_uint(step) & 0xffff0000u);
}

// 8 values of a row of qkv as fp32; VEC: they lie on the 16-byte grid.
template <bool VEC> __device__ __forceinline__ void load8(const float* p, float* x) {
  if (VEC) {
    load_vec(p, x);
    load_vec(p + 4, x + 4);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = p[e];
  }
}
template <bool VEC> __device__ __forceinline__ void load8(const bf16* p, float* x) {
  if (VEC) {
    load_vec(p, x);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = Elem<bf16>::to_f(p[e]);
  }
}

// Where the word of dimensions 64 piece + 8 i .. + 7 of a row lies, in words.
__device__ __forceinline__ int word_at(int i, int piece, int pieces) { return i * pieces + piece; }

// Slot of the token at position t.  (A position that no sequence has, below 0, still falls into the ring.)
__device__ __forceinline__ int slot_of(int t, int slots) { return (int)((unsigned)t % (unsigned)slots); }

// One thread of each CTA, behind a barrier that all of the CTA's threads pass once they have read the positions: whether the CTA is the last, which moves the positions
// on.  Release keeps each CTA's reading ahead of its arrival, acquire the last one's writing behind all arrivals.
__device__ __forceinline__ bool last_to_arrive(int* counter, int ctas) {
  int before;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before == ctas - 1;
}

inline int geometry(int B, int H, int Hk, int hd, int slots, int dtype) {
  if (dtype != STU_F32 && dtype != STU_BF16) return STU_ERR_DTYPE;
  if (B <= 0 || Hk <= 0 || H < Hk || H % Hk || hd <= 0 || slots <= 0 || slots % 16 || slots > 1 << 24) return STU_ERR_SHAPE;   // (offsets within a head's run fit 32 bits)
  if (hd % 8 || hd > 128) return STU_ERR_UNSUPPORTED;
  return STU_OK;
}

}  // namespace kv4
