// Keys and values held in 8 bits, a scale for each block of 16 positions of a page and kv head.
//
// One layer's cache is `codes`, bytes [pages][2 (k, v)][heads][page][d], and `words`, 32 bits
// [pages][heads][page / 16][2 (k, v)].  A word's bits 0..7 are the block's exponent E, bits 16..31 mark the
// tokens of the block with a value that is no finite number.  E == 0: every value is zero.  Otherwise a value x is kept as
// u = floor(x / s) + 128 with the step s = 2^(E - 133) and read back as (u - 127.5) s, at most s / 2 away.
// E is the biased binary exponent of the block's largest finite magnitude, at least 16, so |x| < 128 s.
//
// Steps are powers of two and codes are rounded down, because then a block can take a larger value later on:
// floor(floor(x / s) / 2^n) = floor(x / (2^n s)), so shifting the codes that are there gives what the values
// would have been kept as from the start, and a block's codes do not depend on the portions that its tokens came in.
// u - 127.5 has eight significant bits: what is read back is a bfloat16 exactly.
//
// A marked token is read back as numbers that are not finite, and as nothing that reaches another token: attention
// takes its score as NaN and its value as what the finite part of it says.
#pragma once
#include "common.cuh"

namespace ptl {

constexpr int kKv8Block = 16;
constexpr int kKv8MinExponent = 16;     // 2^-111: below it steps would leave the normal numbers

// Exponent of a block whose largest finite magnitude has these bits.
__device__ __forceinline__ int kv8_exponent(uint32_t amax_bits) {
  return amax_bits == 0u ? 0 : max(kKv8MinExponent, (int)(amax_bits >> 23));
}
// Half a step, 2^(E - 134), and 0 for a block of zeros: a value is (2u - 255) times this.
__device__ __forceinline__ float kv8_half_step(int e) {
  // E - 134 reaches below the smallest normal exponent only for E < 8, which does not occur
  return e == 0 ? 0.f : __uint_as_float((uint32_t)(e - 7) << 23);
}
// 1 / step = 2^(133 - E), for E of 16 to 254 a normal number.
__device__ __forceinline__ float kv8_inverse_step(int e) { return __uint_as_float((uint32_t)(260 - e) << 23); }

// The code of a finite x, in the low byte: x / step + 1.5 * 2^23 + 128 rounded down has the whole part of x / step, rounded down, plus 128 in its
// last bits.  One rounding, so a tiny negative x counts as below 0 too.  With a step of 0 / 0 (inverse 0): 128.
__device__ __forceinline__ uint32_t kv8_code(float x, float inverse_step) { return __float_as_uint(__fmaf_rd(x, inverse_step, 12583040.0f)); }
// Four codes for steps 2^n times as large; from n = 7 on only the sign is left.
__device__ __forceinline__ uint32_t kv8_coarser(uint32_t four, int n) {
  n = min(n, 7);
  return ((four >> n) & (0x01010101u * (0xffu >> n))) + 0x01010101u * (128u - (128u >> n));
}

}  // namespace ptl
