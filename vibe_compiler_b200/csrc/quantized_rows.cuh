// Rows of a KV head held in four bits: what the kernels that write, read and attend over them share.
#pragma once

#include "kernels.h"

namespace wb200 {

__device__ __forceinline__ float quant_step(uint32_t pair, int format) { return widen_bits(pair & 0xffffu, format); }
__device__ __forceinline__ float quant_low(uint32_t pair, int format) { return widen_bits(pair >> 16, format); }
// Element i of the eight in a word of codes. The product is exact (at most 11 bits by 4), the sum is rounded once.
__device__ __forceinline__ float quant_value(uint32_t word, int i, float step, float low) {
  return fmaf(static_cast<float>((word >> (4 * i)) & 15u), step, low);
}

// The smaller of each of two pairs of 16-bit numbers, NaN where either is.
template <int kFormat>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  if constexpr (kFormat == WB200_BF16) {
    const __nv_bfloat162 m = __hmin2_nan(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
  } else {
    const __half2 m = __hmin2_nan(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&m);
  }
}

// Codes of a lane's eight elements (two to a word of `x`) and the (step, low) of their group, which is the 64 elements of the eight
// lanes of an aligned octet (lanes without elements, `live` false, take no part). All lanes of the warp.
//   low = min x,  step = (max x - low) / 15 rounded up to the type,  code = (x - low) / step rounded to the nearest
// Rounded up, fifteen steps reach the largest element: no code is clamped by more than the division's rounding, and an element is
// off by at most half a step. A code is a decision next to a border, so the quotients are the IEEE f32 ones, for all of a group by one
// reciprocal: with y = 1 / step correctly rounded, q = d y and r = d - q step exact, q + r y is d / step correctly rounded (Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", 1990; steps have 11 bits at most, so the one exception,
// a divisor of ones alone, does not occur). A group that holds an infinity or a NaN, or spans more than f32, is NaN as a whole.
template <int kFormat>
__device__ __forceinline__ uint32_t quantize8(const uint32_t (&x)[4], bool live, uint32_t *pair) {
  constexpr uint32_t kSigns = 0x80008000u, kInfinities = kFormat == WB200_BF16 ? 0x7f807f80u : 0x7c007c00u;
  uint32_t least = min2_nan<kFormat>(min2_nan<kFormat>(x[0], x[1]), min2_nan<kFormat>(x[2], x[3]));
  uint32_t most = min2_nan<kFormat>(min2_nan<kFormat>(x[0] ^ kSigns, x[1] ^ kSigns), min2_nan<kFormat>(x[2] ^ kSigns, x[3] ^ kSigns));   // negated
  uint32_t ends = min2_nan<kFormat>(__byte_perm(least, most, 0x5410), __byte_perm(least, most, 0x7632));                                // (low, -high)
  if (!live) ends = kInfinities;
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) ends = min2_nan<kFormat>(ends, __shfl_xor_sync(0xffffffffu, ends, off));
  const float low = widen_bits(ends & 0xffffu, kFormat) + 0.f;     // -0 becomes 0
  const float range = -widen_bits(ends >> 16, kFormat) - low;
  if (!(range < INFINITY)) {
    *pair = kFormat == WB200_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
    return 0;
  }
  const float wanted = __fdiv_rn(range, 15.f);
  uint32_t step_bits = narrow_bits(wanted, kFormat);
  float step = widen_bits(step_bits, kFormat);
  if (step < wanted) step = widen_bits(++step_bits, kFormat);
  *pair = step_bits | (narrow_bits(low, kFormat) << 16);
  if (step == 0.f) return 0;
  // Where the products above could leave the normal numbers, the plain division.
  const bool near_one = step > 0x1p-60f && step < 0x1p60f;
  const float inverse = __frcp_rn(step);
  constexpr uint32_t kInteger = 0x4b400000u;           // 1.5 * 2^23: a sum with it rounds to whole numbers, ties to even, in the low bits
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = widen_bits(i & 1 ? x[i >> 1] >> 16 : x[i >> 1] & 0xffffu, kFormat) - low;
    const float q = d * inverse;
    float quotient = fmaf(fmaf(-q, step, d), inverse, q);
    if (!near_one) quotient = __fdiv_rn(d, step);
    word += __float_as_uint(fminf(quotient, 15.f) + __uint_as_float(kInteger)) << (4 * i);
  }
  return word - kInteger * 0x11111111u;
}

}  // namespace wb200
