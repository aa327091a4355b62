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

// Codes of a lane's eight elements x and the (step, low) of their group, which is the 64 elements of the eight lanes of an aligned
// octet (lanes without elements, `live` false, take no part). All lanes of the warp.
//   low = min x,  step = (max x - low) / 15 rounded up to the type,  code = (x - low) / step rounded to the nearest
// Rounded up, fifteen steps reach the largest element: no code is clamped by more than the division's rounding, and an element is
// off by at most half a step. Division and differences are IEEE f32: a code is a decision next to a border, and a reciprocal's last
// bit would move some. A group that holds an infinity or a NaN, or spans more than f32, is NaN as a whole.
template <int kFormat>
__device__ __forceinline__ uint32_t quantize8(const float (&x)[8], bool live, uint32_t *pair) {
  float low = INFINITY, high = -INFINITY;
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    low = fminf(low, x[i]);
    high = fmaxf(high, x[i]);
    finite = finite && fabsf(x[i]) < INFINITY;
  }
  if (!live) { low = INFINITY; high = -INFINITY; finite = true; }
#pragma unroll
  for (int off = 4; off > 0; off >>= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, off));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, off));
  }
  const unsigned int bad = __ballot_sync(0xffffffffu, !finite);
  const float range = high - low;
  if (((bad >> (threadIdx.x & 24)) & 0xffu) || !(range < INFINITY)) {
    *pair = kFormat == WB200_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
    return 0;
  }
  low += 0.f;                                            // -0 becomes 0
  const float wanted = __fdiv_rn(range, 15.f);
  uint32_t step_bits = narrow_bits(wanted, kFormat);
  float step = widen_bits(step_bits, kFormat);
  if (step < wanted) step = widen_bits(++step_bits, kFormat);
  *pair = step_bits | (narrow_bits(low, kFormat) << 16);
  if (step == 0.f) return 0;
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) word |= static_cast<uint32_t>(fminf(rintf(__fdiv_rn(x[i] - low, step)), 15.f)) << (4 * i);
  return word;
}

}  // namespace wb200
