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

// The eight elements of a word of codes in order: low + code * step in the type, rounded once. A nibble behind the bits of 128 (bf16)
// or 1024 (f16) is that number and the code.
template <bool kBf16>
__device__ __forceinline__ void decode_word(uint32_t word, uint32_t step2, uint32_t low2, uint32_t (&out)[4]) {
  constexpr uint32_t kMagic = kBf16 ? 0x43004300u : 0x64006400u;
  const uint32_t upper = word >> 4;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint32_t pair = (__byte_perm(word, upper, b | (b << 4) | ((4 + b) << 8) | ((4 + b) << 12)) & 0x000f000fu) | kMagic;
    if constexpr (kBf16) {
      const uint32_t magic = kMagic;
      const __nv_bfloat162 code = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&pair), *reinterpret_cast<const __nv_bfloat162 *>(&magic));
      const __nv_bfloat162 v = __hfma2(code, *reinterpret_cast<const __nv_bfloat162 *>(&step2), *reinterpret_cast<const __nv_bfloat162 *>(&low2));
      out[b] = *reinterpret_cast<const uint32_t *>(&v);
    } else {
      const uint32_t magic = kMagic;
      const __half2 code = __hsub2(*reinterpret_cast<const __half2 *>(&pair), *reinterpret_cast<const __half2 *>(&magic));
      const __half2 v = __hfma2(code, *reinterpret_cast<const __half2 *>(&step2), *reinterpret_cast<const __half2 *>(&low2));
      out[b] = *reinterpret_cast<const uint32_t *>(&v);
    }
  }
}

// Two numbers of the type in a word, the first in its low half.
template <int kFormat>
__device__ __forceinline__ uint32_t narrow_pair(float lo, float hi) {
  if constexpr (kFormat == WB200_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
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

// a / b correctly rounded, for y = 1 / b correctly rounded: q = a y leaves the exact r = a - q b, and q + r y is the quotient
// (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990; but for divisors whose bits are all
// ones). Nothing may leave the normal numbers.
__device__ __forceinline__ float quotient_by(float a, float b, float y) {
  const float q = a * y;
  return fmaf(fmaf(-q, b, a), y, q);
}

// Codes of a lane's sixteen elements (two to a word of `x`), eight to a word, and the (step, low) of their group, which is the 64
// elements of the four lanes of an aligned quad; `live`: how many octets of the lane's elements there are (0, 1, 2). All lanes of the
// warp.
//   low = min x,  step = (max x - low) / 15 rounded up to the type,  code = (x - low) / step rounded to the nearest
// Rounded up, fifteen steps reach the largest element: no quotient rounds to sixteen, and an element is off by at most half a step.
// (Where fifteen of them would leave the type, the step is rounded down, by less than its last place, eps of it: the largest element is off
// by up to 15 eps of a step more, 0.117 in bf16, 0.0147 in f16.) A code is a decision next to a border, so the quotients are the IEEE f32
// ones. A group that holds an infinity or a NaN, or spans more than f32, is NaN as a whole.
template <int kFormat>
__device__ __forceinline__ uint2 quantize16(const uint32_t (&x)[8], int live, uint32_t *pair) {
  constexpr uint32_t kSigns = 0x80008000u, kInfinities = kFormat == WB200_BF16 ? 0x7f807f80u : 0x7c007c00u;
  uint32_t ends = kInfinities;                           // (low, -high)
#pragma unroll
  for (int o = 0; o < 2; ++o) {
    const uint32_t least = min2_nan<kFormat>(min2_nan<kFormat>(x[4 * o], x[4 * o + 1]), min2_nan<kFormat>(x[4 * o + 2], x[4 * o + 3]));
    const uint32_t most = min2_nan<kFormat>(min2_nan<kFormat>(x[4 * o] ^ kSigns, x[4 * o + 1] ^ kSigns),
                                            min2_nan<kFormat>(x[4 * o + 2] ^ kSigns, x[4 * o + 3] ^ kSigns));
    const uint32_t mine = min2_nan<kFormat>(__byte_perm(least, most, 0x5410), __byte_perm(least, most, 0x7632));
    if (o < live) ends = min2_nan<kFormat>(ends, mine);
  }
#pragma unroll
  for (int off = 2; off > 0; off >>= 1) ends = min2_nan<kFormat>(ends, __shfl_xor_sync(0xffffffffu, ends, off));
  const float low = widen_bits(ends & 0xffffu, kFormat) + 0.f;     // -0 becomes 0
  const float range = -widen_bits(ends >> 16, kFormat) - low;
  if (!(range < INFINITY)) {
    *pair = kFormat == WB200_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
    return make_uint2(0u, 0u);
  }
  const bool usual = range > 0x1p-50f && range < 0x1p50f;      // products below stay normal numbers
  const float wanted = usual ? quotient_by(range, 15.f, 1.f / 15.f) : __fdiv_rn(range, 15.f);
  uint32_t step_bits = narrow_bits(wanted, kFormat);
  float step = widen_bits(step_bits, kFormat);
  if (step < wanted) step = widen_bits(++step_bits, kFormat);
  const bool beyond = fmaf(15.f, step, low) > (kFormat == WB200_BF16 ? 0x1.fep127f : 65504.f);       // the type's largest
  if (beyond) step = widen_bits(--step_bits, kFormat);
  *pair = step_bits | (narrow_bits(low, kFormat) << 16);
  if (step == 0.f) return make_uint2(0u, 0u);
  constexpr uint32_t kInteger = 0x4b400000u;             // 1.5 * 2^23: a sum with it rounds to whole numbers, ties to even, in the low bits
  uint32_t word[2] = {0u, 0u};
  if (usual && !beyond) {
    const float inverse = __frcp_rn(step);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float d = widen_bits(i & 1 ? x[i >> 1] >> 16 : x[i >> 1] & 0xffffu, kFormat) - low;
      word[i >> 3] += __float_as_uint(quotient_by(d, step, inverse) + __uint_as_float(kInteger)) << (4 * (i & 7));
    }
  } else {
#pragma unroll
    for (int o = 0; o < 2; ++o)
#pragma unroll 1
      for (int i = 7; i >= 0; --i) {
        const uint32_t both = i < 2 ? x[4 * o] : i < 4 ? x[4 * o + 1] : i < 6 ? x[4 * o + 2] : x[4 * o + 3];
        word[o] = (word[o] << 4) + __float_as_uint(fminf(__fdiv_rn(widen_bits((both >> (16 * (i & 1))) & 0xffffu, kFormat) - low, step), 15.f) + __uint_as_float(kInteger));
      }
  }
  return make_uint2(word[0] - kInteger * 0x11111111u, word[1] - kInteger * 0x11111111u);
}

}  // namespace wb200
