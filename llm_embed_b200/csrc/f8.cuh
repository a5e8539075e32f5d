// Eight-bit (e4m3) operands with a power-of-two scale for each block of 128
// values: the rule shared by the quantiser (f8_quant.cu) and the products
// that quantise their activations themselves (f8_gemm.cu).
//
// scale = 2^ceil(log2(amax / 448)), the smallest power of two that brings the
// block's largest magnitude to 448 (e4m3's largest value) or less.  Dividing
// by it is exact, so the one rounding of a value is that to e4m3 (at most
// 2^-4 of the value, or 2^-10 of the scale for the smallest), and every path
// gives the same bytes.  An all-zero block has scale 1; a block that holds a
// NaN or an infinity has scale NaN, so every product with it is NaN.  Scales
// are not smaller than 2^-126.
#pragma once
#include "elem.cuh"

namespace le {
namespace f8 {

constexpr int BLOCK = 128;

// Scale of a block whose largest magnitude has the bits `amax` (sign
// cleared; bits compare like the values, NaN above infinity), and its inverse.
__device__ __forceinline__ float block_scale(uint32_t amax, float* inv) {
  const uint32_t be = amax >> 23;  // 1.f x 2^(be - 127); 448 = 1.75 x 2^8
  int sb = (int)be - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  sb = sb < 1 ? 1 : sb;
  if (amax == 0) sb = 127;
  uint32_t s = (uint32_t)sb << 23, i = (uint32_t)(254 - sb) << 23;
  if (be == 255) s = i = 0x7fc00000u;
  *inv = __uint_as_float(i);
  return __uint_as_float(s);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Four values, already divided by their scale, as e4m3 bytes (v0 lowest).
__device__ __forceinline__ uint32_t pack_e4m3(float v0, float v1, float v2, float v3) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v1), "f"(v0));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v3), "f"(v2));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

}  // namespace f8
}  // namespace le
