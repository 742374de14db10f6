// Device helpers of the 8-bit (e4m3) cache, shared by its write, its read-back and its decode attention.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace fs {

// Slot -> block column and place in the block. Slots below 2^32 (all but the longest caches) take a 32-bit division,
// a tenth of the 64-bit one's instructions.
__device__ __forceinline__ void split_slot(int64_t slot, int64_t block_size, int64_t& col, int64_t& in) {
  if ((static_cast<uint64_t>(slot) | static_cast<uint64_t>(block_size)) >> 32 == 0) {
    const uint32_t s = static_cast<uint32_t>(slot), b = static_cast<uint32_t>(block_size), c = s / b;
    col = c;
    in = s - c * b;
  } else {
    col = slot / block_size;
    in = slot - col * block_size;
  }
}

// Bits of |x|: as integers they order like the values, with infinity above every number and NaN above infinity, so a
// maximum over them does not lose a NaN.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Scale of a row whose largest |x| has the bits `top`: max(|x| / 448, 2^-126), as a product with 1 / 448 (off by 2^-23 of
// itself at most: that constant's rounding and the product's); infinity and NaN stay (an fmaxf would drop the NaN).
__device__ __forceinline__ float row_scale(uint32_t top) {
  const float s = __uint_as_float(top) * (1.f / 448.f);
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;
}
// 1 / scale, off by two steps, 2^-22 of it, at most (scales lie in 2^-126 .. 2^120; infinity gives 0, NaN itself). The
// rounded reciprocal costs the fp32 write 10 % (8192 tokens of 32 + 8 + 8 heads of 128: 54.6 -> 60.3 us), a rounded quotient
// for each value the bf16 one 20 % (16 x 2048 tokens: 115 -> 155).
__device__ __forceinline__ float inverse(float scale) { return __fdividef(1.f, scale); }

// Two values as e4m3 codes, nearest even, saturating: lo in bits 0-7, hi in bits 8-15.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// The values of two codes as a pair of halves (exact: e4m3 has 4 significant bits and exponents -9..8).
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(codes));
  return r;
}

__device__ __forceinline__ float e4m3_to_f(uint8_t code) {
  const uint32_t h = e4m3x2_to_half2(code);
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xffffu)));
}

}  // namespace fs
