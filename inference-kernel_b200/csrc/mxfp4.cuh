// Device conversions of the microscaled 4-bit format (mxfp4.cu describes it).
#pragma once

#include <cstdint>

#include "vec.cuh"

namespace aotk {
namespace mx {

// Codes of v[0..7] (v[0] in the low nibble), e2m1 with round to nearest even,
// saturating.
__device__ __forceinline__ uint32_t encode_e2m1x8(const float* v) {
  uint32_t w;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(w)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return w;
}

// The eight values of a word of codes (exact).
__device__ __forceinline__ void decode_e2m1x8(uint32_t w, float* v) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<__half>::unpack2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// 2^(byte - 127): the smallest is subnormal, 255 is NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  const uint32_t bits = byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23;
  return __uint_as_float(bits);
}

}  // namespace mx
}  // namespace aotk
