// A float32 value as the sum of two half-precision parts.
#pragma once
#include <stdint.h>

namespace b200 {

// two values as (hi, hi) and (lo, lo): lo = fp16(x - hi), the difference in one mixed-precision operation
__device__ __forceinline__ void split_halves(float x, float y, uint32_t& hi, uint32_t& lo) {
  asm("{\n\t.reg .f32 r0, r1;\n\t.reg .b16 h0, h1, m;\n\t"
      "cvt.rn.f16x2.f32 %0, %3, %2;\n\t"
      "mov.b32 {h0, h1}, %0;\n\t"
      "mov.b16 m, 0xBC00;\n\t"                       // -1
      "fma.rn.f32.f16 r0, h0, m, %2;\n\t"
      "fma.rn.f32.f16 r1, h1, m, %3;\n\t"
      "cvt.rn.f16x2.f32 %1, r1, r0;\n\t}"
      : "=&r"(hi), "=r"(lo)
      : "f"(x), "f"(y));
}

}  // namespace b200
