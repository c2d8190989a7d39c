// Rounding to e4m3, for the kernels that store 8-bit values over a scale.
#pragma once

#include "common.h"

namespace sile {

// x / scale, correctly rounded, held to e4m3's range; NaN stays NaN.  rcp is 1 / scale,
// correctly rounded: one correction of x * rcp by its remainder is then the quotient
// (Markstein), wherever it is neither past the range, where it saturates in any case,
// nor so small that it rounds to zero, and scale is no extreme; else (rcp = 0) the division
// (a third of the kernel's instructions: with plain stores, 16382 tokens of 8 heads of 128
// take 31 us with it and 26 so).
SILE_DEV float e4m3_in(float x, float scale, float rcp) {
  float y;
  if (rcp == 0.0f) {
    y = x / scale;
  } else {
    const float q = x * rcp;
    const float exact = __builtin_fmaf(__builtin_fmaf(-q, scale, x), rcp, q);
    const float m = __builtin_fabsf(q);
    y = m < 1024.0f && m > 0x1p-12f ? exact : q;   // (outside: the range's end, or a zero of q's sign)
  }
  return y != y ? y : __builtin_amdgcn_fmed3f(y, -448.0f, 448.0f);
}

// Four values that e4m3_in returned as their codes, the first in bits 0 .. 7.
SILE_DEV uint32_t e4m3_pack4(const float* f) {
  int code = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  code = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], code, true);
  return (uint32_t)code;
}
// One such value.
SILE_DEV uint8_t e4m3_code(float f) {
  return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(f, f, 0, false) & 0xff);
}

}  // namespace sile
