// The FP8 row format of this library, shared by every kernel that writes it: e4m3 values with one fp32 scale per
// (row, 128 columns), scale = max |y| / 448, q = e4m3(y / scale), round to nearest even, saturating.
// A group whose maximum is zero, or so small that max / 448 is zero in fp32, takes scale 1.  fmaxf passes a NaN over,
// so a NaN element stays a NaN and leaves the scale of its group alone; an infinite element makes the scale infinite
// and comes back as a NaN.
#pragma once
#include "common.cuh"

namespace pto {

constexpr int kQuantGroup = 128;

#ifdef __CUDACC__
__device__ __forceinline__ float e4m3_group_scale(float amax) {
  const float s = amax / 448.f;
  return s > 0.f ? s : 1.f;
}
// Eight neighbouring values -> eight e4m3 codes, the first in the low byte of .x.
//
// v / scale rounded as a division rounds it, at three instructions a value instead of a division's dozen: with r the
// correctly rounded 1 / scale, q = v r, e = q scale - v (exact in one fma) and q - e r is the correctly rounded quotient
// (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990, theorem 8.3).  That
// needs e to be exact: a code other than 0 has |v| >= scale 2^-10, so e is a multiple of 2^-56 scale, which the range of
// scales below keeps above the smallest subnormal.  Other scales (also infinite ones) divide.
__device__ __forceinline__ uint2 e4m3x8(const float (&v)[8], float scale) {
  float q[8];
  if (scale > 0x1p-70f && scale < 0x1p100f) {
    const float r = 1.f / scale;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q0 = v[i] * r;
      q[i] = fmaf(-fmaf(q0, scale, -v[i]), r, q0);     // signs so that a -0 stays one
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = v[i] / scale;
  }
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = __nv_cvt_float2_to_fp8x2(make_float2(q[2 * i], q[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}
__device__ __forceinline__ uint8_t e4m3x1(float a, float scale) {
  return __nv_cvt_float_to_fp8(a / scale, __NV_SATFINITE, __NV_E4M3);
}
#endif

}  // namespace pto
