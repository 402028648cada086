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
// Scales for which the quotients below come out exactly as a division's; others (also 0-like and infinite ones) divide.
__device__ __forceinline__ bool e4m3_plain_scale(float s) { return s > 0x1p-70f && s < 0x1p100f; }

// amax / 448 by the same theorem as below, for a maximum well inside the range; the division otherwise.
__device__ __forceinline__ float e4m3_group_scale_fast(float amax) {
  constexpr float r = 1.f / 448.f;
  const float q = amax * r, s = fmaf(-fmaf(q, 448.f, -amax), r, q);
  return e4m3_plain_scale(q) ? s : e4m3_group_scale(amax);
}

// Packed pairs of floats (one instruction for two).
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Eight neighbouring values, given NEGATED as four packed pairs -> eight e4m3 codes, the first in the low byte of .x.
//
// v / scale rounded as a division rounds it, at three operations a value instead of a division's dozen: with r the
// correctly rounded 1 / scale, q = v r, e = q scale - v (exact in one fma) and q - e r is the correctly rounded quotient
// (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990, theorem 8.3).  That
// needs e to be exact: a code other than 0 has |v| >= scale 2^-10, so e is a multiple of 2^-56 scale, which
// e4m3_plain_scale keeps above the smallest subnormal.  Negated values make every sign right, that of a -0 too, without an
// operation of its own: q = (-v)(-r), e = q scale + (-v), q + e (-r).
__device__ __forceinline__ uint2 e4m3x8_of_negated(const unsigned long long (&nv)[4], float scale) {
  float q[8];
  if (e4m3_plain_scale(scale)) {
    const float r = -1.f / scale;
    const unsigned long long r2 = pack_f32x2(r, r), s2 = pack_f32x2(scale, scale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned long long q0 = mul_f32x2(nv[i], r2);
      unpack_f32x2(fma2(fma2(q0, s2, nv[i]), r2, q0), q[2 * i], q[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      unpack_f32x2(nv[i], a, b);
      q[2 * i] = -a / scale;
      q[2 * i + 1] = -b / scale;
    }
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
