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
// Four neighbouring values -> four e4m3 codes, the first in the low byte.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d, float scale) {
  const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a / scale, b / scale), __NV_SATFINITE, __NV_E4M3);
  const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c / scale, d / scale), __NV_SATFINITE, __NV_E4M3);
  return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
}
__device__ __forceinline__ uint8_t e4m3x1(float a, float scale) {
  return __nv_cvt_float_to_fp8(a / scale, __NV_SATFINITE, __NV_E4M3);
}
#endif

}  // namespace pto
