// FP8 linear layer with block scales: e4m3 operands, one fp32 scale per (row, 128 channels) of x and one per 128 x 128
// block of the weight.
//
//   out[m, n] = (acc[m, n] +) sum over K blocks kb of 128 channels of
//               x_scale[m, kb] * w_scale[n / 128, kb] * ( sum_{k in kb} x[m, k] * w[n, k] )
//
// It is the dense counterpart of the grouped expert GEMM (the numerics of the reference's block-scaled golden,
// tests/st/runtime/ops/test_matmul_mx.py:119-131, with fp32 scales per 128).  Products and sums are fp32; out is rounded
// once.  The order of additions depends on the sizes alone: equal calls give equal bits.
#include "common.cuh"
#include "kernels.h"

namespace pto {
namespace {

struct LinFp8Params {
  const uint8_t* x;         // [m, k]
  const float* x_scale;     // [m, kblocks]
  const uint8_t* w;         // [n, k]
  const float* w_scale;     // [ceil(n / 128), kblocks]
  const float* acc;         // [m, n] or NULL; may be out
  void* out;                // [m, n] bf16 or fp32
  int m, n, k, kblocks, out_bf16;
  int* err;
};

__device__ __forceinline__ void store_out(const LinFp8Params& p, size_t o, float v) {
  if (p.acc) v += p.acc[o];
  if (p.out_bf16) static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(v);
  else static_cast<float*>(p.out)[o] = v;
}

__device__ __forceinline__ float e4m3_to_f32(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

// Any K and any alignment: 64 x 64 output tiles on the CUDA cores, 32 channels at a time through shared memory.
constexpr int kAnyTile = 64, kAnyK = 32;
__global__ void __launch_bounds__(256) linear_fp8_any_kernel(const LinFp8Params p) {
  __shared__ float xs[kAnyK][kAnyTile + 1], ws[kAnyK][kAnyTile + 1];
  pdl_launch_dependents();
  pdl_wait();
  const int n0 = blockIdx.x * kAnyTile, m0 = blockIdx.y * kAnyTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {}, part[4][4] = {};
  for (int k0 = 0; k0 < p.k; k0 += kAnyK) {
    for (int i = threadIdx.x; i < kAnyTile * kAnyK; i += 256) {
      const int r = i / kAnyK, c = i - r * kAnyK, k = k0 + c;
      xs[c][r] = m0 + r < p.m && k < p.k ? e4m3_to_f32(p.x[static_cast<size_t>(m0 + r) * p.k + k]) : 0.f;
      ws[c][r] = n0 + r < p.n && k < p.k ? e4m3_to_f32(p.w[static_cast<size_t>(n0 + r) * p.k + k]) : 0.f;
    }
    __syncthreads();
#pragma unroll 8
    for (int c = 0; c < kAnyK; ++c) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { a[i] = xs[c][ty + 16 * i]; b[i] = ws[c][tx + 16 * i]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) part[i][j] += a[i] * b[j];
    }
    __syncthreads();
    if ((k0 + kAnyK) % 128 == 0 || k0 + kAnyK >= p.k) {   // end of a K block
      const int kb = k0 / 128;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty + 16 * i;
        const float sx = m < p.m ? p.x_scale[static_cast<size_t>(m) * p.kblocks + kb] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = n0 + tx + 16 * j;
          const float sw = n < p.n ? p.w_scale[static_cast<size_t>(n / 128) * p.kblocks + kb] : 0.f;
          acc[i][j] += part[i][j] * (sx * sw);
          part[i][j] = 0.f;
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m < p.m && n < p.n) store_out(p, static_cast<size_t>(m) * p.n + n, acc[i][j]);
    }
}

}  // namespace

int linear_fp8_launch(const void* x, const float* x_scale, const void* w, const float* w_scale, const float* acc, void* out,
                      int out_dtype, int m, int n, int k, int* err, cudaStream_t stream) {
  PTO_REQUIRE(m >= 0 && n > 0 && k > 0, "linear_fp8: n and k must be positive, m not negative");
  PTO_REQUIRE(out_dtype == PTO_BF16 || out_dtype == PTO_FP32, "linear_fp8: out must be bf16 or fp32");
  if (m == 0) return kOk;
  PTO_REQUIRE(x && x_scale && w && w_scale && out, "linear_fp8: NULL tensor");
  PTO_REQUIRE(!(acc && acc == out && out_dtype != PTO_FP32), "linear_fp8: only an fp32 out may be the tensor that is added");
  LinFp8Params p;
  p.x = static_cast<const uint8_t*>(x); p.x_scale = x_scale; p.w = static_cast<const uint8_t*>(w); p.w_scale = w_scale;
  p.acc = acc; p.out = out; p.m = m; p.n = n; p.k = k; p.kblocks = (k + 127) / 128; p.out_bf16 = out_dtype == PTO_BF16;
  p.err = err;
  PTO_REQUIRE((m + kAnyTile - 1) / kAnyTile <= 65535, "linear_fp8: too many rows");
  launch_kernel(linear_fp8_any_kernel, dim3((n + kAnyTile - 1) / kAnyTile, (m + kAnyTile - 1) / kAnyTile), dim3(256), 0,
                stream, p);
  return check_cuda(cudaGetLastError(), "linear_fp8_any_kernel launch");
}

}  // namespace pto
