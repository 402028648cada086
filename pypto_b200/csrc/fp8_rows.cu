// Row operators that hand FP8 rows to the FP8 matrix products: RMSNorm with the residual's addition, and SwiGLU.
//
//   add_rms_norm      h = x + residual;  y = h * rsqrt(mean(h^2) + eps) * gamma
//                     -> residual_out = h, out = y (bf16 or fp32), q / scale = FP8 rows of y
//   swiglu_quantize   a = gate * sigmoid(gate) * up -> q / scale = FP8 rows of a
//
// The norm is the one of rms_norm (examples/models/qwen3_jit/kernels/rmsnorm.py:27-89), with the addition that the
// reference's layer does in the projection before it (examples/models/qwen3_jit/kernels/projection.py:146-177) and the
// per-(row, 128 columns) quantisation of quantize_rows behind it, in one pass over the row.  The sum h, the statistics
// and y stay in fp32; what is stored narrower is rounded once, from the fp32 value: the norm of a bf16 residual stream
// is taken of the unrounded sum, and the FP8 rows of the unrounded y.
#include "common.cuh"
#include "fp8_quant.cuh"
#include "kernels.h"

namespace pto {
namespace {

template <typename T>
__device__ __forceinline__ float ld_f32(const T* p);
template <>
__device__ __forceinline__ float ld_f32<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float ld_f32<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st_f32(float* p, float v) { *p = v; }
__device__ __forceinline__ void st_f32(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

constexpr int kRowThreads = 256;
constexpr int kMaxHidden = 49152;   // one fp32 row in shared memory

struct AddNormParams {
  const void* x;
  const void* residual;     // NULL: h = x
  void* residual_out;       // NULL: h is not stored; may be `residual`
  const float* gamma;       // NULL: 1
  void* out;                // NULL: y is not stored
  uint8_t* q;               // NULL: no FP8 rows
  float* scale;
  int hidden, groups, out_bf16;
  float eps;
};

// Any hidden size and alignment: one CTA per row, the row h kept in shared memory between the two passes.
template <typename TX, typename TR>
__global__ void __launch_bounds__(kRowThreads) add_rms_norm_any_kernel(const AddNormParams p) {
  extern __shared__ float row[];
  __shared__ float red[kRowThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const size_t base = static_cast<size_t>(blockIdx.x) * p.hidden;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const TX* x = static_cast<const TX*>(p.x) + base;
  const TR* r = p.residual ? static_cast<const TR*>(p.residual) + base : nullptr;
  TR* ro = p.residual_out ? static_cast<TR*>(p.residual_out) + base : nullptr;
  float ss = 0.f;
  for (int i = threadIdx.x; i < p.hidden; i += kRowThreads) {
    const float h = ld_f32(x + i) + (r ? ld_f32(r + i) : 0.f);
    if (ro) st_f32(ro + i, h);
    row[i] = h;
    ss += h * h;
  }
  ss = warp_sum(ss);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) total += red[w];
  const float inv = rsqrtf(total / static_cast<float>(p.hidden) + p.eps);
  for (int g = warp; g < p.groups; g += kRowThreads / 32) {
    float y[4], amax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = g * kQuantGroup + j * 32 + lane;
      y[j] = i < p.hidden ? row[i] * inv * (p.gamma ? p.gamma[i] : 1.f) : 0.f;
      amax = fmaxf(amax, fabsf(y[j]));
    }
    const float s = e4m3_group_scale(warp_max(amax));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = g * kQuantGroup + j * 32 + lane;
      if (i >= p.hidden) continue;
      if (p.out) {
        if (p.out_bf16) static_cast<__nv_bfloat16*>(p.out)[base + i] = __float2bfloat16_rn(y[j]);
        else static_cast<float*>(p.out)[base + i] = y[j];
      }
      if (p.q) p.q[base + i] = e4m3x1(y[j], s);
    }
    if (p.q && lane == 0) p.scale[static_cast<size_t>(blockIdx.x) * p.groups + g] = s;
  }
}

// a = g * sigmoid(g) * u with the sigmoid as recip(1 + exp(-g)) (examples/models/qwen3_jit/kernels/mlp.py:23-61)
__device__ __forceinline__ float swiglu(float g, float u) { return g / (1.f + __expf(-g)) * u; }

// Any size and alignment: one warp per (row, 128 columns).
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
swiglu_quantize_any_kernel(const T* __restrict__ gate_up, uint8_t* __restrict__ q, float* __restrict__ scale,
                           long long rows, int inter, int groups) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long total = rows * groups, warps = static_cast<long long>(gridDim.x) * (kRowThreads / 32);
  for (long long w = static_cast<long long>(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5); w < total; w += warps) {
    const long long r = w / groups;
    const int c0 = static_cast<int>(w - r * groups) * kQuantGroup;
    const T* gate = gate_up + r * 2 * inter;
    float a[4], amax = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + j * 32 + lane;
      a[j] = c < inter ? swiglu(ld_f32(gate + c), ld_f32(gate + inter + c)) : 0.f;
      amax = fmaxf(amax, fabsf(a[j]));
    }
    const float s = e4m3_group_scale(warp_max(amax));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + j * 32 + lane;
      if (c < inter) q[r * inter + c] = e4m3x1(a[j], s);
    }
    if (lane == 0) scale[w] = s;
  }
}

template <typename TX, typename TR>
int add_norm_any(const AddNormParams& p, long long rows, cudaStream_t stream) {
  const size_t smem = sizeof(float) * static_cast<size_t>(p.hidden);
  if (smem > 48 * 1024)
    PTO_CUDA(cudaFuncSetAttribute(add_rms_norm_any_kernel<TX, TR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  kMaxHidden * 4));
  launch_kernel(add_rms_norm_any_kernel<TX, TR>, dim3(static_cast<unsigned>(rows)), dim3(kRowThreads), smem, stream, p);
  return check_cuda(cudaGetLastError(), "add_rms_norm_any_kernel launch");
}

}  // namespace

int add_rms_norm_launch(const void* x, int x_dtype, const void* residual, void* residual_out, int res_dtype,
                        const float* gamma, void* out, int out_dtype, void* q, float* scale, long long rows, int hidden,
                        float eps, cudaStream_t stream) {
  PTO_REQUIRE(rows >= 0 && rows < (1ll << 31) && hidden > 0 && hidden <= kMaxHidden,
              "add_rms_norm: rows must be 0..2^31-1 and hidden 1..49152");
  PTO_REQUIRE(x_dtype == PTO_BF16 || x_dtype == PTO_FP32, "add_rms_norm: x must be bf16 or fp32");
  PTO_REQUIRE(res_dtype == PTO_BF16 || res_dtype == PTO_FP32, "add_rms_norm: the residual must be bf16 or fp32");
  PTO_REQUIRE(!out || out_dtype == PTO_BF16 || out_dtype == PTO_FP32, "add_rms_norm: out must be bf16 or fp32");
  PTO_REQUIRE(eps >= 0.f, "add_rms_norm: eps must not be negative");
  if (rows == 0) return kOk;
  PTO_REQUIRE(out || q, "add_rms_norm: neither out nor q is given");
  PTO_REQUIRE((q == nullptr) == (scale == nullptr), "add_rms_norm: FP8 rows need both q and scale");
  PTO_REQUIRE(x, "add_rms_norm: NULL tensor");
  AddNormParams p;
  p.x = x; p.residual = residual; p.residual_out = residual_out; p.gamma = gamma; p.out = out;
  p.q = static_cast<uint8_t*>(q); p.scale = scale;
  p.hidden = hidden; p.groups = (hidden + kQuantGroup - 1) / kQuantGroup; p.out_bf16 = out_dtype == PTO_BF16; p.eps = eps;
  if (x_dtype == PTO_BF16)
    return res_dtype == PTO_BF16 ? add_norm_any<__nv_bfloat16, __nv_bfloat16>(p, rows, stream)
                                 : add_norm_any<__nv_bfloat16, float>(p, rows, stream);
  return res_dtype == PTO_BF16 ? add_norm_any<float, __nv_bfloat16>(p, rows, stream) : add_norm_any<float, float>(p, rows, stream);
}

int swiglu_quantize_launch(const void* gate_up, int dtype, void* q, float* scale, long long rows, int inter,
                           cudaStream_t stream) {
  PTO_REQUIRE(rows >= 0 && inter > 0 && inter <= (1 << 30), "swiglu_quantize: bad sizes");
  PTO_REQUIRE(dtype == PTO_BF16 || dtype == PTO_FP32, "swiglu_quantize: gate_up must be bf16 or fp32");
  if (rows == 0) return kOk;
  PTO_REQUIRE(gate_up && q && scale, "swiglu_quantize: NULL tensor");
  const int groups = (inter + kQuantGroup - 1) / kQuantGroup;
  const long long ctas = (rows * groups + kRowThreads / 32 - 1) / (kRowThreads / 32), cap = static_cast<long long>(sm_count()) * 8;
  const dim3 grid(static_cast<unsigned>(ctas < cap ? ctas : cap));
  if (dtype == PTO_BF16)
    launch_kernel(swiglu_quantize_any_kernel<__nv_bfloat16>, grid, dim3(kRowThreads), 0, stream,
                  static_cast<const __nv_bfloat16*>(gate_up), static_cast<uint8_t*>(q), scale, rows, inter, groups);
  else
    launch_kernel(swiglu_quantize_any_kernel<float>, grid, dim3(kRowThreads), 0, stream, static_cast<const float*>(gate_up),
                  static_cast<uint8_t*>(q), scale, rows, inter, groups);
  return check_cuda(cudaGetLastError(), "swiglu_quantize_any_kernel launch");
}

}  // namespace pto
