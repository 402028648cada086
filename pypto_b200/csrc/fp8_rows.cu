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

// Rows too long for registers: one CTA per row, the row h kept in shared memory between the two passes.
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

// Rows of any size and alignment up to 16384: a warp takes whole groups of 128 columns, E neighbouring elements to a lane
// (two where sizes and addresses are even), and keeps its V groups of the row in registers between the two passes.
// All loads, gamma's too, are issued before the first sum, and the groups' maxima are reduced side by side: a warp's groups
// one after the other cost half as much again (3133 x 5003 62 us, 1000 x 16383 112).  Bound by the number of two- and
// four-byte accesses: bf16 with FP8 rows, 3133 x 5003 40 us, 3133 x 5002 32 us, 1000 x 16383 49 us.
// Rows staged through shared memory with 16-byte copies gave 57 us at 3133 x 5003 and x 5002 alike.
template <typename T, int E>
struct RawN;
template <>
struct RawN<float, 1> {
  float a;
  __device__ __forceinline__ void load(const float* p) { a = *p; }
  __device__ __forceinline__ float get(int) const { return a; }
};
template <>
struct RawN<float, 2> {
  float2 a;
  __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float2*>(p); }
  __device__ __forceinline__ float get(int i) const { return i ? a.y : a.x; }
};
template <>
struct RawN<__nv_bfloat16, 1> {
  __nv_bfloat16 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *p; }
  __device__ __forceinline__ float get(int) const { return __bfloat162float(a); }
};
template <>
struct RawN<__nv_bfloat16, 2> {
  uint32_t a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ float get(int i) const { return i ? bf16_hi_to_float(a) : bf16_lo_to_float(a); }
};
template <int E>
__device__ __forceinline__ void st_n(float* p, const float* v) {
  if (E == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[E - 1]);
  else *p = v[0];
}
template <int E>
__device__ __forceinline__ void st_n(__nv_bfloat16* p, const float* v) {
  if (E == 2) *reinterpret_cast<uint32_t*>(p) = pack_bf16x2(v[0], v[E - 1]);
  else *p = __float2bfloat16_rn(v[0]);
}
// Codes of four values of a lane (4 / E runs of E neighbours, 32 E columns apart; `left` columns to the row's end).
template <int E>
__device__ __forceinline__ void st_codes(uint8_t* q, int left, const float (&y)[4], float scale) {
  unsigned long long n[4] = {pack_f32x2(-y[0], -y[1]), pack_f32x2(-y[2], -y[3]), 0ull, 0ull};
  const uint32_t codes = e4m3x8_of_negated(n, scale).x;
#pragma unroll
  for (int j = 0; j < 4 / E; ++j)
    if (j * 32 * E < left) {
      if (E == 2) *reinterpret_cast<uint16_t*>(q + j * 64) = static_cast<uint16_t>(codes >> (16 * j));
      else q[j * 32] = static_cast<uint8_t>(codes >> (8 * j));
    }
}

constexpr int kOddThreads = 512;
template <typename TX, typename TR, int E, int V>
__global__ void __launch_bounds__(kOddThreads) add_rms_norm_odd_kernel(const AddNormParams p) {
  __shared__ float red[kOddThreads / 32];
  pdl_launch_dependents();
  pdl_wait();
  const size_t base = static_cast<size_t>(blockIdx.x) * p.hidden;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const TX* x = static_cast<const TX*>(p.x) + base;
  const TR* r = p.residual ? static_cast<const TR*>(p.residual) + base : nullptr;
  TR* ro = p.residual_out ? static_cast<TR*>(p.residual_out) + base : nullptr;
  RawN<TX, E> xr[V][4 / E];
  RawN<TR, E> rr[V][4 / E];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int j = 0; j < 4 / E; ++j) {      // past the end: the last elements again, counted as zero below
      const int c = min((v * warps + warp) * kQuantGroup + (j * 32 + lane) * E, p.hidden - E);
      xr[v][j].load(x + c);
      if (r) rr[v][j].load(r + c);
    }
  float gm[V][4];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = (v * warps + warp) * kQuantGroup + (i / E * 32 + lane) * E + i % E;
      gm[v][i] = p.gamma ? __ldg(p.gamma + min(c, p.hidden - 1)) : 1.f;
    }
  float h[V][4], ss = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int j = 0; j < 4 / E; ++j) {
      const int c = (v * warps + warp) * kQuantGroup + (j * 32 + lane) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float s = xr[v][j].get(e) + (r ? rr[v][j].get(e) : 0.f);
        h[v][j * E + e] = c < p.hidden ? s : 0.f;
        ss += h[v][j * E + e] * h[v][j * E + e];
      }
      if (ro && c < p.hidden) st_n<E>(ro + c, &h[v][j * E]);
    }
  ss = warp_sum(ss);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  ss = warp_sum(lane < warps ? red[lane] : 0.f);
  const float inv = rsqrtf(ss / static_cast<float>(p.hidden) + p.eps);
  float amax[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    amax[v] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[v][i] = h[v][i] * inv * gm[v][i];
      amax[v] = fmaxf(amax[v], fabsf(h[v][i]));
    }
  }
  if (p.out)
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < 4 / E; ++j) {
        const int c = (v * warps + warp) * kQuantGroup + (j * 32 + lane) * E;
        if (c < p.hidden) {
          if (p.out_bf16) st_n<E>(static_cast<__nv_bfloat16*>(p.out) + base + c, &h[v][j * E]);
          else st_n<E>(static_cast<float*>(p.out) + base + c, &h[v][j * E]);
        }
      }
  if (p.q) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int v = 0; v < V; ++v) amax[v] = fmaxf(amax[v], __shfl_xor_sync(0xffffffffu, amax[v], o));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int g = v * warps + warp, c0 = g * kQuantGroup + lane * E;
      const float s = e4m3_group_scale_fast(amax[v]);
      st_codes<E>(p.q + base + c0, p.hidden - c0, h[v], s);
      if (lane == 0 && g < p.groups) p.scale[static_cast<size_t>(blockIdx.x) * p.groups + g] = s;
    }
  }
}

// n / d for 0 <= n < 2^31 as a multiplication: mul = ceil(2^(31 + l) / d) with 2^l >= d overshoots n / d by less than
// 1 / d.
struct FastDiv {
  uint32_t mul, shift, d;
  explicit FastDiv(uint32_t divisor) : mul(0), shift(0), d(divisor) {
    uint32_t l = 1;
    while ((1ull << l) < d) ++l;
    mul = d > 1 ? static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d) : 0;
    shift = l - 1;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return d > 1 ? __umulhi(n, mul) >> shift : n; }
};

// a = g * sigmoid(g) * u with the sigmoid as recip(1 + exp(-g)) (examples/models/qwen3_jit/kernels/mlp.py:23-61)
// The quotient is the approximate one (2 ulp), as in the GEMMs' epilogues.
__device__ __forceinline__ float swiglu(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// Any size and alignment: a warp takes a group of 128 columns, E neighbouring elements to a lane, two groups under way.
template <typename T, int E>
__global__ void __launch_bounds__(kRowThreads)
swiglu_quantize_odd_kernel(const T* __restrict__ gate_up, uint8_t* __restrict__ q, float* __restrict__ scale, uint32_t total,
                           int inter, const FastDiv groups) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const uint32_t step = gridDim.x * (kRowThreads / 32) * 2;
  for (uint32_t g0 = (blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5)) * 2; g0 < total; g0 += step) {
    RawN<T, E> gr[2][4 / E], ur[2][4 / E];
    uint32_t r[2];
    int c0[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t g = min(g0 + u, total - 1);
      r[u] = groups(g);
      c0[u] = static_cast<int>(g - r[u] * groups.d) * kQuantGroup + lane * E;
      const T* gate = gate_up + static_cast<size_t>(r[u]) * 2 * inter;
#pragma unroll
      for (int j = 0; j < 4 / E; ++j) {
        const int c = min(c0[u] + j * 32 * E, inter - E);      // past the end: not used
        gr[u][j].load(gate + c);
        ur[u][j].load(gate + inter + c);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (g0 + u >= total) break;
      float a[4], amax = 0.f;
#pragma unroll
      for (int j = 0; j < 4 / E; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float v = swiglu(gr[u][j].get(e), ur[u][j].get(e));
          a[j * E + e] = c0[u] + j * 32 * E < inter ? v : 0.f;
          amax = fmaxf(amax, fabsf(a[j * E + e]));
        }
      const float s = e4m3_group_scale_fast(warp_max(amax));
      st_codes<E>(q + static_cast<size_t>(r[u]) * inter + c0[u], inter - c0[u], a, s);
      if (lane == 0) scale[g0 + u] = s;
    }
  }
}

// ---------------------------------------------------------------------------
// Rows of whole 8-element units on 16-byte boundaries: one read and one write of everything.
//
// A thread keeps V units of eight neighbouring elements of its row in registers between the two passes (sum of squares;
// scaling and quantisation), so 16 neighbouring threads hold one group of 128 columns and its maximum is four shuffles.
// DRAM bounds both kernels when the work is large.  8192 x 7168, bf16 in, bf16 residual in and out, FP8 rows out: 70 us = 5.86
// TB/s (80-94 us before all of a thread's loads went out ahead of their first use); 4096 x 4096 fp32: 37 us = 6.3 TB/s.
// SwiGLU 8192 x 14336 bf16: 101 us = 5.8 TB/s, where the special functions and the issue slots come close behind; a division
// for every value instead of the exact quotient of fp8_quant.cuh made it 211 us.
// ---------------------------------------------------------------------------
using Pair = unsigned long long;     // two neighbouring fp32 values

__device__ __forceinline__ void pairs_of(uint4 w, Pair (&v)[4]) {      // eight bf16
  v[0] = pack_f32x2(bf16_lo_to_float(w.x), bf16_hi_to_float(w.x));
  v[1] = pack_f32x2(bf16_lo_to_float(w.y), bf16_hi_to_float(w.y));
  v[2] = pack_f32x2(bf16_lo_to_float(w.z), bf16_hi_to_float(w.z));
  v[3] = pack_f32x2(bf16_lo_to_float(w.w), bf16_hi_to_float(w.w));
}
__device__ __forceinline__ void pairs_of(float4 a, float4 b, Pair (&v)[4]) {
  v[0] = pack_f32x2(a.x, a.y);
  v[1] = pack_f32x2(a.z, a.w);
  v[2] = pack_f32x2(b.x, b.y);
  v[3] = pack_f32x2(b.z, b.w);
}
// Eight neighbouring elements as they come from memory, by plain loads: the residual may be written in place.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0]; b = reinterpret_cast<const float4*>(p)[1]; }
  __device__ __forceinline__ void pairs(Pair (&v)[4]) const { pairs_of(a, b, v); }
};
template <>
struct Raw8<__nv_bfloat16> {
  uint4 a;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void pairs(Pair (&v)[4]) const { pairs_of(a, v); }
};
// The same through the read-only path, for what nothing here writes: these loads may run ahead of the stores before them.
__device__ __forceinline__ void ld8(const float* p, Pair (&v)[4]) {
  pairs_of(__ldg(reinterpret_cast<const float4*>(p)), __ldg(reinterpret_cast<const float4*>(p) + 1), v);
}
__device__ __forceinline__ void ld8(const __nv_bfloat16* p, Pair (&v)[4]) { pairs_of(__ldg(reinterpret_cast<const uint4*>(p)), v); }
__device__ __forceinline__ void st8(float* p, const Pair (&v)[4]) {
  reinterpret_cast<ulonglong2*>(p)[0] = make_ulonglong2(v[0], v[1]);
  reinterpret_cast<ulonglong2*>(p)[1] = make_ulonglong2(v[2], v[3]);
}
__device__ __forceinline__ uint32_t bf16_pair(Pair v) {
  float a, b;
  unpack_f32x2(v, a, b);
  return pack_bf16x2(a, b);
}
__device__ __forceinline__ void st8(__nv_bfloat16* p, const Pair (&v)[4]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pair(v[0]), bf16_pair(v[1]), bf16_pair(v[2]), bf16_pair(v[3]));
}

// Largest magnitude of a group of 128 columns held by 16 neighbouring lanes.
__device__ __forceinline__ float group_max16(const Pair (&v)[4]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    unpack_f32x2(v[i], a, b);
    m = fmaxf(m, fmaxf(fabsf(a), fabsf(b)));
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

template <typename TX, typename TR, int V, int THREADS>
__global__ void __launch_bounds__(THREADS) add_rms_norm_kernel(const AddNormParams p) {
  __shared__ float red[32];
  pdl_launch_dependents();
  pdl_wait();
  const size_t base = static_cast<size_t>(blockIdx.x) * p.hidden;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const TX* x = static_cast<const TX*>(p.x) + base;
  const TR* r = p.residual ? static_cast<const TR*>(p.residual) + base : nullptr;
  TR* ro = p.residual_out ? static_cast<TR*>(p.residual_out) + base : nullptr;
  // Everything a thread reads is under way before the first value is used; a unit past the end reads the last one and
  // counts as zero.
  Raw8<TX> xr[V];
  Raw8<TR> rr[V];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int c = min((u * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8, p.hidden - 8);
    xr[u].load(x + c);
    if (r) rr[u].load(r + c);
  }
  Pair h[V][4];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const bool in = (u * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8 < p.hidden;
    xr[u].pairs(h[u]);
    if (r) {
      Pair v[4];
      rr[u].pairs(v);
#pragma unroll
      for (int j = 0; j < 4; ++j) h[u][j] = add2(h[u][j], v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) h[u][j] = in ? h[u][j] : 0ull;
  }
  Pair s2 = 0ull;
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int c = (u * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * 8;
    if (ro && c < p.hidden) st8(ro + c, h[u]);
#pragma unroll
    for (int j = 0; j < 4; ++j) s2 = fma2(h[u][j], h[u][j], s2);
  }
  float ss, odd;
  unpack_f32x2(s2, ss, odd);
  ss = warp_sum(ss + odd);
  if (lane == 0) red[warp] = ss;
  __syncthreads();
  ss = warp_sum(lane < warps ? red[lane] : 0.f);
  const float inv = rsqrtf(ss / static_cast<float>(p.hidden) + p.eps);
  const Pair inv2 = pack_f32x2(inv, inv), minus = pack_f32x2(-1.f, -1.f);
#pragma unroll
  for (int u = 0; u < V; ++u) {
    const int unit = u * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x), c = unit * 8;
    const bool in = c < p.hidden;
    Pair y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = mul_f32x2(h[u][j], inv2);
    if (p.gamma && in) {
      Pair g[4];
      ld8(p.gamma + c, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = mul_f32x2(y[j], g[j]);
    }
    if (p.out && in) {
      if (p.out_bf16) st8(static_cast<__nv_bfloat16*>(p.out) + base + c, y);
      else st8(static_cast<float*>(p.out) + base + c, y);
    }
    if (p.q) {
      const float s = e4m3_group_scale_fast(group_max16(y));
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = mul_f32x2(y[j], minus);
      if (in) {
        *reinterpret_cast<uint2*>(p.q + base + c) = e4m3x8_of_negated(y, s);
        if ((threadIdx.x & 15) == 0) p.scale[static_cast<size_t>(blockIdx.x) * p.groups + unit / 16] = s;
      }
    }
  }
}

// One pair of groups of 128 columns per warp at a time, sixteen lanes to a group.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
swiglu_quantize_kernel(const T* __restrict__ gate_up, uint8_t* __restrict__ q, float* __restrict__ scale, uint32_t total, int inter,
                       const FastDiv groups) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, hl = lane & 15;
  const uint32_t step = gridDim.x * (kRowThreads / 32) * 2;
  for (uint32_t g0 = (blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5)) * 2; g0 < total; g0 += step) {
    const uint32_t g = g0 + (lane >> 4), r = groups(g);
    const int c = static_cast<int>(g - r * groups.d) * kQuantGroup + hl * 8;
    const bool in = g < total && c < inter;
    Pair a[4] = {}, b[4] = {};
    if (in) {
      const T* src = gate_up + static_cast<size_t>(r) * 2 * inter + c;
      ld8(src, a);
      ld8(src + inter, b);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {      // negated: g u / (-1 - exp(-g))
      float g0f, g1f;
      unpack_f32x2(a[j], g0f, g1f);
      a[j] = mul_f32x2(pack_f32x2(__fdividef(g0f, -1.f - __expf(-g0f)), __fdividef(g1f, -1.f - __expf(-g1f))), b[j]);
    }
    const float s = e4m3_group_scale_fast(group_max16(a));
    if (in) {
      *reinterpret_cast<uint2*>(q + static_cast<size_t>(r) * inter + c) = e4m3x8_of_negated(a, s);
      if (hl == 0) scale[g] = s;
    }
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

template <typename TX, typename TR, int V, int THREADS>
int add_norm_units(const AddNormParams& p, long long rows, int threads, cudaStream_t stream) {
  launch_kernel(add_rms_norm_kernel<TX, TR, V, THREADS>, dim3(static_cast<unsigned>(rows)), dim3(threads), 0, stream, p);
  return check_cuda(cudaGetLastError(), "add_rms_norm_kernel launch");
}

template <typename TX, typename TR, int E>
int add_norm_odd(const AddNormParams& p, long long rows, cudaStream_t stream) {
  // Eight warps, while that leaves a warp no more than six groups, for pairs (3133 x 5002 32 us, with sixteen 37); sixteen
  // for single elements, which need more loads in flight (3133 x 5003 40 us, with eight 44), and for longer rows.
  const int most = E == 2 && p.groups <= 48 ? 8 : kOddThreads / 32;
  const int v = (p.groups + most - 1) / most, warps = (p.groups + v - 1) / v;
  const dim3 grid(static_cast<unsigned>(rows)), block(32 * warps);
  if (v <= 1) launch_kernel(add_rms_norm_odd_kernel<TX, TR, E, 1>, grid, block, 0, stream, p);
  else if (v <= 2) launch_kernel(add_rms_norm_odd_kernel<TX, TR, E, 2>, grid, block, 0, stream, p);
  else if (v <= 3) launch_kernel(add_rms_norm_odd_kernel<TX, TR, E, 3>, grid, block, 0, stream, p);
  else if (v <= 4) launch_kernel(add_rms_norm_odd_kernel<TX, TR, E, 4>, grid, block, 0, stream, p);
  else if (v <= 5) launch_kernel(add_rms_norm_odd_kernel<TX, TR, E, 5>, grid, block, 0, stream, p);
  else if (v <= 6) launch_kernel(add_rms_norm_odd_kernel<TX, TR, E, 6>, grid, block, 0, stream, p);
  else launch_kernel(add_rms_norm_odd_kernel<TX, TR, E, 8>, grid, block, 0, stream, p);
  return check_cuda(cudaGetLastError(), "add_rms_norm_odd_kernel launch");
}

template <typename TX, typename TR>
int add_norm(const AddNormParams& p, long long rows, cudaStream_t stream) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.residual) |
                        reinterpret_cast<uintptr_t>(p.residual_out) | reinterpret_cast<uintptr_t>(p.gamma) |
                        reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.q);
  const int units = p.hidden / 8;
  if (p.hidden > 16384) return add_norm_any<TX, TR>(p, rows, stream);
  if (p.hidden % 8 != 0 || (all & 15) != 0)
    return p.hidden % 2 == 0 && (all & 7) == 0 ? add_norm_odd<TX, TR, 2>(p, rows, stream) : add_norm_odd<TX, TR, 1>(p, rows, stream);
  // Few rows: as many threads as there are units, the row is latency.  Many rows: two or four units a thread, so that more
  // bytes of more rows are under way (8192 x 7168: one unit a thread 94 us where two took 80).
  auto whole_warps = [](int n) { return (n + 31) / 32 * 32; };
  if (units <= 256) return add_norm_units<TX, TR, 1, 256>(p, rows, whole_warps(units), stream);
  if (rows <= 2ll * sm_count())
    return units <= 1024 ? add_norm_units<TX, TR, 1, 1024>(p, rows, whole_warps(units), stream)
                         : add_norm_units<TX, TR, 2, 1024>(p, rows, whole_warps((units + 1) / 2), stream);
  if (units <= 512) return add_norm_units<TX, TR, 2, 256>(p, rows, whole_warps((units + 1) / 2), stream);
  if (units <= 1024) return add_norm_units<TX, TR, 2, 512>(p, rows, whole_warps((units + 1) / 2), stream);
  return add_norm_units<TX, TR, 4, 512>(p, rows, whole_warps((units + 3) / 4), stream);
}

template <typename T>
int swiglu_units(const T* gate_up, uint8_t* q, float* scale, uint32_t total, int inter, int groups, int unit, dim3 grid,
                 cudaStream_t stream) {
  auto* kernel = unit == 8 ? swiglu_quantize_kernel<T> : (unit == 2 ? swiglu_quantize_odd_kernel<T, 2> : swiglu_quantize_odd_kernel<T, 1>);
  launch_kernel(kernel, grid, dim3(kRowThreads), 0, stream, gate_up, q, scale, total, inter, FastDiv(groups));
  return check_cuda(cudaGetLastError(), "swiglu_quantize launch");
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
  // in place on whole rows only: a row is read before any of it is written, but a shifted one may belong to another CTA
  const size_t count = static_cast<size_t>(rows) * hidden, x_bytes = count * (x_dtype == PTO_BF16 ? 2 : 4);
  const size_t res_bytes = count * (res_dtype == PTO_BF16 ? 2 : 4);
  PTO_REQUIRE((residual_out == x && res_dtype == x_dtype) || !overlaps(residual_out, res_bytes, x, x_bytes),
              "add_rms_norm: residual_out overlaps x");
  PTO_REQUIRE(residual_out == residual || !overlaps(residual_out, res_bytes, residual, res_bytes),
              "add_rms_norm: residual_out overlaps residual");
  AddNormParams p;
  p.x = x; p.residual = residual; p.residual_out = residual_out; p.gamma = gamma; p.out = out;
  p.q = static_cast<uint8_t*>(q); p.scale = scale;
  p.hidden = hidden; p.groups = (hidden + kQuantGroup - 1) / kQuantGroup; p.out_bf16 = out_dtype == PTO_BF16; p.eps = eps;
  if (x_dtype == PTO_BF16)
    return res_dtype == PTO_BF16 ? add_norm<__nv_bfloat16, __nv_bfloat16>(p, rows, stream)
                                 : add_norm<__nv_bfloat16, float>(p, rows, stream);
  return res_dtype == PTO_BF16 ? add_norm<float, __nv_bfloat16>(p, rows, stream) : add_norm<float, float>(p, rows, stream);
}

int swiglu_quantize_launch(const void* gate_up, int dtype, void* q, float* scale, long long rows, int inter,
                           cudaStream_t stream) {
  PTO_REQUIRE(rows >= 0 && rows < (1ll << 31) && inter > 0 && inter <= (1 << 30), "swiglu_quantize: bad sizes");
  PTO_REQUIRE(dtype == PTO_BF16 || dtype == PTO_FP32, "swiglu_quantize: gate_up must be bf16 or fp32");
  if (rows == 0) return kOk;
  PTO_REQUIRE(gate_up && q && scale, "swiglu_quantize: NULL tensor");
  const int groups = (inter + kQuantGroup - 1) / kQuantGroup;
  const long long total = rows * groups;
  PTO_REQUIRE(total < (1ll << 31) - (1 << 24), "swiglu_quantize: too many groups of 128 columns");
  // one pair of groups per warp and round, 32 CTAs an SM (8: 111 us, 32: 101 us at 8192 x 14336 in bf16)
  const long long want = (total + 2 * (kRowThreads / 32) - 1) / (2 * (kRowThreads / 32)), most = static_cast<long long>(sm_count()) * 32;
  const dim3 grid(static_cast<unsigned>(want < most ? want : most));
  const uintptr_t all = reinterpret_cast<uintptr_t>(gate_up) | reinterpret_cast<uintptr_t>(q);
  const int unit = inter % 8 == 0 && (all & 15) == 0 ? 8 : (inter % 2 == 0 && (all & 7) == 0 ? 2 : 1);
  return dtype == PTO_BF16 ? swiglu_units(static_cast<const __nv_bfloat16*>(gate_up), static_cast<uint8_t*>(q), scale,
                                          static_cast<uint32_t>(total), inter, groups, unit, grid, stream)
                           : swiglu_units(static_cast<const float*>(gate_up), static_cast<uint8_t*>(q), scale,
                                          static_cast<uint32_t>(total), inter, groups, unit, grid, stream);
}

}  // namespace pto
