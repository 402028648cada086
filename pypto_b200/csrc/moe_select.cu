// Routing to experts: scores, a balance bias, group-limited choice, top-k, weights.
//
//   score[e] = sigmoid(logit[e])  or  softmax over the experts
//   key[e]   = score[e] + bias[e]
//   groups of experts / n_group neighbouring experts; a group's score is the sum of its best `group_top` keys; the
//   best topk_group groups stay in the choice
//   idx = the topk experts by key among them, in descending order;  w = score (not key), divided by the sum of the
//   chosen scores when renormalising, times route_scale
//
// Equal keys and equal group scores go to the lower id.  A choice must not hang on a rounding: keys and group scores
// count as what they are in 64 bits.  An expert whose key is -inf (a bias of -inf takes it out) or NaN is not
// available: it adds nothing to its group's score; a row that runs out of available experts is filled with the lowest
// unused ids at weight 0, so that every index is a valid one.
// The reference has no router; the index contract is that of its descending sort with original indices
// (tests/st/runtime/ops/test_sort.py:602-632), as in moe_topk.
#include "common.cuh"
#include "kernels.h"

namespace pto {
namespace {

constexpr int kRouteWarps = 4;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopk = 32;

struct RouteParams {
  const void* logits;       // [tokens, experts] fp32 or bf16
  const float* bias;        // [experts] or NULL
  int32_t* idx;             // [tokens, topk]
  float* weights;           // [tokens, topk]
  int tokens, experts, topk, n_group, topk_group, group_top, softmax, renormalize, logits_bf16;
  float route_scale;
};

__device__ __forceinline__ float route_logit(const RouteParams& p, size_t i) {
  return p.logits_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[i]) : static_cast<const float*>(p.logits)[i];
}
__device__ __forceinline__ double warp_max_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One token by one warp, in 64 bits, for any expert count: score [experts], key [experts] and group [n_group] live in
// shared memory.
__device__ void route_token_f64(const RouteParams& p, int t, int lane, double* score, double* key, double* group) {
  const double kOut = -INFINITY;
  const size_t row = static_cast<size_t>(t) * p.experts;
  double top = kOut;
  if (p.softmax) {
    for (int e = lane; e < p.experts; e += 32) top = fmax(top, static_cast<double>(route_logit(p, row + e)));   // passes NaN over
    top = warp_max_f64(top);
  }
  double sum = 0.0;
  for (int e = lane; e < p.experts; e += 32) {
    const double x = route_logit(p, row + e);
    double s;
    if (!p.softmax) s = 1.0 / (1.0 + exp(-x));
    else if (isinf(top)) s = x == top && top > 0 ? 1.0 : (x == x ? 0.0 : x);   // +inf logits share the row; all -inf: 0
    else s = exp(x - top);
    score[e] = s;
    if (s == s) sum += s;
  }
  sum = warp_sum_f64(sum);
  for (int e = lane; e < p.experts; e += 32) {
    if (p.softmax) score[e] = sum > 0.0 ? score[e] / sum : score[e];
    const double k = score[e] + (p.bias ? static_cast<double>(p.bias[e]) : 0.0);
    key[e] = k == k ? k : kOut;
    if (key[e] == kOut) score[e] = 0.0;
  }
  __syncwarp();
  if (p.topk_group < p.n_group) {
    const int per = p.experts / p.n_group;
    for (int g = lane; g < p.n_group; g += 32) {
      double b1 = kOut, b2 = kOut;
      for (int j = 0; j < per; ++j) {
        const double k = key[g * per + j];
        if (k > b1) { b2 = b1; b1 = k; } else if (k > b2) { b2 = k; }
      }
      group[g] = p.group_top == 2 && b2 > kOut ? b1 + b2 : b1;
    }
    __syncwarp();
    for (int g = lane; g < p.n_group; g += 32) {
      int before = 0;
      for (int o = 0; o < p.n_group; ++o) before += group[o] > group[g] || (group[o] == group[g] && o < g);
      if (before >= p.topk_group)
        for (int j = 0; j < per; ++j) {
          key[g * per + j] = kOut;
          score[g * per + j] = 0.0;
        }
    }
    __syncwarp();
  }
  double picked = 0.0, mine = 0.0;
  int my_idx = 0;
  for (int k = 0; k < p.topk; ++k) {
    double best = kOut;
    int best_e = 0x7fffffff;
    for (int e = lane; e < p.experts; e += 32)
      if (key[e] == key[e] && (key[e] > best || best_e == 0x7fffffff)) { best = key[e]; best_e = e; }   // a taken expert's key is NaN
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, best, o);
      const int oe = __shfl_xor_sync(0xffffffffu, best_e, o);
      if (oe != 0x7fffffff && (best_e == 0x7fffffff || ob > best || (ob == best && oe < best_e))) { best = ob; best_e = oe; }
    }
    const double s = score[best_e];
    picked += s;
    if (lane == k) { mine = s; my_idx = best_e; }
    __syncwarp();
    if (lane == 0) key[best_e] = __longlong_as_double(0x7ff8000000000000ll);
    __syncwarp();
  }
  if (lane < p.topk) {
    const double w = p.renormalize ? (picked > 0.0 ? mine / picked : 0.0) : mine;
    p.idx[static_cast<size_t>(t) * p.topk + lane] = my_idx;
    p.weights[static_cast<size_t>(t) * p.topk + lane] = static_cast<float>(w * p.route_scale);
  }
}

// One warp per token.
__global__ void __launch_bounds__(kRouteWarps * 32) moe_route_any_kernel(const RouteParams p) {
  extern __shared__ double route_smem[];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x * kRouteWarps + warp;
  if (t >= p.tokens) return;
  double* score = route_smem + static_cast<size_t>(warp) * (2 * p.experts + p.n_group);
  route_token_f64(p, t, lane, score, score + p.experts, score + 2 * p.experts);
}

}  // namespace

int moe_route_launch(const void* logits, int logits_dtype, const float* bias, int scoring, int tokens, int experts,
                     int n_group, int topk_group, int group_top, int topk, int renormalize, float route_scale,
                     int32_t* idx, float* weights, cudaStream_t stream) {
  PTO_REQUIRE(logits_dtype == PTO_FP32 || logits_dtype == PTO_BF16, "moe_route: logits must be fp32 or bf16");
  PTO_REQUIRE(scoring == PTO_SCORE_SIGMOID || scoring == PTO_SCORE_SOFTMAX, "moe_route: unknown scoring");
  PTO_REQUIRE(tokens >= 0 && experts > 0 && experts <= kRouteMaxExperts, "moe_route: 1..1024 experts");
  PTO_REQUIRE(n_group > 0 && experts % n_group == 0, "moe_route: the experts must split evenly into n_group groups");
  PTO_REQUIRE(topk_group > 0 && topk_group <= n_group, "moe_route: topk_group must be 1..n_group");
  PTO_REQUIRE(group_top == 1 || group_top == 2, "moe_route: group_top must be 1 or 2");
  PTO_REQUIRE(topk > 0 && topk <= kRouteMaxTopk && topk <= topk_group * (experts / n_group),
              "moe_route: topk must be 1..32 and at most the experts of topk_group groups");
  if (tokens == 0) return kOk;
  PTO_REQUIRE(logits && idx && weights, "moe_route: NULL tensor");
  RouteParams p;
  p.logits = logits; p.bias = bias; p.idx = idx; p.weights = weights;
  p.tokens = tokens; p.experts = experts; p.topk = topk; p.n_group = n_group; p.topk_group = topk_group;
  p.group_top = group_top; p.softmax = scoring == PTO_SCORE_SOFTMAX; p.renormalize = renormalize;
  p.logits_bf16 = logits_dtype == PTO_BF16; p.route_scale = route_scale;
  const size_t smem = sizeof(double) * kRouteWarps * static_cast<size_t>(2 * experts + n_group);
  if (smem > 48 * 1024)
    PTO_CUDA(cudaFuncSetAttribute(moe_route_any_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(sizeof(double) * kRouteWarps * 3 * kRouteMaxExperts)));
  launch_kernel(moe_route_any_kernel, dim3((tokens + kRouteWarps - 1) / kRouteWarps), dim3(kRouteWarps * 32), smem, stream, p);
  return check_cuda(cudaGetLastError(), "moe_route_any_kernel launch");
}

}  // namespace pto
