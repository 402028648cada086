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
#include <cfloat>

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
// shared memory.  The definition itself; what the kernel below cannot decide in 32 bits ends here.
__device__ __noinline__ void route_token_f64(const RouteParams& p, int t, int lane, double* score, double* key, double* group) {
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

// One warp per token, any expert count and grouping, everything in 64 bits.
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

// One warp per token, keys in 32 bits with a bound on their error, 64 bits only where that bound leaves a
// choice open.
//
// A lane holds PER neighbouring experts, so a group is a power-of-two run of lanes.  The largest key of a lane is one of
// 32 lane maxima; at least topk experts have keys no smaller than the topk-th largest of those, so every expert of the
// answer has a key of at least that (less the error): a handful of candidates instead of topk rounds over all experts.
// They go to shared memory, one lane takes one of them and counts how many come before it.  If two candidates, or a
// group that stays and one that goes, are closer than the error bound, the warp works the keys concerned out in 64 bits
// and counts again; more than 32 candidates, too few available experts and infinite or NaN inputs go to route_lanes_f64.
// The weights come from the chosen experts' logits with full 32-bit functions, whatever the keys went through.
//
// What bounds it is the number of instructions, 500 to 800 warp instructions a token (the 17 MB of logits of 16384 tokens
// are 2.7 us of memory).  Measured, 256 experts, top 8: 16384 tokens 18.2 us with 4 of 8 groups (19.6 us when a close border
// works out all keys in 64 bits, not only those that may be among a group's best), 16.0 us without groups (63 us with
// everything in 64 bits and a round over all experts per choice), 4096 tokens 6.5 us, one token 3.1 us.  Tried:
// putting close tokens off to the CTA's end (fewer registers, but 21-22 us: the late ones are a tail), five or six CTAs an
// SM instead of four (spills, 23-28 us), eight or sixteen rounds of CTAs instead of one resident set (20.5 us, but 7.8-8.4
// us at 4096 tokens).
//
// Error of a key: __expf is off by 2 + 1.173 |x| ulp of itself, which a sigmoid turns into at most s (1 - s) (2 + 1.173
// |x|) 2^-23 < 0.8 * 2^-23; the sum and the approximate quotient add 3 ulp of s <= 1, adding the bias half an ulp of the
// key: below 5e-7 + 2^-24 |key|.  Softmax: expf is within 2 ulp of its rounded argument, p (2 + |x - max| / 2) 2^-23 <
// 2.2 * 2^-23 for p <= exp(x - max); the sum takes up to 31 additions in a lane and five across, its reciprocal and the
// product round once each, p * 38 * 2^-24: below 2.6e-6 + 2^-24 |key|.  Two keys can be told apart beyond twice that (the
// last bits of kTolRel are the comparison's own rounding).
constexpr float kTolSigmoid = 1.1e-6f, kTolSoftmax = 5.2e-6f, kTolRel = 2.4e-7f;

// Floats as integers of the same order (no NaN), for the integer reductions of a warp.
__device__ __forceinline__ int ordered_int(float v) {
  const int i = __float_as_int(v);
  return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }
__device__ __forceinline__ float warp_max_fast(float v) {
  return from_ordered(__reduce_max_sync(0xffffffffu, ordered_int(v)));
}

// The group stage in 64 bits: whether this lane's group stays, from the lane's two best keys (-inf: not there).
__device__ __forceinline__ bool route_keeps_f64(const RouteParams& p, int lane, int group_lanes, double b1, double b2) {
  for (int o = 1; o < group_lanes; o <<= 1) {
    const double o1 = __shfl_xor_sync(0xffffffffu, b1, o), o2 = __shfl_xor_sync(0xffffffffu, b2, o);
    b2 = fmax(fmax(b2, o2), fmin(b1, o1));
    b1 = fmax(b1, o1);
  }
  const double gs = p.group_top == 2 && b2 > -INFINITY ? b1 + b2 : b1;
  const int g = lane / group_lanes;
  int before = 0;
  for (int o = 0; o < p.n_group; ++o) {
    const double v = __shfl_sync(0xffffffffu, gs, o * group_lanes);
    before += v > gs || (v == gs && o < g);
  }
  return g < p.n_group && before < p.topk_group;
}

// What a close choice asks for: the 64-bit denominator of a softmax over finite logits, and a key.
__device__ __noinline__ double route_sum_f64(const RouteParams& p, size_t row, int lane, float top) {
  double v = 0.0;
  for (int e = lane; e < p.experts; e += 32) v += exp(static_cast<double>(route_logit(p, row + e)) - static_cast<double>(top));
  return warp_sum_f64(v);
}
__device__ __noinline__ double route_key_f64(const RouteParams& p, size_t row, int e, float top, double total) {
  const double x = route_logit(p, row + e);
  const double s = p.softmax ? exp(x - static_cast<double>(top)) / total : 1.0 / (1.0 + exp(-x));
  return s + (p.bias ? static_cast<double>(p.bias[e]) : 0.0);
}

// route_token_f64 for a lane that holds the PER experts from lane * PER on and groups that are runs of lanes: no shared
// memory, the lane's numbers in local memory.
template <int PER>
__device__ __noinline__ void route_lanes_f64(const RouteParams& p, int t, int lane, int group_lanes) {
  const double kOut = -INFINITY;
  const size_t row = static_cast<size_t>(t) * p.experts;
  const int e0 = lane * PER, mine = min(PER, p.experts - e0);
  double score[PER], key[PER];
  double top = kOut, sum = 0.0;
  if (p.softmax) {
#pragma unroll 1
    for (int j = 0; j < mine; ++j) top = fmax(top, static_cast<double>(route_logit(p, row + e0 + j)));   // passes NaN over
    top = warp_max_f64(top);
  }
#pragma unroll 1
  for (int j = 0; j < mine; ++j) {
    const double x = route_logit(p, row + e0 + j);
    double v;
    if (!p.softmax) v = 1.0 / (1.0 + exp(-x));
    else if (isinf(top)) v = x == top && top > 0 ? 1.0 : (x == x ? 0.0 : x);   // +inf logits share the row; all -inf: 0
    else v = exp(x - top);
    score[j] = v;
    if (v == v) sum += v;
  }
  sum = warp_sum_f64(sum);
  double b1 = kOut, b2 = kOut;
#pragma unroll 1
  for (int j = 0; j < mine; ++j) {
    if (p.softmax && sum > 0.0) score[j] /= sum;
    const double k = score[j] + (p.bias ? static_cast<double>(p.bias[e0 + j]) : 0.0);
    key[j] = k == k ? k : kOut;
    b2 = fmax(b2, fmin(b1, key[j]));
    b1 = fmax(b1, key[j]);
  }
  if (p.topk_group < p.n_group && !route_keeps_f64(p, lane, group_lanes, b1, b2))
#pragma unroll 1
    for (int j = 0; j < mine; ++j) key[j] = kOut;
  double picked = 0.0, my_score = 0.0;
  int my_idx = 0;
  for (int k = 0; k < p.topk; ++k) {
    double best = kOut;
    int best_e = 0x7fffffff;
#pragma unroll 1
    for (int j = 0; j < mine; ++j)
      if (key[j] == key[j] && (key[j] > best || best_e == 0x7fffffff)) { best = key[j]; best_e = e0 + j; }   // taken: NaN
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, best, o);
      const int oe = __shfl_xor_sync(0xffffffffu, best_e, o);
      if (oe != 0x7fffffff && (best_e == 0x7fffffff || ob > best || (ob == best && oe < best_e))) { best = ob; best_e = oe; }
    }
    const int owner = best_e / PER;
    double v = 0.0;
    if (lane == owner) {
      v = best > kOut ? score[best_e - e0] : 0.0;        // no expert left to choose: an unused id at weight 0
      key[best_e - e0] = __longlong_as_double(0x7ff8000000000000ll);
    }
    v = __shfl_sync(0xffffffffu, v, owner);
    picked += v;
    if (lane == k) { my_score = v; my_idx = best_e; }
  }
  if (lane < p.topk) {
    const double w = p.renormalize ? (picked > 0.0 ? my_score / picked : 0.0) : my_score;
    p.idx[static_cast<size_t>(t) * p.topk + lane] = my_idx;
    p.weights[static_cast<size_t>(t) * p.topk + lane] = static_cast<float>(w * p.route_scale);
  }
}

// FULL: every lane holds PER experts.
template <int PER, bool FULL>
__global__ void __launch_bounds__(256, PER <= 8 ? 4 : 2) moe_route_kernel(const RouteParams p, int group_lanes, int vec) {
  __shared__ __align__(16) float cand_key[8][32];
  __shared__ int cand_id[8][32];
  __shared__ double cand_key64[8][32];
  pdl_launch_dependents();
  pdl_wait();
  constexpr unsigned kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int e0 = lane * PER;
  const bool grouped = p.topk_group < p.n_group;
  // softmax without bias and groups orders like the logits
  const bool by_logit = p.softmax && !p.bias && !grouped;

  // this lane's experts of a row of fp32 numbers
  auto load = [&](const float* from, size_t row, bool vectors, float (&x)[PER]) {
    if constexpr (PER % 4 == 0) {
      if (vectors) {
        const float4* src = reinterpret_cast<const float4*>(from + row + e0);
#pragma unroll
        for (int j = 0; j < PER; j += 4) {
          const float4 v = FULL || e0 + j < p.experts ? __ldg(src + j / 4) : make_float4(0.f, 0.f, 0.f, 0.f);
          x[j] = v.x; x[j + 1] = v.y; x[j + 2] = v.z; x[j + 3] = v.w;
        }
        return;
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = FULL || e0 + j < p.experts ? __ldg(from + row + e0 + j) : 0.f;
  };
  const float tol_abs = p.softmax ? kTolSoftmax : kTolSigmoid;

  for (int t = blockIdx.x * warps + warp; t < p.tokens; t += gridDim.x * warps) {
    const size_t row = static_cast<size_t>(t) * p.experts;
    // A group border that 32 bits leave open is settled in 64 bits and the token begun again with that answer, so that its
    // registers are free meanwhile.
    bool slow = false, settled = false, stays = true;
    for (bool again = true; again;) {
      again = false;
      float x[PER], key[PER];
      if (p.logits_bf16) {
#pragma unroll
        for (int j = 0; j < PER; ++j) x[j] = FULL || e0 + j < p.experts ? route_logit(p, row + e0 + j) : 0.f;
      } else {
        load(static_cast<const float*>(p.logits), row, vec & 1, x);
      }
      float top = -INFINITY, sum = 0.f;
      bool odd = false;                              // an input that 32-bit keys do not handle
#pragma unroll
      for (int j = 0; j < PER; ++j) odd |= !(fabsf(x[j]) < INFINITY);
      if (p.softmax) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (FULL || e0 + j < p.experts) top = fmaxf(top, x[j]);
        top = warp_max_fast(odd ? 0.f : top);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const float v = FULL || e0 + j < p.experts ? expf(x[j] - top) : 0.f;
          key[j] = v;
          sum += v;
        }
        sum = warp_sum(sum);
      }
      const float inv = p.softmax ? 1.f / sum : 0.f;
      float bias[PER];
      if (p.bias) {
        load(p.bias, 0, vec & 2, bias);
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) bias[j] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        float k = by_logit ? x[j] : (p.softmax ? key[j] * inv : __fdividef(1.f, 1.f + __expf(-x[j])));
        k += bias[j];
        odd |= !(k < INFINITY);                      // NaN or +inf; -inf takes the expert out
        key[j] = FULL || e0 + j < p.experts ? k : -INFINITY;
      }
      slow = __any_sync(kAll, odd);
      if (settled) {
        if (!stays)
#pragma unroll
          for (int j = 0; j < PER; ++j) key[j] = -INFINITY;
      } else if (grouped && !slow) {
        float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          b2 = fmaxf(b2, fminf(b1, key[j]));
          b1 = fmaxf(b1, key[j]);
        }
        for (int o = 1; o < group_lanes; o <<= 1) {
          const float o1 = __shfl_xor_sync(kAll, b1, o), o2 = __shfl_xor_sync(kAll, b2, o);
          b2 = fmaxf(fmaxf(b2, o2), fminf(b1, o1));
          b1 = fmaxf(b1, o1);
        }
        const bool two = p.group_top == 2 && b2 > -INFINITY;
        const float gs = two ? b1 + b2 : b1;
        // the topk_group best by as many maxima; equal groups go together, and then there are too many
        constexpr int kNone = static_cast<int>(0x80000000u);
        const bool in = lane < p.n_group * group_lanes;
        const int mine = in ? ordered_int(gs) : kNone;
        int left = mine, at = kNone;
        for (int k = 0; k < p.topk_group; ++k) {
          at = __reduce_max_sync(kAll, left);
          if (left == at) left = kNone;
        }
        const bool kept = in && mine >= at;
        const float lo = from_ordered(at), hi = from_ordered(max(__reduce_max_sync(kAll, left), ordered_int(-FLT_MAX)));
        // A group that stays must lie above one that goes by more than the errors of both (two keys' each); a sum far
        // below any choice (a mask's) takes no part.
        const float err = gs > -1e30f ? tol_abs + kTolRel * (fabsf(b1) + (two ? fabsf(b2) : 0.f)) : 0.f;
        const float most = __int_as_float(__reduce_max_sync(kAll, in ? __float_as_int(err) : 0));
        if (at <= ordered_int(-FLT_MAX)) {
          slow = true;                               // fewer groups with an available expert than stay
        } else if (!(lo - hi > 2.f * most) || lo < -1e29f || __popc(__ballot_sync(kAll, kept)) != p.topk_group * group_lanes) {
          // only the keys that may be among the group's best, a lane's own one after the other: one or two of its PER
          const float cut = two ? b2 : b1, from = cut - (tol_abs + kTolRel * fabsf(cut));
          unsigned open = 0;
#pragma unroll
          for (int j = 0; j < PER; ++j) open |= static_cast<unsigned>(key[j] > -INFINITY && key[j] >= from) << j;
          const double total = p.softmax ? route_sum_f64(p, row, lane, top) : 1.0;
          double d1 = -INFINITY, d2 = -INFINITY;
#pragma unroll 1
          for (; open; open &= open - 1) {
            const double k = route_key_f64(p, row, e0 + __ffs(open) - 1, top, total);
            d2 = fmax(d2, fmin(d1, k));
            d1 = fmax(d1, k);
          }
          stays = route_keeps_f64(p, lane, group_lanes, d1, d2);
          settled = again = true;
          continue;
        }
        if (!kept)
#pragma unroll
          for (int j = 0; j < PER; ++j) key[j] = -INFINITY;
      }
      if (!slow) {
        float m = key[0];
#pragma unroll
        for (int j = 1; j < PER; ++j) m = fmaxf(m, key[j]);
        // the topk-th largest lane maximum, or less where maxima are equal
        int left = ordered_int(m), at_k = __reduce_max_sync(kAll, left);
        const float largest = from_ordered(at_k);
        for (int k = 1; k < p.topk; ++k) {
          if (left == at_k) left = static_cast<int>(0x80000000u);
          at_k = __reduce_max_sync(kAll, left);
        }
        const float kth = at_k > ordered_int(-FLT_MAX) ? from_ordered(at_k) : -INFINITY;
        const float tol = tol_abs + kTolRel * fmaxf(fabsf(largest), kth > -INFINITY ? fabsf(kth) : 0.f);
        // without topk lanes that hold an available expert every available one is a candidate
        const float least = kth > -INFINITY ? kth - tol : -FLT_MAX;
        int mine = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) mine += key[j] >= least;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(kAll, upto, o);
          if (lane >= o) upto += u;
        }
        const int n = __shfl_sync(kAll, upto, 31);
        slow = n > 32 || n < p.topk;
        if (!slow) {
          int at = upto - mine;
#pragma unroll
          for (int j = 0; j < PER; ++j)
            if (key[j] >= least) {
              cand_key[warp][at] = key[j];
              cand_id[warp][at] = e0 + j;
              ++at;
            }
          if (lane >= n) cand_key[warp][lane] = -INFINITY;
          __syncwarp();
          const float ki = cand_key[warp][lane];
          const int id = lane < n ? cand_id[warp][lane] : 0;
          const float xi = lane < n ? route_logit(p, row + id) : 0.f;
          // how many lie above, and how many above or too close to tell (itself among them): equal keys are close
          const float low = ki - tol;
          int rank = 0, above = 0;
          for (int j = 0; j < n; j += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(&cand_key[warp][j]);
            rank += (k4.x > ki) + (k4.y > ki) + (k4.z > ki) + (k4.w > ki);
            above += (k4.x >= low) + (k4.y >= low) + (k4.z >= low) + (k4.w >= low);
          }
          const bool near = lane < n && above != rank + 1;
          // Scores near the lowest 32-bit numbers lose the ratio that renormalising keeps, and no longer order like the
          // logits: 64 bits.
          if (__any_sync(kAll, lane < n && (p.softmax ? xi - top : xi) < -80.f)) {
            slow = true;
          } else if (__any_sync(kAll, near)) {
            const double total = p.softmax ? route_sum_f64(p, row, lane, top) : 1.0;
            const double k64 = lane < n ? route_key_f64(p, row, id, top, total) : 0.0;
            cand_key64[warp][lane] = k64;
            __syncwarp();
            rank = 0;
            for (int j = 0; j < n; ++j) {
              const double kj = cand_key64[warp][j];
              rank += kj > k64 || (kj == k64 && j < lane);
            }
          }
          if (!slow) {
            const bool chosen = lane < n && rank < p.topk;
            float s = 0.f;
            if (chosen) s = p.softmax ? expf(xi - top) * inv : __fdividef(1.f, 1.f + expf(-xi));
            const float picked = warp_sum(s);
            if (chosen) {
              const size_t o = static_cast<size_t>(t) * p.topk + rank;
              p.idx[o] = id;
              p.weights[o] = (p.renormalize ? (picked > 0.f ? s / picked : 0.f) : s) * p.route_scale;
            }
          }
        }
      }
    }
    if (slow) route_lanes_f64<PER>(p, t, lane, group_lanes);
    __syncwarp();                                      // the candidates are read before the next token's are written
  }
}

template <int PER>
int route_launch_per(const RouteParams& p, int group_lanes, cudaStream_t stream) {
  // 16-byte loads of the logits (1) and of the bias (2)
  const int vec = p.experts % 4 != 0 ? 0 : ((reinterpret_cast<uintptr_t>(p.logits) & 15) == 0 ? 1 : 0) |
                                                 ((reinterpret_cast<uintptr_t>(p.bias) & 15) == 0 ? 2 : 0);
  const int blocks = (p.tokens + 7) / 8, resident = sm_count() * 4;   // the CTAs that run at once
  launch_kernel(p.experts == 32 * PER ? moe_route_kernel<PER, true> : moe_route_kernel<PER, false>,
                dim3(blocks < resident ? blocks : resident), dim3(256), 0, stream, p, group_lanes, vec);
  return check_cuda(cudaGetLastError(), "moe_route_kernel launch");
}

}  // namespace

int moe_route_launch(const void* logits, int logits_dtype, const float* bias, int scoring, int tokens, int experts,
                     int n_group, int topk_group, int group_top, int topk, int renormalize, float route_scale,
                     int32_t* idx, float* weights, cudaStream_t stream) {
  PTO_REQUIRE(logits_dtype == PTO_FP32 || logits_dtype == PTO_BF16, "moe_route: logits must be fp32 or bf16");
  PTO_REQUIRE(scoring == PTO_SCORE_SIGMOID || scoring == PTO_SCORE_SOFTMAX, "moe_route: unknown scoring");
  PTO_REQUIRE(tokens >= 0 && tokens <= (1 << 30) && experts > 0 && experts <= kRouteMaxExperts, "moe_route: 1..1024 experts, at most 2^30 tokens");
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
  // experts per lane: a size the kernel is built for that covers them and, with groups, cuts no group inside a lane
  const int per_group = experts / n_group;
  for (int per : {1, 2, 3, 4, 5, 6, 8, 12, 16, 32}) {
    const int lanes = per_group / per;
    if (per * 32 < experts) continue;
    if (topk_group < n_group && (per_group % per != 0 || (lanes & (lanes - 1)) != 0)) continue;
    switch (per) {
      case 1: return route_launch_per<1>(p, lanes, stream);
      case 2: return route_launch_per<2>(p, lanes, stream);
      case 3: return route_launch_per<3>(p, lanes, stream);
      case 4: return route_launch_per<4>(p, lanes, stream);
      case 5: return route_launch_per<5>(p, lanes, stream);
      case 6: return route_launch_per<6>(p, lanes, stream);
      case 8: return route_launch_per<8>(p, lanes, stream);
      case 12: return route_launch_per<12>(p, lanes, stream);
      case 16: return route_launch_per<16>(p, lanes, stream);
      default: return route_launch_per<32>(p, lanes, stream);
    }
  }
  const size_t smem = sizeof(double) * kRouteWarps * static_cast<size_t>(2 * experts + n_group);
  if (smem > 48 * 1024)
    PTO_CUDA(cudaFuncSetAttribute(moe_route_any_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(sizeof(double) * kRouteWarps * 3 * kRouteMaxExperts)));
  launch_kernel(moe_route_any_kernel, dim3((tokens + kRouteWarps - 1) / kRouteWarps), dim3(kRouteWarps * 32), smem, stream, p);
  return check_cuda(cudaGetLastError(), "moe_route_any_kernel launch");
}

}  // namespace pto
