// FP8 linear layer with block scales: e4m3 operands, one fp32 scale per (row, 128 channels) of x and one per 128 x 128
// block of the weight.
//
//   out[m, n] = (acc[m, n] +) sum over K blocks kb of 128 channels of
//               x_scale[m, kb] * w_scale[n / 128, kb] * ( sum_{k in kb} x[m, k] * w[n, k] )
//
// It is the dense counterpart of the grouped expert GEMM (the numerics of the reference's block-scaled golden,
// tests/st/runtime/ops/test_matmul_mx.py:119-131, with fp32 scales per 128).  Products and sums are fp32; out is rounded
// once.  The order of additions depends on sizes and alignment alone: equal calls give equal bits.
#include "common.cuh"
#include "kernels.h"
#include "pair.cuh"

namespace pto {
namespace {

struct LinFp8Params {
  const uint8_t* x;         // [m, k]
  const float* x_scale;     // [m, kblocks]
  const uint8_t* w;         // [n, k]
  const float* w_scale;     // [ceil(n / 128), kblocks]
  const float* acc;         // [m, n] or NULL; may be out
  void* out;                // [m, n] bf16 or fp32
  int m, n, k, kblocks, out_bf16, vec;
  int* err;
};

__device__ __forceinline__ void store_out(const LinFp8Params& p, size_t o, float v) {
  if (p.acc) v += p.acc[o];
  if (p.out_bf16) static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(v);
  else static_cast<float*>(p.out)[o] = v;
}

// Four neighbouring outputs of row m, the first in column n (columns past the end are left alone).
__device__ __forceinline__ void store_out4(const LinFp8Params& p, int m, int n, float4 v) {
  const size_t o = static_cast<size_t>(m) * p.n + n;
  if (p.vec && n + 4 <= p.n) {      // rows of whole 4-element units on whole boundaries
    if (p.acc) {
      const float4 a = *reinterpret_cast<const float4*>(p.acc + o);
      v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
    }
    if (p.out_bf16) *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
    else *reinterpret_cast<float4*>(static_cast<float*>(p.out) + o) = v;
  } else {
    if (n < p.n) store_out(p, o, v.x);
    if (n + 1 < p.n) store_out(p, o + 1, v.y);
    if (n + 2 < p.n) store_out(p, o + 2, v.z);
    if (n + 3 < p.n) store_out(p, o + 3, v.w);
  }
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
  const int n_tiles = (p.n + kAnyTile - 1) / kAnyTile, mt = static_cast<int>(blockIdx.x) / n_tiles;
  const int n0 = (static_cast<int>(blockIdx.x) - mt * n_tiles) * kAnyTile, m0 = mt * kAnyTile;
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

// Whole-warp wait for the K loop: parked by the hardware for the short time that a try takes without a hint, and bounded
// by the number of tries instead of the clock.  Reading the timer costs about as much as the usual wait, and polling
// without parking takes issue slots from the products (2088 instead of 2297 TFLOP/s at 8192 x 28672 x 4096).
__device__ __forceinline__ bool mbar_try_once(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_park_warp(uint64_t* bar, uint32_t parity) {
  bool ok = mbar_try_once(bar, parity);
#pragma unroll 1
  for (int i = 0; i < (1 << 19) && !ok; ++i) ok = mbar_try_once(bar, parity);
  return __all_sync(0xffffffffu, ok) != 0;
}

// Loads that stay where they are written: the compiler moves an ordinary read-only load down to its use, and a scale that
// is fetched a K block ahead then arrives a memory latency late (300 of 950 cycles per K block).
__device__ __forceinline__ float ldg_ahead(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float4 ldg_ahead4(const float* p) {
  float4 v;
  asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

// ---------------------------------------------------------------------------
// Narrow tiles: 128 output features on the TMEM lanes, BN tokens in the columns, K split over a cluster.
//
// For few tokens the product reads the weight once and does little else, so the work is cut by weight bytes: one CTA
// takes 128 features and every S-th part of K, S CTAs of a cluster meet in one tile.  Warp 0 keeps the TMA ring full,
// warp 1 issues four MMAs per K block into one of four TMEM buffers, the promotion warps multiply the raw product of a
// K block by x_scale * w_scale -- a table of the CTA's own K blocks in shared memory, one number per token, the same
// for all lanes -- and add it up in fp32 registers.  The partial sums of a cluster are pushed to the CTA that owns their
// tokens through distributed shared memory and added in rank order: no atomics and no workspace.
// Features on the lanes, because the other way round a batch of one would use one lane in 128.  What bounds it is DRAM once
// it streams, and 3 us of set-up and first loads before: m = 1, n = 28672, k = 4096 takes 21.5 us (5.4 TB/s), m = 64
// 24.7 us, m = 1, n = 4096, k = 7168 9.4 us; a fetch of the partial sums by their owner instead of the push cost 2 to 20 us
// more (a round trip per rank and token).
// ---------------------------------------------------------------------------
constexpr int kNarrowBufs = 4;
constexpr int kNarrowMaxStages = 12;
constexpr uint32_t kWTileBytes = 128 * 128;

template <int BN>
struct Narrow {
  static constexpr int kCols = BN < 64 ? BN : 64;          // columns of one promotion warp
  static constexpr int kPromoWarps = 4 * (BN / kCols);
  static constexpr int kThreads = (2 + kPromoWarps) * 32;
  static constexpr int kCtasPerSm = BN <= 64 ? 2 : 1;
  static constexpr uint32_t kStageBytes = kWTileBytes + BN * 128;
  static constexpr int kTabStride = BN + 4;                // floats: rows of 16-byte units, neighbours on other banks
  static constexpr uint32_t kTmemCols = kNarrowBufs * BN < 32 ? 32 : kNarrowBufs * BN;
};

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ float4 lds_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

template <int BN>
__global__ void __launch_bounds__(Narrow<BN>::kThreads, Narrow<BN>::kCtasPerSm)
linear_fp8_narrow_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                         const LinFp8Params p, int token_tiles, int split, int stages, int kb_max) {
  using C = Narrow<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* table = reinterpret_cast<float*>(smem + static_cast<size_t>(stages) * C::kStageBytes);   // [kb_max][kTabStride]
  float* recv = reinterpret_cast<float*>(smem);            // after the K loop, over the stages: [split][per][128]
  const int per = (BN + split - 1) / split;                // tokens of the tile that this CTA adds up and stores
  uint64_t* full = reinterpret_cast<uint64_t*>(table + kb_max * C::kTabStride);
  uint64_t* empty = full + kNarrowMaxStages;
  uint64_t* pfull = empty + kNarrowMaxStages;
  uint64_t* pempty = pfull + kNarrowBufs;
  uint64_t* drain = pempty + kNarrowBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = static_cast<int>(blockIdx.x) / split, rank = static_cast<int>(blockIdx.x) - tile * split;
  const int nt = tile / token_tiles, tt = tile - nt * token_tiles;
  const int kb0 = static_cast<int>(static_cast<long long>(p.kblocks) * rank / split);
  const int kbs = static_cast<int>(static_cast<long long>(p.kblocks) * (rank + 1) / split) - kb0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kNarrowBufs; ++i) {
      mbar_init(&pfull[i], 1);
      mbar_init(&pempty[i], C::kPromoWarps);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_x);
  }
  if (warp == 1) tmem_alloc(tmem_slot, C::kTmemCols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // Not before this CTA holds its tensor memory: a kernel that starts early could otherwise take it and then wait for
  // this grid to end.
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tmem_base = *tmem_slot;

  float acc[C::kCols];
  const int pw = warp - 2, q = warp & 3, c0 = (pw >> 2) * C::kCols;   // promotion: lane quarter, first column
  if (warp == 0) {
    // ------------------------------ TMA producer ------------------------------
    int s = 0;
    uint32_t ph = 1;
    for (int kb = 0; kb < kbs; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait(&empty[s], ph))) {
        if (lane == 0) report_error(p.err, kErrBarrierTimeout, 100, kb);
        break;
      }
      if (elect_one()) {
        uint8_t* st = smem + static_cast<size_t>(s) * C::kStageBytes;
        mbar_arrive_expect_tx(&full[s], C::kStageBytes);
        tma_load_2d(st, &tm_w, (kb0 + kb) * 128, nt * 128, &full[s]);           // past the matrix: zeros
        tma_load_2d(st + kWTileBytes, &tm_x, (kb0 + kb) * 128, tt * BN, &full[s]);
      }
      __syncwarp();
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer -------------------------------
    const uint32_t idesc = umma_idesc(128, BN, 0, 0);
    const uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);   // stride byte offset, version, 128-byte swizzle
    const uint32_t lo0 = ((smem_u32(smem) & 0x3FFFFu) >> 4) | (1u << 16);
    int s = 0;
    uint32_t ph = 0;
    for (int kb = 0; kb < kbs; ++kb) {
      const uint32_t b = kb & 3u, bph = ((kb >> 2) & 1u) ^ 1u;
      const bool ok = mbar_wait(&full[s], ph) && mbar_wait(&pempty[b], bph);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) report_error(p.err, kErrBarrierTimeout, 101, kb);
        break;
      }
      tc_fence_after_sync();
      if (elect_one()) {
        const uint32_t w_lo = lo0 + s * (C::kStageBytes >> 4), x_lo = w_lo + (kWTileBytes >> 4);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)   // 32 bytes of K per MMA
          umma_fp8(tmem_base + b * BN, (static_cast<uint64_t>(desc_hi) << 32) | (w_lo + 2 * k),
                   (static_cast<uint64_t>(desc_hi) << 32) | (x_lo + 2 * k), idesc, k > 0 ? 1u : 0u);
        umma_commit(&empty[s]);
        umma_commit(&pfull[b]);
      }
      __syncwarp();
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
    // tensor memory is released only after every MMA has completed, also when a wait gave up
    if (elect_one()) {
      umma_commit(drain);
      if (!mbar_wait(drain, 0)) report_error(p.err, kErrBarrierTimeout, 103, 0);
    }
    __syncwarp();
  } else {
    // -------------------------------- promotion --------------------------------
    // the table: x_scale[token, kb] * w_scale[tile, kb] (tokens past the end read the last row and are not stored)
    constexpr int kPromoThreads = C::kPromoWarps * 32;
    const float* wsp = p.w_scale + static_cast<size_t>(nt) * p.kblocks + kb0;
    constexpr int kAhead = 8;      // entries of a thread under way at once: the table is on the way to the first result
    for (int i0 = threadIdx.x - 64; i0 < kbs * BN; i0 += kAhead * kPromoThreads) {
      float sx[kAhead], sw[kAhead];
      int at[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = min(i0 + a * kPromoThreads, kbs * BN - 1), j = i / kbs, kb = i - j * kbs, t = min(tt * BN + j, p.m - 1);
        at[a] = kb * C::kTabStride + j;
        sx[a] = ldg_ahead(p.x_scale + static_cast<size_t>(t) * p.kblocks + kb0 + kb);
        sw[a] = ldg_ahead(wsp + kb);
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) table[at[a]] = sx[a] * sw[a];
    }
    named_bar_sync(1, kPromoThreads);
#pragma unroll
    for (int j = 0; j < C::kCols; ++j) acc[j] = 0.f;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + c0;
    uint32_t tab = smem_u32(table) + c0 * 4;
    for (int kb = 0; kb < kbs; ++kb, tab += C::kTabStride * 4) {
      const uint32_t b = kb & 3u;
      if (!mbar_wait_warp(&pfull[b], (kb >> 2) & 1u)) {
        if (lane == 0) report_error(p.err, kErrBarrierTimeout, 102, kb);
        break;
      }
      tc_fence_after_sync();
      uint32_t raw[C::kCols / 16][16];
#pragma unroll
      for (int c = 0; c < C::kCols / 16; ++c) tmem_ld_32x16(taddr + b * BN + c * 16, raw[c]);
      tmem_ld_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&pempty[b]);
#pragma unroll
      for (int j = 0; j < C::kCols; j += 4) {
        const float4 sc = lds_f32x4(tab + j * 4);
        acc[j] = fmaf(__uint_as_float(raw[j / 16][j % 16]), sc.x, acc[j]);
        acc[j + 1] = fmaf(__uint_as_float(raw[j / 16][j % 16 + 1]), sc.y, acc[j + 1]);
        acc[j + 2] = fmaf(__uint_as_float(raw[j / 16][j % 16 + 2]), sc.z, acc[j + 2]);
        acc[j + 3] = fmaf(__uint_as_float(raw[j / 16][j % 16 + 3]), sc.w, acc[j + 3]);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, C::kTmemCols);
  // Token j of the tile is added up by rank j / per: every CTA stores its partial sums there, [rank][token][feature],
  // over operand stages that no CTA of the cluster reads any more.
  if (split > 1) cluster_sync_all();
  if (warp >= 2) {
    const uint32_t mine = smem_u32(recv) + (rank * per * 128 + q * 32 + lane) * 4;
    int owner = c0 / per, slot = c0 - owner * per;
    uint32_t to = split > 1 ? mapa_u32(mine, owner) : mine;
#pragma unroll
    for (int j = 0; j < C::kCols; ++j) {
      st_cluster_f32(to + slot * 512, acc[j]);
      if (++slot == per && j + 1 < C::kCols) {
        slot = 0;
        ++owner;
        to = mapa_u32(mine, owner);
      }
    }
  }
  if (split > 1) cluster_sync_all();
  else __syncthreads();
  if (warp >= 2) {
    // a warp adds up a token's 128 features, four to a lane, in rank order
    const int first = tt * BN + rank * per, count = min(min(per, BN - rank * per), p.m - first);
    for (int t = pw; t < count; t += C::kPromoWarps) {
      const uint32_t from = smem_u32(recv) + (t * 128 + lane * 4) * 4;
      float4 v = lds_f32x4(from);
      for (int r = 1; r < split; ++r) {
        const float4 a = lds_f32x4(from + r * per * 512);
        v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
      }
      store_out4(p, first + t, nt * 128 + lane * 4, v);
    }
  }
}

size_t narrow_fixed_bytes(int bn, int kb_max);
size_t narrow_budget(int bn);

template <int BN>
int narrow_launch(const LinFp8Params& p, int split, cudaStream_t stream) {
  using C = Narrow<BN>;
  const int token_tiles = (p.m + BN - 1) / BN, feature_tiles = (p.n + 127) / 128;
  const int kb_max = (p.kblocks + split - 1) / split;
  static_assert(C::kTabStride == BN + 4 && (C::kCtasPerSm == 2) == (BN <= 64), "narrow_split sizes the same tile");
  const size_t fixed = narrow_fixed_bytes(BN, kb_max), budget = narrow_budget(BN);
  int stages = fixed < budget ? static_cast<int>((budget - fixed) / C::kStageBytes) : 0;
  if (stages > kNarrowMaxStages) stages = kNarrowMaxStages;
  PTO_REQUIRE(stages >= 2 && static_cast<size_t>(stages) * C::kStageBytes >= static_cast<size_t>(split) * ((BN + split - 1) / split) * 512,
              "linear_fp8: k does not fit the scale table of a tile");
  // never less than a third of an SM: with at most 256 TMEM columns a CTA, those on one SM cannot ask for more than 512
  const size_t smem = fixed + static_cast<size_t>(stages) * C::kStageBytes;
  CUtensorMap tm_w, tm_x;
  int st = make_tensor_map_2d(&tm_w, p.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.n, p.k, p.k, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != kOk) return st;
  st = make_tensor_map_2d(&tm_x, p.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.m, p.k, p.k, 128, BN, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != kOk) return st;
  constexpr int kUseKey = BN == 16 ? 8 : (BN == 32 ? 9 : (BN == 64 ? 10 : 11));
  if (first_use_on_device(kUseKey))
    PTO_CUDA(cudaFuncSetAttribute(linear_fp8_narrow_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
  const long long ctas = static_cast<long long>(token_tiles) * feature_tiles * split;
  PTO_REQUIRE(ctas < (1ll << 31), "linear_fp8: problem too large");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  PTO_CUDA(cudaLaunchKernelEx(&cfg, linear_fp8_narrow_kernel<BN>, tm_w, tm_x, p, token_tiles, split, stages, kb_max));
  return check_cuda(cudaGetLastError(), "linear_fp8_narrow_kernel launch");
}

// Shared memory of a CTA without its stages.
size_t narrow_fixed_bytes(int bn, int kb_max) {
  return 1024 + sizeof(float) * static_cast<size_t>(kb_max) * (bn + 4) + 8 * (2 * kNarrowMaxStages + 2 * kNarrowBufs + 1) + 16;
}
size_t narrow_budget(int bn) { return (bn <= 64 ? 113 : 227) * 1024; }

// K split over up to eight CTAs of a cluster: as many CTAs as run at once (a second round costs its own start-up:
// m = 1, n = 28672, k = 4096 takes 21 us unsplit and 25 us split in two), two K blocks at least for each.  More when the
// scale table of a longer part would leave less than three stages.  0: K is too long for this kernel.
int narrow_split(const LinFp8Params& p, int bn) {
  const long long tiles = static_cast<long long>((p.m + bn - 1) / bn) * ((p.n + 127) / 128);
  long long s = static_cast<long long>(sm_count()) * (bn <= 64 ? 2 : 1) / tiles;
  if (s > p.kblocks / 2) s = p.kblocks / 2;
  s = s < 1 ? 1 : (s > 8 ? 8 : s);
  const size_t stage = kWTileBytes + static_cast<size_t>(bn) * 128;
  while (s <= 8 && narrow_fixed_bytes(bn, static_cast<int>((p.kblocks + s - 1) / s)) + 3 * stage > narrow_budget(bn)) ++s;
  return s > 8 ? 0 : static_cast<int>(s);
}

// ---------------------------------------------------------------------------
// Wide tiles on pairs of SMs (tcgen05.mma.cta_group::2): 256 tokens x 256 features.
//
// Each CTA of a pair keeps 128 token rows on its TMEM lanes and loads its own rows and half of the weight rows: 32 KB per
// K block for 128 x 256 x 128 products of its own.  A K block must leave the tensor core on its own, because its scale
// differs from the next one's: its raw product goes to TMEM and from there, times x_scale[row, kb] * w_scale[128
// features, kb] -- one number for a thread, which owns one row -- into fp32 registers.  The 256 columns are two
// halves of 128 with two TMEM buffers each: four promotion warps work for either half, and while one buffer of a half
// is drained the tensor core fills the other three.  A half has an issuer warp of its own, since one thread takes most
// of a K block's tensor time to issue its MMAs and commits.
//   full[s]        in the leader (the even CTA), bytes of both CTAs' loads
//   empty[s]       in each CTA, two arrivals: the commits of both issuers
//   pfull[h][b]    in each CTA, the commit of issuer h
//   pempty[h][b]   in the leader, eight arrivals: four promotion warps of either CTA
// No load is multicast; every mbarrier wait is bounded; the cluster barriers are reached by every thread on every path.
// What bounds it is the way round tensor core -> TMEM -> promotion -> tensor core: 840 cycles per K block where the MMAs take
// 512 (the tensor pipe is 63 % active), and under sustained load the power cap.  8192 x 28672 x 4096: 0.82 ms in short
// runs (2.34 PFLOP/s), 0.94 ms sustained; with single CTAs and 128-token tiles it was 1.69 ms.
// Scalar FMAs: a packed fma.rn.f32x2 holds the pipe for three cycles here and cost 3 % more time.
// ---------------------------------------------------------------------------
constexpr int kPairThreads = 12 * 32;                       // producer, two issuers, one idle; eight promotion warps
// 128 accumulators a thread need more than the 168 registers that 384 threads start with: the first four warps give
// some of theirs up.  What is asked for afterwards must not be more than the block was launched with, or the
// request waits for ever: pair_launch checks the kernel's register count.
constexpr int kPairRegs = 168, kPairRoleRegs = 56, kPairPromoRegs = 224;
static_assert(128 * kPairRoleRegs + 256 * kPairPromoRegs <= kPairThreads * kPairRegs, "register split");
constexpr int kPairStages = 6;
constexpr uint32_t kPairStageBytes = 2 * 128 * 128;
constexpr uint32_t kPairStoreBytes = 4096;                  // per promotion warp: 32 rows of 128 bytes on their way out

// Waits for the TMEM loads; the registers pass through, so that their uses stay behind the wait.
__device__ __forceinline__ void tmem_ld_wait_regs(uint32_t (&a)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(a[0]), "+r"(a[1]), "+r"(a[2]), "+r"(a[3]), "+r"(a[4]), "+r"(a[5]), "+r"(a[6]), "+r"(a[7]),
                 "+r"(a[8]), "+r"(a[9]), "+r"(a[10]), "+r"(a[11]), "+r"(a[12]), "+r"(a[13]), "+r"(a[14]), "+r"(a[15])
               :
               : "memory");
}

template <bool SCALE4>
__device__ __forceinline__ float4 load_scales(const float* p, int kb, int kblocks) {
  if (SCALE4) return ldg_ahead4(p + min(kb, kblocks - 4));
  return make_float4(ldg_ahead(p + min(kb, kblocks - 1)), ldg_ahead(p + min(kb + 1, kblocks - 1)),
                     ldg_ahead(p + min(kb + 2, kblocks - 1)), ldg_ahead(p + min(kb + 3, kblocks - 1)));
}

__device__ __forceinline__ void sts_u32x4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// SCALE4: K blocks come in fours and the scale arrays are 16-byte aligned, so four scales are one load.
template <bool SCALE4>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
linear_fp8_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, const LinFp8Params p,
                       int m_tiles, int n_tiles, int group, int vec8) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* store = smem + static_cast<size_t>(kPairStages) * kPairStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(store + 8 * kPairStoreBytes);
  uint64_t* empty = full + kPairStages;
  uint64_t* pfull = empty + kPairStages;      // [half][buffer]
  uint64_t* pempty = pfull + 4;
  uint64_t* drain = pempty + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();          // 0 = leader
  const int pair = static_cast<int>(blockIdx.x >> 1), npairs = static_cast<int>(gridDim.x >> 1);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPairStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&pfull[i], 1);
      mbar_init(&pempty[i], 8);
    }
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    fence_barrier_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);   // the same warp in each CTA of the pair, together
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();              // both CTAs' barriers are initialised before anything is signalled across the pair
  tc_fence_after_sync();
  pdl_launch_dependents();         // not before this CTA holds its tensor memory
  pdl_wait();
  const uint32_t tmem_base = *tmem_slot;
  const int tiles = m_tiles * n_tiles;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairRoleRegs));
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairPromoRegs));
  }
  if (warp == 0) {
    // ------------------------------ TMA producer (both CTAs) ------------------------------
    uint32_t s = 0, ph = 1;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += npairs) {
      int mt, nt;
      grouped_tile_coords(tile, group, m_tiles, n_tiles, mt, nt);
      const int row = mt * 256 + static_cast<int>(rank) * 128, feat = nt * 256 + static_cast<int>(rank) * 64;
      for (int kb = 0; kb < p.kblocks; ++kb) {
        if (!mbar_park_warp(&empty[s], ph)) {
          if (lane == 0) report_error(p.err, kErrBarrierTimeout, 110, kb);
          ok = false;
          break;
        }
        if (elect_one()) {
          uint8_t* st = smem + static_cast<size_t>(s) * kPairStageBytes;
          const uint32_t leader_full = mapa_u32(smem_u32(&full[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kPairStageBytes);
          tma_load_2d_pair(st, &tm_x, kb * 128, row, leader_full);                    // past the matrix: zeros
          tma_load_2d_pair(st + 16384, &tm_w, kb * 128, feat, leader_full);           // first half: 64 rows of each CTA
          tma_load_2d_pair(st + 24576, &tm_w, kb * 128, feat + 128, leader_full);     // second half
        }
        __syncwarp();
        if (++s == kPairStages) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
  } else if (warp < 3) {
    // ------------------------------- MMA issuers (leader only) -------------------------------
    if (rank == 0) {
      const uint32_t h = static_cast<uint32_t>(warp - 1);
      const uint32_t idesc = umma_idesc(256, 128, 0, 0);
      const uint32_t desc_hi = (1024u >> 4) | (1u << 14) | (2u << 29);   // stride byte offset, version, 128-byte swizzle
      const uint32_t lo0 = ((smem_u32(smem) & 0x3FFFFu) >> 4) | (1u << 16);
      const long long my_tiles = pair < tiles ? (tiles - 1 - pair) / npairs + 1 : 0;
      const uint32_t total = static_cast<uint32_t>(my_tiles * p.kblocks);
      uint32_t s = 0, ph = 0;
      for (uint32_t i = 0; i < total; ++i) {
        const uint32_t b = i & 1u;
        if (!mbar_park_warp(&full[s], ph) || !mbar_park_warp(&pempty[h * 2 + b], ((i >> 1) & 1u) ^ 1u)) {
          if (lane == 0) report_error(p.err, kErrBarrierTimeout, 111, static_cast<int>(i));
          break;
        }
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t x_lo = lo0 + s * (kPairStageBytes >> 4), w_lo = x_lo + ((16384 + h * 8192) >> 4);
          const uint32_t d = tmem_base + (h * 2 + b) * 128;
#pragma unroll
          for (uint32_t k = 0; k < 4; ++k)   // 32 bytes of K per MMA
            umma_fp8_pair(d, (static_cast<uint64_t>(desc_hi) << 32) | (x_lo + 2 * k),
                          (static_cast<uint64_t>(desc_hi) << 32) | (w_lo + 2 * k), idesc, k > 0 ? 1u : 0u);
          umma_commit_pair(&pfull[h * 2 + b]);
          umma_commit_pair(&empty[s]);
        }
        __syncwarp();
        if (++s == kPairStages) {
          s = 0;
          ph ^= 1u;
        }
      }
      // no CTA of the pair releases tensor memory before every MMA has completed, also when a wait gave up
      if (elect_one()) {
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(&drain[h])) : "memory");
        if (!mbar_wait(&drain[h], 0)) report_error(p.err, kErrBarrierTimeout, 113, 0);
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ------------------------- promotion and epilogue (both CTAs) -------------------------
    const int pw = warp - 4, h = pw >> 2, q = warp & 3;
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(h) * 256;
    const uint32_t my_store = smem_u32(store) + pw * kPairStoreBytes;
    const uint32_t free0 = mapa_u32(smem_u32(&pempty[h * 2]), 0), free1 = mapa_u32(smem_u32(&pempty[h * 2 + 1]), 0);
    const int n_blocks = (p.n + 127) / 128;
    uint32_t i = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += npairs) {
      int mt, nt;
      grouped_tile_coords(tile, group, m_tiles, n_tiles, mt, nt);
      const int row0 = mt * 256 + static_cast<int>(rank) * 128 + q * 32, col0 = nt * 256 + h * 128;
      const float* xs = p.x_scale + static_cast<size_t>(min(row0 + lane, p.m - 1)) * p.kblocks;
      const float* ws = p.w_scale + static_cast<size_t>(min(nt * 2 + h, n_blocks - 1)) * p.kblocks;
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.f;
      // One K block: its raw product times `sc` onto the accumulators; b = its TMEM buffer, ph the phase to wait for.
      auto block = [&](float sc, uint32_t b, uint32_t ph) {
        if (!mbar_park_warp(&pfull[h * 2 + b], ph)) {
          if (lane == 0) report_error(p.err, kErrBarrierTimeout, 112, static_cast<int>(i));
          ok = false;
          return;
        }
        tc_fence_after_sync();
        const uint32_t t = lane_base + b * 128;
        uint32_t raw[2][16];
        tmem_ld_32x16(t, raw[0]);
#pragma unroll
        for (int g = 0; g < 8; ++g) {      // sixteen columns at a time, the next sixteen in flight during the products
          tmem_ld_wait_regs(raw[g & 1]);
          if (g < 7) {
            tmem_ld_32x16(t + (g + 1) * 16, raw[(g + 1) & 1]);
          } else {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_peer(b ? free1 : free0);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[g * 16 + j] = fmaf(__uint_as_float(raw[g & 1][j]), sc, acc[g * 16 + j]);
        }
      };
      // Scales four K blocks at a time, fetched four blocks ahead; what lies past the end is clamped and not used.
      float4 x4 = load_scales<SCALE4>(xs, 0, p.kblocks), w4 = load_scales<SCALE4>(ws, 0, p.kblocks);
      for (int kb = 0; kb < p.kblocks && ok; kb += 4) {
        const float s0 = x4.x * w4.x, s1 = x4.y * w4.y, s2 = x4.z * w4.z, s3 = x4.w * w4.w;
        x4 = load_scales<SCALE4>(xs, kb + 4, p.kblocks);
        w4 = load_scales<SCALE4>(ws, kb + 4, p.kblocks);
        if (SCALE4) {       // a tile starts at a multiple of four K blocks
          const uint32_t ph = (i >> 1) & 1u;
          block(s0, 0, ph);
          if (ok) block(s1, 1, ph);
          if (ok) block(s2, 0, ph ^ 1u);
          if (ok) block(s3, 1, ph ^ 1u);
          i += 4;
        } else {
          const int n = min(4, p.kblocks - kb);
          for (int j = 0; j < n && ok; ++j, ++i)
            block(j == 0 ? s0 : (j == 1 ? s1 : (j == 2 ? s2 : s3)), i & 1u, (i >> 1) & 1u);
        }
      }
      if (!ok) break;
      // Out through shared memory, 32 rows of 128 bytes at a time (16-byte units swizzled by row), so that a store
      // instruction writes whole lines: with every lane on a row of its own the stores cost as much as the K loop.
      if (vec8) {         // bf16, nothing to add: 64 columns at a time
#pragma unroll
        for (int part = 0; part < 2; ++part) {
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(acc[part * 64 + u * 8 + 2 * j], acc[part * 64 + u * 8 + 2 * j + 1]);
            sts_u32x4(my_store + lane * 128 + ((u ^ (lane & 7)) << 4), o[0], o[1], o[2], o[3]);
          }
          __syncwarp();
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int rr = r * 4 + (lane >> 3), cc = lane & 7, col = col0 + part * 64 + cc * 8;
            const float4 v = lds_f32x4(my_store + rr * 128 + ((cc ^ (rr & 7)) << 4));
            if (row0 + rr < p.m && col < p.n)
              *reinterpret_cast<float4*>(static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(row0 + rr) * p.n + col) = v;
          }
          __syncwarp();
        }
      } else {
#pragma unroll
        for (int part = 0; part < 4; ++part) {
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float* v = acc + part * 32 + u * 4;
            sts_u32x4(my_store + lane * 128 + ((u ^ (lane & 7)) << 4), __float_as_uint(v[0]), __float_as_uint(v[1]),
                      __float_as_uint(v[2]), __float_as_uint(v[3]));
          }
          __syncwarp();
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int rr = r * 4 + (lane >> 3), cc = lane & 7;
            const float4 v = lds_f32x4(my_store + rr * 128 + ((cc ^ (rr & 7)) << 4));
            if (row0 + rr < p.m) store_out4(p, row0 + rr, col0 + part * 32 + cc * 4, v);
          }
          __syncwarp();
        }
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();   // neither CTA leaves, or frees tensor memory, while its partner may still signal or read it
  if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

int pair_launch(const LinFp8Params& p, cudaStream_t stream) {
  const int m_tiles = (p.m + 255) / 256, n_tiles = (p.n + 255) / 256;
  const long long tiles = static_cast<long long>(m_tiles) * n_tiles;
  PTO_REQUIRE(tiles * p.kblocks < (1ll << 31), "linear_fp8: problem too large");
  const int pairs = tiles < sm_count() / 2 ? static_cast<int>(tiles) : sm_count() / 2;
  const size_t smem = 1024 + static_cast<size_t>(kPairStages) * kPairStageBytes + 8 * kPairStoreBytes + 8 * (2 * kPairStages + 10) + 16;
  CUtensorMap tm_x, tm_w;
  int st = make_tensor_map_2d(&tm_x, p.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.m, p.k, p.k, 128, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != kOk) return st;
  st = make_tensor_map_2d(&tm_w, p.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.n, p.k, p.k, 128, 64, CU_TENSOR_MAP_SWIZZLE_128B);
  if (st != kOk) return st;
  static const int regs = [] {
    cudaFuncAttributes f4, f1;
    if (cudaFuncGetAttributes(&f4, linear_fp8_pair_kernel<true>) != cudaSuccess ||
        cudaFuncGetAttributes(&f1, linear_fp8_pair_kernel<false>) != cudaSuccess)
      return 0;
    return f4.numRegs < f1.numRegs ? f4.numRegs : f1.numRegs;
  }();
  if (regs < kPairRegs) return fail(kUnsupported, "linear_fp8: the pair kernel has too few registers for its split");
  if (first_use_on_device(12)) {
    PTO_CUDA(cudaFuncSetAttribute(linear_fp8_pair_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    PTO_CUDA(cudaFuncSetAttribute(linear_fp8_pair_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
  }
  const int vec8 = p.out_bf16 && !p.acc && p.n % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
  const bool scale4 = p.kblocks % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.x_scale) | reinterpret_cast<uintptr_t>(p.w_scale)) & 15) == 0;
  launch_kernel(scale4 ? linear_fp8_pair_kernel<true> : linear_fp8_pair_kernel<false>, dim3(2 * pairs), dim3(kPairThreads), smem,
                stream, tm_x, tm_w, p, m_tiles, n_tiles, 16, vec8);
  return check_cuda(cudaGetLastError(), "linear_fp8_pair_kernel launch");
}

// Which tile: the time of each in nanoseconds, from a start-up, a cost per round of tiles and a cost per K block that fit the
// measurements (us; 128-token / 32-token narrow tiles / pair): 256 x 4096 x 4096 12.4 / 16.4 / 20.7;  512 x 4096 x 4096
// 18.7 / - / 19.4;  1024 x 1024 x 4096 12.1 / - / 16.9;  777 x 1000 x 2000 9.4 / 11.7 / 11.6;  300 x 640 x 4096 8.6 / 7.7 / -;
// 150 x 512 x 512 7.8 / 4.4 / -;  1024 x 4096 x 4096 36.3 / - / 17.7;  256 x 28672 x 4096 71.3 / - / 34.4.  A pair is not
// asked up to 64 tokens (64 x 28672 x 4096: 25.4 narrow, 30.3 pair).
long long narrow_time(const LinFp8Params& p, int bn, int split) {
  const long long ctas = static_cast<long long>((p.m + bn - 1) / bn) * ((p.n + 127) / 128) * split;
  const long long slots = static_cast<long long>(sm_count()) * (bn <= 64 ? 2 : 1), rounds = (ctas + slots - 1) / slots;
  const long long start = bn <= 32 ? 1800 : (bn <= 64 ? 2400 : 3000);
  return 2000 + rounds * (start + 450ll * ((p.kblocks + split - 1) / split)) + (split > 1 ? (bn <= 64 ? 300 : 1000) : 0);
}
long long pair_time(const LinFp8Params& p) {
  const long long tiles = static_cast<long long>((p.m + 255) / 256) * ((p.n + 255) / 256), pairs = sm_count() / 2;
  return 3000 + (tiles + pairs - 1) / pairs * (1500 + 410ll * p.kblocks);
}

}  // namespace

int linear_fp8_launch(const void* x, const float* x_scale, const void* w, const float* w_scale, const float* acc, void* out,
                      int out_dtype, int m, int n, int k, int* err, cudaStream_t stream) {
  PTO_REQUIRE(m >= 0 && n > 0 && k > 0, "linear_fp8: n and k must be positive, m not negative");
  PTO_REQUIRE(m <= (1 << 30) && n <= (1 << 30) && k <= (1 << 30), "linear_fp8: sizes up to 2^30");
  PTO_REQUIRE(out_dtype == PTO_BF16 || out_dtype == PTO_FP32, "linear_fp8: out must be bf16 or fp32");
  if (m == 0) return kOk;
  PTO_REQUIRE(x && x_scale && w && w_scale && out, "linear_fp8: NULL tensor");
  PTO_REQUIRE(!(acc && acc == out && out_dtype != PTO_FP32), "linear_fp8: only an fp32 out may be the tensor that is added");
  const size_t outputs = static_cast<size_t>(m) * n;
  PTO_REQUIRE(acc == out || !overlaps(out, outputs * (out_dtype == PTO_BF16 ? 2 : 4), acc, outputs * 4), "linear_fp8: out overlaps acc");
  LinFp8Params p;
  p.x = static_cast<const uint8_t*>(x); p.x_scale = x_scale; p.w = static_cast<const uint8_t*>(w); p.w_scale = w_scale;
  p.acc = acc; p.out = out; p.m = m; p.n = n; p.k = k; p.kblocks = (k + 127) / 128; p.out_bf16 = out_dtype == PTO_BF16;
  p.err = err;
  p.vec = n % 4 == 0 && ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(acc)) & 15) == 0;
  const bool tma = k % 16 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0;
  if (tma) {
    int bn = m <= 16 ? 16 : (m <= 32 ? 32 : (m <= 64 ? 64 : 128)), split = narrow_split(p, bn);
    if (m > 32) {       // more and smaller tiles where the problem is small
      const int split32 = narrow_split(p, 32);
      if (split32 && (!split || narrow_time(p, 32, split32) < narrow_time(p, bn, split))) {
        bn = 32;
        split = split32;
      }
    }
    if (split == 0 || (m > 64 && pair_time(p) < narrow_time(p, bn, split))) return pair_launch(p, stream);
    switch (bn) {
      case 16: return narrow_launch<16>(p, split, stream);
      case 32: return narrow_launch<32>(p, split, stream);
      case 64: return narrow_launch<64>(p, split, stream);
      default: return narrow_launch<128>(p, split, stream);
    }
  }
  const long long tiles = ((m + kAnyTile - 1ll) / kAnyTile) * ((n + kAnyTile - 1ll) / kAnyTile);
  PTO_REQUIRE(tiles < (1ll << 31), "linear_fp8: problem too large");
  launch_kernel(linear_fp8_any_kernel, dim3(static_cast<unsigned>(tiles)), dim3(256), 0, stream, p);
  return check_cuda(cudaGetLastError(), "linear_fp8_any_kernel launch");
}

}  // namespace pto
