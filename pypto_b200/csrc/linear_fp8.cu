// FP8 linear layer with block scales: e4m3 operands, one fp32 scale per (row, 128 channels) of x and one per 128 x 128
// block of the weight.
//
//   out[m, n] = (acc[m, n] +) sum over K blocks kb of 128 channels of
//               x_scale[m, kb] * w_scale[n / 128, kb] * ( sum_{k in kb} x[m, k] * w[n, k] )
//
// It is the dense counterpart of the grouped expert GEMM (the numerics of the reference's block-scaled golden,
// tests/st/runtime/ops/test_matmul_mx.py:119-131, with fp32 scales per 128).  Products and sums are fp32; out is rounded
// once.  The order of additions depends on the sizes alone: equal calls give equal bits.
#include <cstdlib>
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

// ---------------------------------------------------------------------------
// Narrow tiles: 128 output features on the TMEM lanes, BN tokens in the columns, K split over a cluster.
//
// For few tokens the product reads the weight once and does little else, so the work is cut by weight bytes: one CTA
// takes 128 features and every S-th part of K, S CTAs of a cluster meet in one tile.  Warp 0 keeps the TMA ring full,
// warp 1 issues four MMAs per K block into one of four TMEM buffers, the promotion warps multiply the raw product of a
// K block by x_scale * w_scale -- a table of the CTA's own K blocks in shared memory, one number per token, the same
// for all lanes -- and add it up in fp32 registers.  The partial sums of a cluster are added through distributed
// shared memory in rank order: no atomics and no workspace.
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
    for (int i = threadIdx.x - 64; i < kbs * BN; i += kPromoThreads) {
      const int j = i / kbs, kb = i - j * kbs, t = min(tt * BN + j, p.m - 1);
      table[kb * C::kTabStride + j] = __ldg(p.x_scale + static_cast<size_t>(t) * p.kblocks + kb0 + kb) * __ldg(wsp + kb);
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

template <int BN>
int narrow_launch(const LinFp8Params& p, int split, cudaStream_t stream) {
  using C = Narrow<BN>;
  const int token_tiles = (p.m + BN - 1) / BN, feature_tiles = (p.n + 127) / 128;
  const int kb_max = (p.kblocks + split - 1) / split;
  const size_t fixed = 1024 + sizeof(float) * static_cast<size_t>(kb_max) * C::kTabStride +
                       8 * (2 * kNarrowMaxStages + 2 * kNarrowBufs + 1) + 16;
  const size_t budget = (C::kCtasPerSm == 2 ? 113 : 227) * 1024;
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

// K split over up to eight CTAs of a cluster: enough CTAs for the SMs, but whole K blocks (four at least) for each.
int narrow_split(const LinFp8Params& p, int bn, int ctas_per_sm) {
  const long long tiles = static_cast<long long>((p.m + bn - 1) / bn) * ((p.n + 127) / 128);
  long long s = static_cast<long long>(sm_count()) * ctas_per_sm / tiles;
  if (const char* e = getenv("LS")) s = atoi(e);
  static const int mk = [] { const char* e = getenv("MK"); return e ? atoi(e) : 2; }();
  if (s > p.kblocks / mk) s = p.kblocks / mk;
  return static_cast<int>(s < 1 ? 1 : (s > 8 ? 8 : s));
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
  p.vec = n % 4 == 0 && ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(acc)) & 15) == 0;
  const bool tma = k % 16 == 0 && ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0;
  if (tma) {
    if (m <= 16) return narrow_launch<16>(p, narrow_split(p, 16, 2), stream);
    if (m <= 32) return narrow_launch<32>(p, narrow_split(p, 32, 2), stream);
    if (m <= 64) return narrow_launch<64>(p, narrow_split(p, 64, 2), stream);
    return narrow_launch<128>(p, narrow_split(p, 128, 1), stream);
  }
  PTO_REQUIRE((m + kAnyTile - 1) / kAnyTile <= 65535, "linear_fp8: too many rows");
  launch_kernel(linear_fp8_any_kernel, dim3((n + kAnyTile - 1) / kAnyTile, (m + kAnyTile - 1) / kAnyTile), dim3(256), 0,
                stream, p);
  return check_cuda(cudaGetLastError(), "linear_fp8_any_kernel launch");
}

}  // namespace pto
