// Matrix product with bias, activation and residual in its epilogue, and its gradients.
//
//   out[M, N] = act(A . B^T + bias) + res        bf16 or fp16 operands, fp32 accumulation,
//                                                one rounding at the end
//
// Either operand may be stored K-major (rows of K elements) or MN-major (its transpose, rows of M
// or N elements), so the gradients of a Linear need no transposed copies:
//   forward   A = x [M, K]           B = W [N, K]                 both K-major
//   dx        A = dpre [M, N]        B = W read as [K, N]         B MN-major
//   dW        A = dpre read as [N, M]  B = x read as [K, M]       both MN-major
// with dpre = dout * act'(pre) from act_backward_kernel (one pass, which also sums the columns
// for the bias gradient).
//
// The product is a persistent warp-specialized tcgen05 kernel: warps 0 and 10 load the tiles of A
// and B by TMA into a shared-memory ring (128-byte swizzle, 64-wide K blocks), warp 1 issues the
// MMAs into one of two TMEM accumulators, warps 2-9 apply the epilogue of the other: 32 x 32
// pieces, the residual in and the result out by TMA through the warp's own shared memory. Two
// loading threads rather than one gain where a K block takes three loads (B MN-major in pieces:
// 1024 x 1536 x 8960 27.2 us, one thread 28.1), nothing elsewhere. A piece takes an epilogue warp
// about 800 clocks without an activation and 2000 with GELU, under the next tile's products; what
// made it slow (1800 and 3000) were arrivals that release at cluster scope, which wait for all of
// the thread's stores, bias loads piece by piece, and the tile's place computed for every piece.
//
// What bounds it: the tensor pipe for many rows (8192 x 13824 x 5120 fp16 with GELU and residual 836 - 846
// us, 1.37 - 1.39 PFLOP/s, the pipe 93% busy; in a loop of nothing else 971 by the card's power; 4096^3
// 93 us, the library's product 90), the fixed costs below (1024 x 1536 x 4096 with bias and tanh-GELU
// 18.2 us, 15.7 bare in a graph where the library's takes 11.2: set-up 0.9 us, first loads 0.8, last
// epilogue 1, then 270 clocks a K block at least), the weights' bytes for few (1 x 1536 x 8960 10.6 us).
// Tile forms (plan()):
//   pair    256 x bn tiles over CTA pairs (tcgen05 cta_group::2): many rows
//   single  128 x bn tiles
//   split   either of them with the K range divided over a cluster; the partial tiles are exchanged
//           through distributed shared memory and added in rank order: few tiles, where reading B
//           once or filling the SMs is the bound
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>
#include <type_traits>

#include "ptx.cuh"
#include "tmap.h"
#include "wdit_internal.h"

namespace wdit {
namespace {

constexpr int BM = 128;
constexpr int BK = 64;
constexpr int kThreads = 352;  // warp 0 loads A, 1 MMA, 2-9 epilogue, 10 loads B
constexpr int kEpiThreads = 256;
constexpr uint32_t kTileABytes = BM * BK * 2;
constexpr uint32_t kTmemCols = 512;  // two accumulators of up to 256 columns
constexpr int kMaxStages = 8;
constexpr int kBarriers = 2 * kMaxStages + 4 + 24;  // full, empty; TMEM full, empty; residual pieces
constexpr uint32_t kPieceBytes = 32 * 32 * 2;
constexpr uint32_t kWarpBytes = 4 * kPieceBytes;   // three rotating pieces and one of pre-activations
constexpr uint32_t kEpiBytes = 8 * (kWarpBytes + 32 * 4);  // ... and a line of 32 bias values
constexpr uint32_t kBarBytes = 512;
constexpr uint32_t kSmemLimit = 232448;
constexpr uint32_t kRingBudget = kSmemLimit - 1024 - kBarBytes - kEpiBytes;
constexpr int kMaxExtent = 1 << 30;  // M, N, K: coordinates past a matrix's end stay inside 32 bits
constexpr int kRasterRows = 8;
constexpr long long kRasterBytes = 64ll << 20;

enum Act { kNone = 0, kGeluTanh = 1, kRelu = 2, kSilu = 3, kGelu = 4 };

struct LinArgs {
  int M, N, K;
  int m_blocks, n_blocks, k_blocks, tiles, raster_rows;
  int bn, stages, splits;
  int a_one, b_one;  // MN-major operand whose 64-wide pieces come in one box (M or N and the tile % 64 == 0)
  int is_bf16, act, bias_dtype;
  const void* bias;
  const void* res;
  long long ldr;
  void* out;
  long long ldo;
  void* pre;
  long long ldp;
  WaitCtx ctx;
};

// Staged bytes of `rows` rows of a K block; MN-major ones come in whole pieces of 64 (of the last only
// the first columns may be used: 96 rows of B in a 256 x 192 pair tile).
__host__ __device__ __forceinline__ uint32_t operand_bytes(int rows, bool mn) {
  return static_cast<uint32_t>(mn ? (rows + 63) / 64 * 64 : rows) * (BK * 2);
}

// MN-major tile written by TMA with the 128-byte swizzle: pieces of 64 elements (128 B) along M
// or N, 64 K rows each. Leading offset: between pieces (64 rows x 128 B); stride offset: between
// groups of 8 K rows.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(8192u >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

// kind::f16 with fp32 accumulation; bits 7-9 / 10-12 operand format (0 fp16, 1 bf16), bits 15 / 16
// operand A / B is MN-major.
__device__ __forceinline__ uint32_t make_idesc(int m, int n, int is_bf16, bool ta, bool tb) {
  return (1u << 4) | (static_cast<uint32_t>(is_bf16) << 7) | (static_cast<uint32_t>(is_bf16) << 10) |
         (ta ? 1u << 15 : 0u) | (tb ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint64_t splat2(float v) { return f2_pack(v, v); }

__device__ __forceinline__ uint64_t exp2_2(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return f2_pack(exp2_approx(a), exp2_approx(b));
}

__device__ __forceinline__ uint64_t rcp_2(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return f2_pack(rcp_approx(a), rcp_approx(b));
}

constexpr float kLog2e = 1.4426950408889634f;
// tanh-GELU as x / (1 + exp(-2 z)), z = sqrt(2/pi) (x + 0.044715 x^3): no cancellation for x < 0
constexpr float kGeluA = 2.f * 0.7978845608028654f;
constexpr float kGeluB = 2.f * 0.7978845608028654f * 0.044715f;

// Q(u) = 1 - Phi(u) for u >= 0 as exp(-u^2 / 2) R(t), t = 1 / (1 + 0.312 u): R is a polynomial of
// degree 6 fitted to Q exp(u^2 / 2) with relative error below 2^-17.3 for every u (a least-squares
// fit with weights driven to equal ripple; half a step of fp16 is 2^-11). e receives exp(-u^2 / 2).
// u is |x| cut at 30, where Q is 0 in fp32, so that infinities make no 0 * inf.
constexpr float kQc = 0.312f;
__device__ __forceinline__ uint64_t gauss_tail2(uint64_t u, uint64_t& e) {
  const uint64_t t = rcp_2(ffma2(u, splat2(kQc), splat2(1.f)));
  uint64_t r = ffma2(t, splat2(-0.07296360501607355f), splat2(0.17343308598567092f));
  r = ffma2(r, t, splat2(0.021109508863869385f));
  r = ffma2(r, t, splat2(0.1324384307670562f));
  r = ffma2(r, t, splat2(0.12126615653403806f));
  r = ffma2(r, t, splat2(0.12472093351055727f));
  r = ffma2(r, t, splat2(-7.4565507634441656e-06f));
  e = exp2_2(fmul2(fmul2(u, u), splat2(-0.5f * kLog2e)));
  return fmul2(e, r);
}

// Two columns at a time (packed fp32).
__device__ __forceinline__ uint64_t act2(uint64_t x, int act) {
  float a, b;
  switch (act) {
    case kRelu:
      f2_unpack(x, a, b);
      return f2_pack(a < 0.f ? 0.f : a, b < 0.f ? 0.f : b);  // NaN stays
    case kSilu:
      return fmul2(x, rcp_2(fadd2(exp2_2(fmul2(x, splat2(-kLog2e))), splat2(1.f))));
    case kGeluTanh: {
      const uint64_t z = fmul2(x, ffma2(fmul2(x, x), splat2(-kLog2e * kGeluB), splat2(-kLog2e * kGeluA)));
      return fmul2(x, rcp_2(fadd2(exp2_2(z), splat2(1.f))));
    }
    case kGelu: {  // max(x, 0) - |x| Q(|x|)
      f2_unpack(x, a, b);
      const uint64_t u = f2_pack(fminf(fabsf(a), 30.f), fminf(fabsf(b), 30.f));
      uint64_t e;
      const uint64_t q = gauss_tail2(u, e);
      return ffma2(fmul2(u, splat2(-1.f)), q, f2_pack(a < 0.f ? 0.f : a, b < 0.f ? 0.f : b));
    }
    default:
      return x;
  }
}

template <int N>
__device__ __forceinline__ void apply_act(float (&v)[N], int act) {
  if (act == kNone) return;
  // one branch for the whole piece
  auto all = [&](auto kind) {
#pragma unroll
    for (int i = 0; i < N; i += 2) f2_unpack(act2(f2_pack(v[i], v[i + 1]), decltype(kind)::value), v[i], v[i + 1]);
  };
  if (act == kRelu) {
    all(std::integral_constant<int, kRelu>{});
  } else if (act == kSilu) {
    all(std::integral_constant<int, kSilu>{});
  } else if (act == kGeluTanh) {
    all(std::integral_constant<int, kGeluTanh>{});
  } else {
    all(std::integral_constant<int, kGelu>{});
  }
}

// act'(x) of two columns, cut where it is 0 or 1 in fp32 so that x, x^2 and infinities make no inf * 0
// (NaN passes): GELU's from 20 on (at -15 both are below 2^-126), SiLU's, (1 + x) e^x on the left, from 100 on.
template <int ACT>
__device__ __forceinline__ uint64_t act_grad2(float a, float b) {
  if constexpr (ACT == kRelu) return f2_pack(a > 0.f ? 1.f : 0.f, b > 0.f ? 1.f : 0.f);
  constexpr float kCut = ACT == kSilu ? 100.f : 20.f;
  if (fabsf(a) > kCut) a = copysignf(kCut, a);
  if (fabsf(b) > kCut) b = copysignf(kCut, b);
  const uint64_t x = f2_pack(a, b);
  if constexpr (ACT == kSilu) {  // s + x s (1 - s)
    const uint64_t s = rcp_2(fadd2(exp2_2(fmul2(x, splat2(-kLog2e))), splat2(1.f)));
    return ffma2(fmul2(x, s), ffma2(s, splat2(-1.f), splat2(1.f)), s);
  } else if constexpr (ACT == kGeluTanh) {  // s + x s (1 - s) (2 z)'
    const uint64_t xx = fmul2(x, x);
    const uint64_t s =
        rcp_2(fadd2(exp2_2(fmul2(x, ffma2(xx, splat2(-kLog2e * kGeluB), splat2(-kLog2e * kGeluA)))), splat2(1.f)));
    const uint64_t dz = ffma2(xx, splat2(3.f * kGeluB), splat2(kGeluA));
    return ffma2(fmul2(fmul2(x, dz), s), ffma2(s, splat2(-1.f), splat2(1.f)), s);
  } else {  // Phi(x) + x phi(x)
    uint64_t e;
    float q0, q1;
    f2_unpack(gauss_tail2(f2_pack(fabsf(a), fabsf(b)), e), q0, q1);
    return ffma2(fmul2(x, splat2(0.3989422804014327f)), e, f2_pack(a < 0.f ? q0 : 1.f - q0, b < 0.f ? q1 : 1.f - q1));
  }
}

__device__ __forceinline__ float2 unpack2(uint32_t w, int is_bf16) {
  if (is_bf16) return unpack_bf16x2(w);
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}

__device__ __forceinline__ uint32_t pack2(float a, float b, int is_bf16) {
  if (is_bf16) return pack_bf16x2(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float load_scalar(const void* p, long long i, int dtype) {
  if (dtype == 0) return static_cast<const float*>(p)[i];
  if (dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_scalar(void* p, long long i, int dtype, float v) {
  if (dtype == 0) {
    static_cast<float*>(p)[i] = v;
  } else if (dtype == 1) {
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  } else {
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  }
}

// Epilogue of eight columns of one row (n < N, N % 8 == 0): residual, stores.
__device__ __forceinline__ void finish8(const LinArgs& p, float (&v)[8], long long row, int n) {
  if (p.pre != nullptr) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1], p.is_bf16);
    st_global_v4(static_cast<uint16_t*>(p.pre) + row * p.ldp + n, w[0], w[1], w[2], w[3]);
  }
  apply_act<8>(v, p.act);
  if (p.res != nullptr) {
    // plain (coherent) load: res may be out, and this thread writes the same eight columns below
    const uint4 r = ld_global_cg_v4(static_cast<const uint16_t*>(p.res) + row * p.ldr + n);
    const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(rw[i], p.is_bf16);
      v[2 * i] += f.x;
      v[2 * i + 1] += f.y;
    }
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack2(v[2 * i], v[2 * i + 1], p.is_bf16);
  st_global_v4(static_cast<uint16_t*>(p.out) + row * p.ldo + n, w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Completes on the pair leader's barrier (a shared::cluster address).
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Operand maps are 3-D in either storage: K-major {K, rows, 1}, box {64, rows of the tile, 1};
// MN-major {64, K, pieces of 64} with all of a tile's pieces in one box, or, when M or N or the
// tile is no multiple of 64, {M or N, K, 1} with one box per piece.
template <bool PAIR, bool SPLIT, bool TA, bool TB>
__global__ void __launch_bounds__(kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmRes,
                  const __grid_constant__ CUtensorMap tmPre, const __grid_constant__ LinArgs p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int b_rows = PAIR ? p.bn / 2 : p.bn;  // B rows this CTA stages
  const uint32_t b_bytes = operand_bytes(b_rows, TB);
  const uint32_t SB = kTileABytes + b_bytes;
  const int stages = p.stages;
  uint8_t* epi = smem + stages * SB;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(epi + kEpiBytes);
  uint64_t* empty_bar = full_bar + kMaxStages;
  uint64_t* tfull_bar = empty_bar + kMaxStages;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* res_bar = tempty_bar + 2;  // 3 per epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_bar + 24);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = PAIR || SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
  const int cta_rank = PAIR ? rank & 1 : 0;
  const int split = SPLIT ? (PAIR ? rank >> 1 : rank) : 0;
  const int leader = rank & ~1;  // pair: the even CTA arms barriers and issues the MMAs
  const int group = (PAIR ? 2 : 1) * (SPLIT ? p.splits : 1);  // CTAs that share a tile
  const int t_first = static_cast<int>(blockIdx.x) / group;
  const int t_step = static_cast<int>(gridDim.x) / group;
  const int my_count = t_first < p.tiles ? (p.tiles - 1 - t_first) / t_step + 1 : 0;
  // K blocks of this CTA (split: a contiguous share, the first ranks one more)
  int kb0 = 0, kb1 = p.k_blocks;
  if constexpr (SPLIT) {
    const int base = p.k_blocks / p.splits, rem = p.k_blocks % p.splits;
    kb0 = split * base + min(split, rem);
    kb1 = kb0 + base + (split < rem ? 1 : 0);
  }
  auto coords = [&](int i, int& m_blk, int& n_blk) {
    const int t = t_first + i * t_step;
    const int mg = PAIR ? (p.m_blocks + 1) / 2 : p.m_blocks;
    const int per_group = p.raster_rows * p.n_blocks;
    const int grp = t / per_group;
    const int first = grp * p.raster_rows;
    const int gm = min(p.raster_rows, mg - first);
    const int r = t - grp * per_group;
    n_blk = r / gm;
    const int mq = first + (r - n_blk * gm);
    m_blk = PAIR ? 2 * mq + cta_rank : mq;
  };

  // One barrier a thread: set up one after the other they take as long as the first loads.
  if (threadIdx.x < kBarriers) {
    const int i = threadIdx.x;
    uint32_t arrivals = 1;
    if (i < kMaxStages) arrivals = 2;  // full_bar: armed by the loaders of A and B
    if (i >= 2 * kMaxStages + 2 && i < 2 * kMaxStages + 4) arrivals = (PAIR ? 2 : 1) * (kEpiThreads / 32);  // tempty_bar
    mbar_init(&full_bar[i], arrivals);
    fence_mbar_init();
  } else if (threadIdx.x == 10 * 32) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_slot, kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (PAIR || SPLIT) {
    cluster_sync_all();
  } else {
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0 || warp == 10) {
    // Loaders: warp 0 the A tiles, warp 10 the B tiles of the same stages.
    if (elect_one()) {
      const bool is_a = warp == 0;
      const CUtensorMap* map = is_a ? &tmA : &tmB;
      const bool mn = is_a ? TA : TB;
      const uint32_t bytes = is_a ? kTileABytes : b_bytes;
      const int pieces = ((is_a ? BM : b_rows) + 63) / 64;
      const bool one = (is_a ? p.a_one : p.b_one) != 0;
      const uint32_t full0 = PAIR ? mapa_shared(smem_u32(full_bar), leader) : smem_u32(full_bar);
      uint8_t* const dst0 = smem + (is_a ? 0 : kTileABytes);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < my_count && ok; ++i) {
        int m_blk, n_blk;
        coords(i, m_blk, n_blk);
        const int row = is_a ? m_blk * BM : n_blk * p.bn + cta_rank * b_rows;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_parity<PAIR>(&empty_bar[stage], phase ^ 1u, kSiteProducerEmpty, p.ctx)) {
            ok = false;
            break;
          }
          uint8_t* dst = dst0 + stage * SB;
          const uint32_t bar = full0 + stage * 8;
          // Pair: both CTAs' loads complete on the leader's barrier; only the leader arms it.
          if (!PAIR || cta_rank == 0) mbar_arrive_expect_tx(&full_bar[stage], PAIR ? 2 * bytes : bytes);
          auto load = [&](uint8_t* to, int x, int y, int z) {
            if constexpr (PAIR) {
              tma_load_3d_pair(to, map, bar, x, y, z);
            } else {
              tma_load_3d(to, map, bar, x, y, z);
            }
          };
          if (!mn) {
            load(dst, kb * BK, row, 0);
          } else if (one) {
            load(dst, 0, kb * BK, row / 64);
          } else {
            for (int c = 0; c < pieces; ++c) load(dst + c * 8192, row + c * 64, kb * BK, 0);
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // Drain: do not leave the CTA while TMA writes into its shared memory are pending.
      for (int i = 0; i < stages; ++i) {
        if (!wait_parity<PAIR>(&empty_bar[stage], phase ^ 1u, kSiteDrain, p.ctx)) break;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (cta_rank == 0 && elect_one()) {
      const uint32_t idesc = make_idesc(PAIR ? 2 * BM : BM, p.bn, p.is_bf16, TA, TB);
      const uint32_t ring = smem_u32(smem);
      const uint32_t empty0 = smem_u32(empty_bar), peer0 = PAIR ? mapa_shared(empty0, rank | 1) : 0u;
      int stage = 0;
      uint32_t phase = 0;
      for (int it = 0; it < my_count; ++it) {
        const int buf = it & 1;
        const uint32_t tphase = (it >> 1) & 1;
        if (!wait_parity<PAIR>(&tempty_bar[buf], tphase ^ 1u, kSiteMmaTmemEmpty, p.ctx)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * 256;
        bool ok = true;
        uint32_t acc = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_parity<PAIR>(&full_bar[stage], phase, kSiteMmaFull, p.ctx)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = ring + stage * SB;
          const uint64_t a_desc = TA ? smem_desc_mn(a_addr) : smem_desc_sw128(a_addr);
          const uint64_t b_desc = TB ? smem_desc_mn(a_addr + kTileABytes) : smem_desc_sw128(a_addr + kTileABytes);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            // 16 K elements on: 32 bytes inside a K-major row, 16 rows of 128 bytes MN-major
            const uint64_t ad = a_desc + (TA ? 128 : 2) * k;
            const uint64_t bd = b_desc + (TB ? 128 : 2) * k;
            if constexpr (PAIR) {
              mma_bf16_pair(d_tmem, ad, bd, idesc, acc);
            } else {
              mma_bf16(d_tmem, ad, bd, idesc, acc);
            }
            acc = 1;
          }
          if constexpr (PAIR) {
            mma_commit_pair(empty0 + stage * 8);
            mma_commit_pair(peer0 + stage * 8);
          } else {
            mma_commit(&empty_bar[stage]);
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if constexpr (PAIR) {
          mma_commit_pair(smem_u32(&tfull_bar[buf]));
          mma_commit_pair(mapa_shared(smem_u32(&tfull_bar[buf]), rank | 1));
        } else {
          mma_commit(&tfull_bar[buf]);
        }
      }
    }
    __syncwarp();
  } else {
    // Epilogue: warp w reads TMEM lanes [32 (w % 4), + 32) (its thread owns one accumulator row);
    // warps 2-5 take the even 32-column pieces of the tile, warps 6-9 the odd ones.
    const int ew = warp - 2;
    const int wq = warp & 3;
    const int half = ew >> 2;
    const int r = wq * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const int pieces = p.bn / 32;
    uint8_t* const bufs = epi + ew * kWarpBytes;
    float* const bias_line = reinterpret_cast<float*>(epi + 8 * kWarpBytes) + ew * 32;
    uint64_t* const rbar = res_bar + ew * 3;
    uint32_t rphase = 0;  // phase of each residual buffer's barrier
    int cur = 0;          // rotating piece buffer
    const bool has_res = !SPLIT && p.res != nullptr;
    // first row of the warp and first column of a tile
    auto place = [&](int it, int& row, int& col) {
      int m_blk, n_blk;
      coords(it, m_blk, n_blk);
      row = m_blk * BM + wq * 32;
      col = n_blk * p.bn;
    };
    int in_flight = -1;  // lane 0: buffer of the last residual piece asked for
    auto fetch_res = [&](int row0, int n0, int buf) {  // lane 0
      if (row0 >= p.M || n0 >= p.N) return;
      mbar_arrive_expect_tx(&rbar[buf], kPieceBytes);
      tma_load_2d(bufs + buf * kPieceBytes, &tmRes, &rbar[buf], n0, row0);
      in_flight = buf;
    };
    int row0 = 0, col = 0, next_row = 0, next_col = 0;
    if (my_count > 0) place(0, next_row, next_col);
    if (has_res && lane == 0 && my_count > 0) fetch_res(next_row, next_col + half * 32, 0);
    bool failed = false;
    for (int it = 0; it < my_count && !failed; ++it) {
      const int buf = it & 1;
      const uint32_t tphase = (it >> 1) & 1;
      row0 = next_row, col = next_col;
      if (it + 1 < my_count) place(it + 1, next_row, next_col);
      // this lane's bias of the warp's pieces, loaded while the tile is computed
      float bias[4] = {0.f, 0.f, 0.f, 0.f};
      if (!SPLIT && p.bias != nullptr) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int n = col + (half + 2 * q) * 32 + lane;
          if (half + 2 * q < pieces && n < p.N) bias[q] = load_scalar(p.bias, n, p.bias_dtype);
        }
      }
      failed = !__all_sync(0xffffffffu, wait_parity<PAIR>(&tfull_bar[buf], tphase, kSiteEpiTmemFull, p.ctx));
      if (failed) break;
      tc_fence_after();
      const uint32_t tbase = tmem_base + lane_off + buf * 256;
#pragma unroll 1
      for (int c = half; c < pieces; c += 2) {
        const int n0 = col + c * 32;
        const bool inside = row0 < p.M && n0 < p.N;
        float v[32];
        tmem_ld32(tbase + c * 32, v);
        if (c + 2 >= pieces) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR) {
              mbar_arrive_tmem_cluster(mapa_shared(smem_u32(&tempty_bar[buf]), leader));
            } else {
              mbar_arrive(&tempty_bar[buf]);
            }
          }
        }
        if constexpr (SPLIT) {
          // this rank's partial tile, rows of bn + 4 floats, over the drained ring
          if (row0 + lane < p.M) {
            float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(smem) + r * (p.bn + 4) + c * 32);
#pragma unroll
            for (int q = 0; q < 8; ++q) dst[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          }
        } else {
          const int next = cur == 2 ? 0 : cur + 1;
          if (lane == 0) {
            bulk_wait_read<1>();  // every store but the last has left its buffer
            if (has_res) {
              if (c + 2 < pieces) {
                fetch_res(row0, n0 + 64, next);
              } else if (it + 1 < my_count) {
                fetch_res(next_row, next_col + half * 32, next);
              }
            }
          }
          if (inside) {
            if (p.bias != nullptr) {
              const int q = c >> 1;
              __syncwarp();
              bias_line[lane] = q == 0 ? bias[0] : (q == 1 ? bias[1] : (q == 2 ? bias[2] : bias[3]));
            }
            __syncwarp();
            if (p.bias != nullptr) {
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                const float4 b4 = reinterpret_cast<const float4*>(bias_line)[q];
                v[4 * q] += b4.x;
                v[4 * q + 1] += b4.y;
                v[4 * q + 2] += b4.z;
                v[4 * q + 3] += b4.w;
              }
            }
            auto stage_out = [&](uint8_t* to, const CUtensorMap* map) {
              const uint32_t row = smem_u32(to) + lane * 64;
#pragma unroll
              for (int q = 0; q < 4; ++q)
                st_shared_v4(row + ((q ^ ((lane >> 1) & 3)) << 4), pack2(v[8 * q], v[8 * q + 1], p.is_bf16),
                             pack2(v[8 * q + 2], v[8 * q + 3], p.is_bf16), pack2(v[8 * q + 4], v[8 * q + 5], p.is_bf16),
                             pack2(v[8 * q + 6], v[8 * q + 7], p.is_bf16));
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(map, to, n0, row0);
                bulk_commit();
              }
            };
            if (p.pre != nullptr) stage_out(bufs + 3 * kPieceBytes, &tmPre);
            apply_act<32>(v, p.act);
            uint8_t* mine = bufs + cur * kPieceBytes;
            if (has_res) {
              failed = !__all_sync(0xffffffffu, wait_parity(&rbar[cur], (rphase >> cur) & 1u, kSiteEpiCLoad, p.ctx));
              if (failed) break;
              rphase ^= 1u << cur;
              const uint32_t row = smem_u32(mine) + lane * 64;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const uint4 w = ld_shared_u4(row + ((q ^ ((lane >> 1) & 3)) << 4));
                const uint32_t rw[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 f = unpack2(rw[e], p.is_bf16);
                  v[8 * q + 2 * e] += f.x;
                  v[8 * q + 2 * e + 1] += f.y;
                }
              }
            }
            stage_out(mine, &tmOut);
          }
          cur = next;
        }
      }
    }
    if (lane == 0) {
      bulk_wait_read<0>();  // the stores have read shared memory
      // After a wait that ran out the last residual piece may still be on its way.
      if (failed && in_flight >= 0) wait_parity(&rbar[in_flight], (rphase >> in_flight) & 1u, kSiteDrain, p.ctx);
    }
    __syncwarp();
  }
  if constexpr (SPLIT) {
    // One tile per cluster. The tile's valid rows, in pieces of eight columns, are shared out over
    // the splits in order (whole rows, so that the remote reads are contiguous); each adds all the
    // splits' partial values of its pieces (pair: of its own 128 rows), split 0 first.
    cluster_sync_all();
    if (warp >= 2 && warp < 10 && my_count > 0) {
      int m_blk, n_blk;
      coords(0, m_blk, n_blk);
      const int per_row = p.bn / 8;
      const int total = min(BM, p.M - m_blk * BM) * per_row;
      const int share = (total + p.splits - 1) / p.splits;
      const int end = min(total, (split + 1) * share);
      const uint32_t mine = smem_u32(smem);
      for (int x = split * share + threadIdx.x - 64; x < end; x += kEpiThreads) {
        const int rr = x / per_row;
        const int c = (x - rr * per_row) * 8;
        const int n = n_blk * p.bn + c;
        if (n >= p.N) continue;
        float4 f[8][2];  // all ranks' loads are in flight together
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          f[s][0] = f[s][1] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (s < p.splits) {
            const uint32_t a = mapa_shared(mine + (rr * (p.bn + 4) + c) * 4, PAIR ? 2 * s + cta_rank : s);
            f[s][0] = ld_cluster_f4(a);
            f[s][1] = ld_cluster_f4(a + 16);
          }
        }
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p.bias != nullptr ? load_scalar(p.bias, n + i, p.bias_dtype) : 0.f;
#pragma unroll
        for (int s = 0; s < 8; ++s) {
          v[0] += f[s][0].x; v[1] += f[s][0].y; v[2] += f[s][0].z; v[3] += f[s][0].w;
          v[4] += f[s][1].x; v[5] += f[s][1].y; v[6] += f[s][1].z; v[7] += f[s][1].w;
        }
        finish8(p, v, m_blk * BM + rr, n);
      }
    }
  }
  tc_fence_before();
  if constexpr (PAIR || SPLIT) {
    cluster_sync_all();  // peers may still read this CTA's shared memory / signal its barriers
  } else {
    __syncthreads();
  }
  tc_fence_after();
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_dealloc_pair(tmem_base, kTmemCols);
    } else {
      tmem_dealloc(tmem_base, kTmemCols);
    }
  }
}

// ---------------------------------------------------------------------------
// dpre = dout * act'(pre), and the column sums of dpre by row chunks (bias gradient). One pass bound
// by HBM: 4095 x 8960 bf16 SiLU 43.5 us, 5.1 TB/s
// ---------------------------------------------------------------------------
constexpr int kBackRows = 64;  // rows of one block
constexpr int kBackCols = 256;

template <bool BF16, int ACT>
__global__ void __launch_bounds__(256)
    act_backward_kernel(const uint16_t* __restrict__ dout, long long ldd, const uint16_t* __restrict__ pre,
                        long long ldp, uint16_t* __restrict__ dpre, long long ldq,
                        float* __restrict__ part, void* __restrict__ dbias, int dbias_dtype, int M, int N) {
  __shared__ float sums[8][kBackCols];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col_blocks = (N + kBackCols - 1) / kBackCols;
  const int chunk = blockIdx.x / col_blocks;  // (one grid dimension: rows may pass the others' 65535)
  const int n0 = (blockIdx.x - chunk * col_blocks) * kBackCols;
  const int n = n0 + lane * 8;
  const int m0 = chunk * kBackRows;
  const int m1 = min(m0 + kBackRows, M);
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  if (n < N) {
#pragma unroll 2  // (8 rows at a time take registers from other warps: 52 us, 4 47, 2 43.5)
    for (int m = m0 + warp; m < m1; m += 8) {
      const uint4 g = __ldg(reinterpret_cast<const uint4*>(dout + m * ldd + n));
      const uint32_t gw[4] = {g.x, g.y, g.z, g.w};
      float d[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2(gw[i], BF16);
        d[2 * i] = f.x;
        d[2 * i + 1] = f.y;
      }
      if constexpr (ACT != kNone) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(pre + m * ldp + n));
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack2(xw[i], BF16);
          f2_unpack(fmul2(f2_pack(d[2 * i], d[2 * i + 1]), act_grad2<ACT>(f.x, f.y)), d[2 * i], d[2 * i + 1]);
        }
        st_global_v4(dpre + m * ldq + n, pack2(d[0], d[1], BF16), pack2(d[2], d[3], BF16), pack2(d[4], d[5], BF16),
                     pack2(d[6], d[7], BF16));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += d[i];
    }
  }
  if (part == nullptr && dbias == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[warp][lane * 8 + i] = acc[i];
  __syncthreads();
  const int c = n0 + threadIdx.x;
  if (c < N) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][threadIdx.x];
    if (part != nullptr) {
      part[static_cast<size_t>(chunk) * N + c] = s;
    } else {  // one chunk: this is all of it
      store_scalar(dbias, c, dbias_dtype, s);
    }
  }
}

__global__ void __launch_bounds__(256)
    col_sum_kernel(const float* __restrict__ part, int chunks, int N, void* __restrict__ out, int dtype) {
  // 32 columns a block, 8 threads a column
  __shared__ float sums[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (n < N)
    for (int c = w; c < chunks; c += 8) s += part[static_cast<size_t>(c) * N + n];
  sums[w][lane] = s;
  __syncthreads();
  if (w != 0 || n >= N) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += sums[i][lane];
  store_scalar(out, n, dtype, s);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct Plan {
  int pair, bn, splits;
};

// The tile form by estimated clocks. Measured at 1.9 GHz, one K block (64) of a tile takes a CTA 270
// clocks at least (its issuing threads), 2.1 per column otherwise (the tensor pipe: 128 x 192 398,
// 128 x 256 548; pairs 256 x 192 394, 256 x 256 530), and all CTAs together load about 11 KB a clock
// from L2 (128 x 128 tiles on every SM: 418 instead of 270). The last tile's epilogue adds 17 clocks
// per column (12 bare, 30 with GELU), an exchange between splits 4200 and 0.45 per element that
// crosses. What that picks (wdit_linear_act_residual_form) and what else was measured (bf16, us a launch,
// twenty in a graph):
//   1024 x 1536 x 4096  pairs 256 x 128 15.7 (halves of K over 128 x 192 17.3, 128 x 128 18.1, pairs 256 x 192 20.0)
//   256 x 1536 x 8960   quarters of K over pairs 256 x 128 15.8 (over 128 x 128 16.3, halves 19.1)
//   2048 x 1536 x 8960  pairs 256 x 192 43.8 (128 x 192 46.7, pairs 256 x 256 48.8)
//   1024 x 8960 x 1536  pairs 256 x 256 24.8 (pairs 256 x 128 25.0)
// and where it misses by more than a twentieth:
//   1 x 1536 x 8960     eighths of K over 128 x 128 13.4 (over 128 x 192 11.0, over 128 x 256 11.9)
//   1 x 4096 x 10240    quarters of K over 128 x 128 22.6 (over 128 x 256 18.6)
// With B MN-major a 256 x 192 pair tile stages 128 rows of B a CTA for the 96 it uses; 5% on its blocks:
//   4095 x 1536 x 8960  pairs 256 x 192 87 - 97 by the card's power (128 x 192 99, pairs 256 x 256 104)
//   4096 x 5120 x 13824 pairs 256 x 256 393 - 451 by the card's power (pairs 256 x 192 451)
Plan plan(int M, int N, int K, bool mn_b, int sms) {
  const int kb = (K + BK - 1) / BK;
  Plan best = {0, 128, 1};
  double best_cost = 1e30;
  auto consider = [&](int pair, int bn, int s) {
    const long long mb = (M + BM - 1) / BM, nb = (N + bn - 1) / bn;
    const long long tiles = (pair ? (mb + 1) / 2 : mb) * nb;
    const int group = (pair ? 2 : 1) * s;
    // co-resident clusters of this kernel on 148 SMs (cudaOccupancyMaxActiveClusters): 74, 33, 15
    const long long slots =
        group == 1 ? sms : (group == 2 ? sms / 2 : (group == 4 ? sms * 33 / 148 : sms * 15 / 148));
    if (s > 1 && tiles > slots) return;
    const long long waves = (tiles + slots - 1) / slots;
    const double active = static_cast<double>(tiles < slots ? tiles : slots) * group;
    double block = 2.1 * bn;
    const double l2 = active * (kTileABytes + operand_bytes(pair ? bn / 2 : bn, mn_b)) / 11000;
    if (l2 > block) block = l2;
    if (block < 270) block = 270;
    if (pair && mn_b && bn == 192) block *= 1.05;
    const int rows = M < BM ? M : BM;
    const double end = (s > 1 ? 4200 + 0.45 * rows * bn * (s - 1) / s : 17.0 * bn) + (pair ? 500 : 0);
    const double cost = waves * ((kb + s - 1) / s) * block + end;
    if (cost < best_cost) {
      best_cost = cost;
      best = {pair, bn, s};
    }
  };
  for (int bn = 256; bn >= 64; bn -= 64)
    for (int s = 1; s <= 8 && s <= kb; s *= 2) {
      consider(0, bn, s);
      if (M > BM && bn != 64 && s <= 4) consider(1, bn, s);
    }
  return best;
}

int launch_error(cudaError_t e) {
  if (e == cudaSuccess) return WDIT_OK;
  cudaGetLastError();  // reported here, not by the next launch too
  return WDIT_ERR_CUDA_BASE + static_cast<int>(e);
}

struct Maps {
  CUtensorMap a, b, out, res, pre;
};

template <bool PAIR, bool SPLIT, bool TA, bool TB>
int launch(const Maps& m, LinArgs p, cudaStream_t stream) {
  static bool attr_set[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return launch_error(e);
  const int b_rows = PAIR ? p.bn / 2 : p.bn;
  const uint32_t sb = kTileABytes + operand_bytes(b_rows, TB);
  p.stages = static_cast<int>(kRingBudget / sb);
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  if (!attr_set[dev & 63]) {
    e = cudaFuncSetAttribute(linear_kernel<PAIR, SPLIT, TA, TB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kSmemLimit);
    if (e != cudaSuccess) return launch_error(e);
    attr_set[dev & 63] = true;
  }
  const int group = (PAIR ? 2 : 1) * (SPLIT ? p.splits : 1);
  p.tiles = (PAIR ? (p.m_blocks + 1) / 2 : p.m_blocks) * p.n_blocks;
  long long grid = static_cast<long long>(p.tiles) * group;
  if (!SPLIT) {
    const long long slots = sm_count() / group * group;
    if (grid > slots) grid = slots;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 1024 + p.stages * sb + kEpiBytes + kBarBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = group;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = group > 1 ? 1 : 0;
  return launch_error(
      cudaLaunchKernelEx(&cfg, linear_kernel<PAIR, SPLIT, TA, TB>, m.a, m.b, m.out, m.res, m.pre, p));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

CUtensorMapDataType map_type(int is_bf16) {
  return is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// Operand map (see linear_kernel): `rows` along M or N of which a CTA's tile takes `tile`.
int map_operand(CUtensorMap* m, int is_bf16, const void* ptr, int rows, int K, long long ld, int mn, int tile,
                int* one) {
  typedef unsigned long long u64;
  *one = mn && rows % 64 == 0 && tile % 64 == 0 ? 1 : 0;
  const u64 row_bytes = static_cast<u64>(ld) * 2;
  if (!mn) {
    const u64 dims[3] = {static_cast<u64>(K), static_cast<u64>(rows), 1};
    const u64 st[2] = {row_bytes, row_bytes};
    const unsigned box[3] = {64, static_cast<unsigned>(tile), 1};
    return encode_tiled(m, map_type(is_bf16), 3, ptr, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const u64 dims[3] = {static_cast<u64>(*one ? 64 : rows), static_cast<u64>(K), static_cast<u64>(*one ? rows / 64 : 1)};
  const u64 st[2] = {row_bytes, 128};
  const unsigned box[3] = {64, BK, static_cast<unsigned>(*one ? tile / 64 : 1)};
  return encode_tiled(m, map_type(is_bf16), 3, ptr, dims, st, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// 32 x 32 pieces of a row-major matrix, for the epilogue
int map_pieces(CUtensorMap* m, int is_bf16, const void* ptr, int cols, int rows, long long ld) {
  const unsigned long long dims[2] = {static_cast<unsigned long long>(cols), static_cast<unsigned long long>(rows)};
  const unsigned long long st[1] = {static_cast<unsigned long long>(ld) * 2};
  const unsigned box[2] = {32, 32};
  return encode_tiled(m, map_type(is_bf16), 2, ptr, dims, st, box, CU_TENSOR_MAP_SWIZZLE_64B);
}

int run_linear(const void* A, long long lda, int a_mn, const void* B, long long ldb, int b_mn, LinArgs p,
               cudaStream_t stream) {
  const Plan pl = plan(p.M, p.N, p.K, b_mn != 0, sm_count());
  p.bn = pl.bn;
  p.splits = pl.splits;
  p.m_blocks = (p.M + BM - 1) / BM;
  p.n_blocks = (p.N + p.bn - 1) / p.bn;
  p.k_blocks = (p.K + BK - 1) / BK;
  // Tiles go along the columns of a row block (or pair), or, where B does not stay in L2, down groups of
  // eight row blocks (us: B of 142 MB, 8192 x 13824 x 5120, 768 by groups, 985 without; 34 MB, 4096^3, 93 and 91).
  p.raster_rows = static_cast<long long>(p.N) * p.K * 2 > kRasterBytes ? kRasterRows : 1;
  int rc = error_record_ptr(&p.ctx.rec);
  if (rc) return rc;
  p.ctx.limit_ns = wait_limit_ns();
  Maps m;
  memset(&m, 0, sizeof(m));
  if ((rc = map_operand(&m.a, p.is_bf16, A, p.M, p.K, lda, a_mn, BM, &p.a_one)) ||
      (rc = map_operand(&m.b, p.is_bf16, B, p.N, p.K, ldb, b_mn, pl.pair ? p.bn / 2 : p.bn, &p.b_one)))
    return rc;
  if (pl.splits == 1) {
    if ((rc = map_pieces(&m.out, p.is_bf16, p.out, p.N, p.M, p.ldo))) return rc;
    if (p.res != nullptr && (rc = map_pieces(&m.res, p.is_bf16, p.res, p.N, p.M, p.ldr))) return rc;
    if (p.pre != nullptr && (rc = map_pieces(&m.pre, p.is_bf16, p.pre, p.N, p.M, p.ldp))) return rc;
  }
  auto go = [&](auto pair, auto split) {
    constexpr bool P = decltype(pair)::value, S = decltype(split)::value;
    if (a_mn) return launch<P, S, true, true>(m, p, stream);
    if (b_mn) return launch<P, S, false, true>(m, p, stream);
    return launch<P, S, false, false>(m, p, stream);
  };
  if (pl.pair) return pl.splits > 1 ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
  return pl.splits > 1 ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
}

int check_operand(const void* p, long long ld, long long cols) {
  if (p == nullptr) return WDIT_ERR_ARG;
  if (ld < cols) return WDIT_ERR_SHAPE;
  if (!aligned16(p) || ld % 8 != 0) return WDIT_ERR_ALIGN;
  return WDIT_OK;
}

}  // namespace

int sm_count() {
  static int n[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (n[dev] == 0) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) return 148;
    n[dev] = v;
  }
  return n[dev];
}

}  // namespace wdit

using namespace wdit;

extern "C" {


int wdit_linear_act_residual(const void* A, long long lda, int a_mn, const void* B, long long ldb, int b_mn, int M,
                             int N, int K, int dtype, const void* bias, int bias_dtype, int act, const void* res,
                             long long ldr, void* out, long long ldo, void* pre_out, long long ldp, void* stream) {
  if (M < 0 || N < 0 || K < 0 || N % 8 != 0 || M > kMaxExtent || N > kMaxExtent || K > kMaxExtent) return WDIT_ERR_SHAPE;
  if (M == 0 || N == 0) return WDIT_OK;  // nothing to write
  if (K == 0) return WDIT_ERR_SHAPE;
  if (dtype != 1 && dtype != 2) return WDIT_ERR_ARG;
  if (act < kNone || act > kGelu || (bias != nullptr && (bias_dtype < 0 || bias_dtype > 2))) return WDIT_ERR_ARG;
  if (a_mn && !b_mn) return WDIT_ERR_ARG;  // no gradient needs it: not built
  int rc;
  if ((rc = check_operand(A, lda, a_mn ? M : K)) || (rc = check_operand(B, ldb, b_mn ? N : K)) ||
      (rc = check_operand(out, ldo, N)))
    return rc;
  if (res != nullptr && (rc = check_operand(res, ldr, N))) return rc;
  if (pre_out != nullptr && (rc = check_operand(pre_out, ldp, N))) return rc;
  LinArgs p = {};
  p.M = M;
  p.N = N;
  p.K = K;
  p.is_bf16 = dtype == 1 ? 1 : 0;
  p.act = act;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.res = res;
  p.ldr = ldr;
  p.out = out;
  p.ldo = ldo;
  p.pre = pre_out;
  p.ldp = ldp;
  return run_linear(A, lda, a_mn, B, ldb, b_mn, p, static_cast<cudaStream_t>(stream));
}

int wdit_linear_act_residual_form(int M, int N, int K, int b_mn, int* form) {
  if (form == nullptr) return WDIT_ERR_ARG;
  if (M < 1 || N < 1 || K < 1 || N % 8 != 0 || M > kMaxExtent || N > kMaxExtent || K > kMaxExtent) return WDIT_ERR_SHAPE;
  const Plan pl = plan(M, N, K, b_mn != 0, sm_count());
  form[0] = pl.pair;
  form[1] = pl.bn;
  form[2] = pl.splits;
  return WDIT_OK;
}

long long wdit_act_backward_workspace_bytes(int M, int N) {
  if (M <= kBackRows || N <= 0) return 0;  // one chunk of rows needs no second kernel
  return 4ll * ((M + kBackRows - 1) / kBackRows) * N;
}

int wdit_act_backward(const void* dout, long long ldd, const void* pre, long long ldp, int act, int dtype, int M, int N,
                      void* dpre, long long ldq, void* dbias, int dbias_dtype, void* workspace,
                      long long workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || N % 8 != 0 || M > kMaxExtent || N > kMaxExtent) return WDIT_ERR_SHAPE;
  if (dtype != 1 && dtype != 2) return WDIT_ERR_ARG;
  if (act < kNone || act > kGelu || (dbias != nullptr && (dbias_dtype < 0 || dbias_dtype > 2))) return WDIT_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (N == 0) return WDIT_OK;
  if (M == 0) {  // no rows: the bias gradient is zero
    if (dbias == nullptr) return WDIT_OK;
    return launch_error(cudaMemsetAsync(dbias, 0, static_cast<size_t>(N) * (dbias_dtype == 0 ? 4 : 2), st));
  }
  if (act == kNone && dbias == nullptr) return WDIT_OK;  // dpre is dout
  int rc = check_operand(dout, ldd, N);
  if (rc) return rc;
  if (act != kNone && ((rc = check_operand(pre, ldp, N)) || (rc = check_operand(dpre, ldq, N)))) return rc;
  const int chunks = (M + kBackRows - 1) / kBackRows;
  if (dbias != nullptr && chunks > 1) {
    if (workspace == nullptr || workspace_bytes < wdit_act_backward_workspace_bytes(M, N)) return WDIT_ERR_WORKSPACE;
    if (!aligned16(workspace)) return WDIT_ERR_ALIGN;
  }
  float* part = dbias != nullptr && chunks > 1 ? static_cast<float*>(workspace) : nullptr;
  const long long blocks = static_cast<long long>((N + kBackCols - 1) / kBackCols) * chunks;
  if (blocks > 0x7fffffffll) return WDIT_ERR_SHAPE;
  const unsigned grid = static_cast<unsigned>(blocks);
  const uint16_t* g = static_cast<const uint16_t*>(dout);
  const uint16_t* x = static_cast<const uint16_t*>(pre);
  uint16_t* d = static_cast<uint16_t*>(dpre);
  auto go = [&](auto kind) {
    constexpr int A = decltype(kind)::value;
    if (dtype == 1)
      act_backward_kernel<true, A><<<grid, 256, 0, st>>>(g, ldd, x, ldp, d, ldq, part, dbias, dbias_dtype, M, N);
    else
      act_backward_kernel<false, A><<<grid, 256, 0, st>>>(g, ldd, x, ldp, d, ldq, part, dbias, dbias_dtype, M, N);
  };
  switch (act) {
    case kRelu: go(std::integral_constant<int, kRelu>{}); break;
    case kSilu: go(std::integral_constant<int, kSilu>{}); break;
    case kGeluTanh: go(std::integral_constant<int, kGeluTanh>{}); break;
    case kGelu: go(std::integral_constant<int, kGelu>{}); break;
    default: go(std::integral_constant<int, kNone>{}); break;
  }
  rc = launch_error(cudaGetLastError());
  if (rc || part == nullptr) return rc;
  col_sum_kernel<<<(N + 31) / 32, 256, 0, st>>>(part, chunks, N, dbias, dbias_dtype);
  return launch_error(cudaGetLastError());
}

}  // extern "C"
