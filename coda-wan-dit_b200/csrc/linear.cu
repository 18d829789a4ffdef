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
// The product is a persistent warp-specialized tcgen05 kernel: warp 0 loads tiles by TMA into a
// shared-memory ring (128-byte swizzle, 64-wide K blocks), warp 1 issues the MMAs into one of two
// TMEM accumulators, warps 2-9 apply the epilogue of the other. Three tile forms (plan()):
//   pair    256 x bn tiles over CTA pairs (tcgen05 cta_group::2): many rows
//   single  128 x bn tiles, bn 64 .. 256: few tiles to spread over the SMs
//   split   128 x bn tiles whose K range is divided over a cluster of CTAs; the partial sums are
//           exchanged through distributed shared memory and added in rank order: few rows, where
//           reading B once is the bound and one CTA per tile cannot keep enough loads in flight
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
constexpr int kThreads = 320;
constexpr int kEpiThreads = 256;
constexpr uint32_t kTileABytes = BM * BK * 2;
constexpr uint32_t kTmemCols = 512;  // two accumulators of up to 256 columns
constexpr int kMaxStages = 8;
constexpr uint32_t kSmemLimit = 232448;
constexpr uint32_t kBarBytes = 256;
constexpr uint32_t kRingBudget = kSmemLimit - 1024 - kBarBytes;
constexpr int kRasterRows = 8;
constexpr long long kRasterBytes = 64ll << 20;

enum Act { kNone = 0, kGeluTanh = 1, kRelu = 2, kSilu = 3, kGelu = 4 };

struct LinArgs {
  int M, N, K;
  int m_blocks, n_blocks, k_blocks, tiles, raster_rows;
  int bn, stages, splits;
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

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// x / (1 + exp(-2 z)) = 0.5 x (1 + tanh z): no cancellation for negative x
constexpr float kGeluA = 2.f * 0.7978845608028654f;
constexpr float kGeluB = 2.f * 0.7978845608028654f * 0.044715f;

template <int N>
__device__ __forceinline__ void apply_act(float (&v)[N], int act) {
  switch (act) {
    case kRelu:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];
      break;
    case kSilu:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __fdividef(v[i], 1.f + __expf(-v[i]));
      break;
    case kGeluTanh:
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float z = v[i] * (kGeluA + kGeluB * v[i] * v[i]);
        v[i] = __fdividef(v[i], 1.f + __expf(-z));
      }
      break;
    case kGelu:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = 0.5f * v[i] * erfcf(-0.70710678118654752f * v[i]);
      break;
    default:
      break;
  }
}

__device__ __forceinline__ float act_grad(float x, int act) {
  // Past |x| = 20 every act' here is 0 or 1 to fp32; the clamp keeps x^2 finite (NaN passes).
  if (fabsf(x) > 20.f) x = copysignf(20.f, x);
  switch (act) {
    case kRelu:
      return x > 0.f ? 1.f : 0.f;
    case kSilu: {
      const float s = sigmoid(x);
      return s * (1.f + x * (1.f - s));
    }
    case kGeluTanh: {
      const float s = sigmoid(x * (kGeluA + kGeluB * x * x));
      return s + x * s * (1.f - s) * (kGeluA + 3.f * kGeluB * x * x);
    }
    case kGelu:
      return 0.5f * erfcf(-0.70710678118654752f * x) + x * 0.3989422804014327f * __expf(-0.5f * x * x);
    default:
      return 1.f;
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

enum Form { kSingle = 0, kPair = 1, kSplit = 2 };

template <int FORM, bool TA, bool TB>
__global__ void __launch_bounds__(kThreads, 1)
    linear_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                  const __grid_constant__ LinArgs p) {
  constexpr bool PAIR = FORM == kPair;
  constexpr bool SPLIT = FORM == kSplit;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int b_rows = PAIR ? p.bn / 2 : p.bn;  // B rows this CTA stages
  const uint32_t SB = kTileABytes + static_cast<uint32_t>(b_rows) * (BK * 2);
  const int stages = p.stages;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + stages * SB);
  uint64_t* empty_bar = full_bar + kMaxStages;
  uint64_t* tfull_bar = empty_bar + kMaxStages;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int cta_rank = FORM != kSingle ? static_cast<int>(cluster_ctarank()) : 0;
  const int group = PAIR ? 2 : (SPLIT ? p.splits : 1);  // CTAs that share a tile
  const int t_first = static_cast<int>(blockIdx.x) / group;
  const int t_step = static_cast<int>(gridDim.x) / group;
  const int my_count = t_first < p.tiles ? (p.tiles - 1 - t_first) / t_step + 1 : 0;
  // K blocks of this CTA (split: a contiguous share, the first ranks one more)
  int kb0 = 0, kb1 = p.k_blocks;
  if constexpr (SPLIT) {
    const int base = p.k_blocks / p.splits, rem = p.k_blocks % p.splits;
    kb0 = cta_rank * base + min(cta_rank, rem);
    kb1 = kb0 + base + (cta_rank < rem ? 1 : 0);
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

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full_bar[i], 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull_bar[i], 1);
      mbar_init(&tempty_bar[i], PAIR ? 2 * (kEpiThreads / 32) : kEpiThreads / 32);
    }
    fence_mbar_init();
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
  if constexpr (FORM != kSingle) {
    cluster_sync_all();
  } else {
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < my_count && ok; ++i) {
        int m_blk, n_blk;
        coords(i, m_blk, n_blk);
        const int n_row = n_blk * p.bn + (PAIR ? cta_rank * b_rows : 0);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_parity<PAIR, true>(&empty_bar[stage], phase ^ 1u, kSiteProducerEmpty, p.ctx)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + stage * SB;
          // Pair: both CTAs' loads complete on the leader's full barrier; only the leader arms it.
          const uint32_t fb = PAIR ? mapa_shared(smem_u32(&full_bar[stage]), 0) : smem_u32(&full_bar[stage]);
          if (!PAIR || cta_rank == 0) mbar_arrive_expect_tx(&full_bar[stage], PAIR ? 2 * SB : SB);
          auto load = [&](uint8_t* dst, const CUtensorMap* map, int x, int y) {
            if constexpr (PAIR) {
              tma_load_2d_pair(dst, map, fb, x, y);
            } else {
              tma_load_2d(dst, map, &full_bar[stage], x, y);
            }
          };
          if constexpr (TA) {
#pragma unroll
            for (int c = 0; c < BM / 64; ++c) load(st + c * 8192, &tmA, m_blk * BM + c * 64, kb * BK);
          } else {
            load(st, &tmA, kb * BK, m_blk * BM);
          }
          if constexpr (TB) {
            for (int c = 0; c < b_rows / 64; ++c) load(st + kTileABytes + c * 8192, &tmB, n_row + c * 64, kb * BK);
          } else {
            load(st + kTileABytes, &tmB, kb * BK, n_row);
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // Drain: do not leave the CTA while TMA writes into its shared memory are pending.
      for (int i = 0; i < stages; ++i) {
        if (!wait_parity<PAIR, true>(&empty_bar[stage], phase ^ 1u, kSiteDrain, p.ctx)) break;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && (!PAIR || cta_rank == 0)) {
      const uint32_t idesc = make_idesc(PAIR ? 2 * BM : BM, p.bn, p.is_bf16, TA, TB);
      int stage = 0;
      uint32_t phase = 0;
      for (int it = 0; it < my_count; ++it) {
        const int buf = it & 1;
        const uint32_t tphase = (it >> 1) & 1;
        if (!wait_parity<PAIR, true>(&tempty_bar[buf], tphase ^ 1u, kSiteMmaTmemEmpty, p.ctx)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * 256;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_parity<PAIR, true>(&full_bar[stage], phase, kSiteMmaFull, p.ctx)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + stage * SB);
          const uint64_t a_desc = TA ? smem_desc_mn(a_addr) : smem_desc_sw128(a_addr);
          const uint64_t b_desc = TB ? smem_desc_mn(a_addr + kTileABytes) : smem_desc_sw128(a_addr + kTileABytes);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            // 16 K elements on: 32 bytes inside a K-major row, 16 rows of 128 bytes MN-major
            const uint64_t ad = a_desc + (TA ? 128 : 2) * k;
            const uint64_t bd = b_desc + (TB ? 128 : 2) * k;
            const uint32_t acc = kb != kb0 || k != 0 ? 1u : 0u;
            if constexpr (PAIR) {
              mma_bf16_pair(d_tmem, ad, bd, idesc, acc);
            } else {
              mma_bf16(d_tmem, ad, bd, idesc, acc);
            }
          }
          if constexpr (PAIR) {
            mma_commit_pair(smem_u32(&empty_bar[stage]));
            mma_commit_pair(mapa_shared(smem_u32(&empty_bar[stage]), 1));
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
          mma_commit_pair(mapa_shared(smem_u32(&tfull_bar[buf]), 1));
        } else {
          mma_commit(&tfull_bar[buf]);
        }
      }
    }
    __syncwarp();
  } else {
    // Epilogue: warp w reads TMEM lanes [32 (w % 4), + 32) (its thread owns one accumulator row);
    // warps 2-5 take the even 32-column pieces of the tile, warps 6-9 the odd ones.
    const int wq = warp & 3;
    const int half = (warp - 2) >> 2;
    const int r = wq * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    for (int it = 0; it < my_count; ++it) {
      int m_blk, n_blk;
      coords(it, m_blk, n_blk);
      const int buf = it & 1;
      const uint32_t tphase = (it >> 1) & 1;
      const int row = m_blk * BM + r;
      const bool ok = wait_parity<PAIR, true>(&tfull_bar[buf], tphase, kSiteEpiTmemFull, p.ctx);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t tbase = tmem_base + lane_off + buf * 256;
      const int pieces = p.bn / 32;
      for (int c = half; c < pieces; c += 2) {
        const int n0 = n_blk * p.bn + c * 32;
        float v[32];
        tmem_ld32(tbase + c * 32, v);
        if (c + 2 >= pieces) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR) {
              mbar_arrive_cluster(mapa_shared(smem_u32(&tempty_bar[buf]), 0));
            } else {
              mbar_arrive(&tempty_bar[buf]);
            }
          }
        }
        if constexpr (SPLIT) {
          // this rank's partial tile, rows of bn + 4 floats, over the drained ring
          if (row < p.M) {
            float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(smem) + r * (p.bn + 4) + c * 32);
#pragma unroll
            for (int q = 0; q < 8; ++q) dst[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          }
        } else {
          if (n0 >= p.N) continue;
          float bias = 0.f;
          if (p.bias != nullptr) {
            if (n0 + lane < p.N) bias = load_scalar(p.bias, n0 + lane, p.bias_dtype);
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] += __shfl_sync(0xffffffffu, bias, q);
          }
          if (row < p.M) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (n0 + 8 * q >= p.N) break;
              float o[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) o[i] = v[8 * q + i];
              finish8(p, o, row, n0 + 8 * q);
            }
          }
        }
      }
    }
  }
  if constexpr (SPLIT) {
    // One tile per cluster. Rank c adds columns [c * bn / splits, + bn / splits) of all ranks'
    // partial tiles, rank 0 first.
    cluster_sync_all();
    if (warp >= 2) {
      int m_blk, n_blk;
      coords(0, m_blk, n_blk);
      const int cols = p.bn / p.splits;
      const int rows = min(BM, p.M - m_blk * BM);
      const int per_row = cols / 8;
      const uint32_t mine = smem_u32(smem);
      for (int x = threadIdx.x - 64; x < rows * per_row; x += kEpiThreads) {
        const int rr = x / per_row;
        const int c = cta_rank * cols + (x - rr * per_row) * 8;
        const int n = n_blk * p.bn + c;
        if (n >= p.N) continue;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = p.bias != nullptr ? load_scalar(p.bias, n + i, p.bias_dtype) : 0.f;
        for (int s = 0; s < p.splits; ++s) {
          const uint32_t a = mapa_shared(mine + (rr * (p.bn + 4) + c) * 4, s);
          const float4 f = ld_cluster_f4(a), g = ld_cluster_f4(a + 16);
          v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
          v[4] += g.x; v[5] += g.y; v[6] += g.z; v[7] += g.w;
        }
        finish8(p, v, m_blk * BM + rr, n);
      }
    }
  }
  tc_fence_before();
  if constexpr (FORM != kSingle) {
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
// dpre = dout * act'(pre), and the column sums of dpre by row chunks (bias gradient)
// ---------------------------------------------------------------------------
constexpr int kBackRows = 64;  // rows of one block
constexpr int kBackCols = 256;

template <bool BF16>
__global__ void __launch_bounds__(256)
    act_backward_kernel(const uint16_t* __restrict__ dout, long long ldd, const uint16_t* __restrict__ pre,
                        long long ldp, int act, uint16_t* __restrict__ dpre, long long ldq,
                        float* __restrict__ part, int M, int N) {
  __shared__ float sums[8][kBackCols];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = blockIdx.x * kBackCols + lane * 8;
  const int m0 = blockIdx.y * kBackRows;
  const int m1 = min(m0 + kBackRows, M);
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  if (n < N) {
#pragma unroll 4
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
      if (act != kNone) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(pre + m * ldp + n));
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack2(xw[i], BF16);
          d[2 * i] *= act_grad(f.x, act);
          d[2 * i + 1] *= act_grad(f.y, act);
        }
        st_global_v4(dpre + m * ldq + n, pack2(d[0], d[1], BF16), pack2(d[2], d[3], BF16), pack2(d[4], d[5], BF16),
                     pack2(d[6], d[7], BF16));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += d[i];
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[warp][lane * 8 + i] = acc[i];
  __syncthreads();
  const int c = blockIdx.x * kBackCols + threadIdx.x;
  if (c < N) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][threadIdx.x];
    part[static_cast<size_t>(blockIdx.y) * N + c] = s;
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
  if (dtype == 0) {
    static_cast<float*>(out)[n] = s;
  } else if (dtype == 1) {
    static_cast<__nv_bfloat16*>(out)[n] = __float2bfloat16_rn(s);
  } else {
    static_cast<__half*>(out)[n] = __float2half_rn(s);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
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

struct Plan {
  int form, bn, splits;
};

// Cost of one K block of a tile per CTA, in clocks: its MMAs (2 clocks per column of a 128-row
// accumulator) or its loads from L2 (about 48 bytes per clock and SM).
double block_cost(int load_rows, int bn_mma) {
  const double mma = 2.0 * bn_mma, ld = load_rows * BK * 2 / 48.0;
  return mma > ld ? mma : ld;
}

Plan plan(int M, int N, int K, int sms) {
  const int kb = (K + BK - 1) / BK;
  Plan best = {kSingle, 128, 1};
  double best_cost = 1e30;
  auto consider = [&](int form, int bn, int splits, long long tiles, long long slots, double per_block, double fixed) {
    const long long waves = (tiles + slots - 1) / slots;
    const double cost = static_cast<double>(waves) * ((kb + splits - 1) / splits * per_block + fixed) + 2000;
    if (cost < best_cost) {
      best_cost = cost;
      best = {form, bn, splits};
    }
  };
  const long long mb = (M + BM - 1) / BM;
  for (int bn = 256; bn >= 64; bn -= 64) {
    const long long nb = (N + bn - 1) / bn;
    if (M > BM && (bn == 256 || bn == 128))
      consider(kPair, bn, 1, (mb + 1) / 2 * nb, sms / 2, block_cost(BM + bn / 2, bn), 500);
    consider(kSingle, bn, 1, mb * nb, sms, block_cost(BM + bn, bn), 500);
    if (bn <= 128)
      for (int s = 2; s <= 8 && s <= kb; s *= 2)
        // one tile per cluster; 8 CTAs of a cluster need a GPC with room, so count 7/8 of the SMs
        if (mb * nb * s <= sms * 7 / 8) consider(kSplit, bn, s, mb * nb, mb * nb, block_cost(BM + bn, bn), 1500);
  }
  return best;
}

int launch_error(cudaError_t e) { return e == cudaSuccess ? WDIT_OK : WDIT_ERR_CUDA_BASE + static_cast<int>(e); }

template <int FORM, bool TA, bool TB>
int launch(const CUtensorMap& a, const CUtensorMap& b, LinArgs p, cudaStream_t stream) {
  static bool attr_set[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return launch_error(e);
  const int b_rows = FORM == kPair ? p.bn / 2 : p.bn;
  const uint32_t sb = kTileABytes + static_cast<uint32_t>(b_rows) * BK * 2;
  p.stages = static_cast<int>(kRingBudget / sb);
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  if (!attr_set[dev & 63]) {
    e = cudaFuncSetAttribute(linear_kernel<FORM, TA, TB>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (e != cudaSuccess) return launch_error(e);
    attr_set[dev & 63] = true;
  }
  const int group = FORM == kPair ? 2 : (FORM == kSplit ? p.splits : 1);
  p.tiles = (FORM == kPair ? (p.m_blocks + 1) / 2 : p.m_blocks) * p.n_blocks;
  long long grid = static_cast<long long>(p.tiles) * group;
  if (FORM != kSplit) {
    const long long slots = sm_count() / group * group;
    if (grid > slots) grid = slots;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 1024 + p.stages * sb + kBarBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = group;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = FORM != kSingle ? 1 : 0;
  return launch_error(cudaLaunchKernelEx(&cfg, linear_kernel<FORM, TA, TB>, a, b, p));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// rows x cols matrix (cols contiguous, row stride ld elements), box of box_cols x box_rows
int map_2d(CUtensorMap* m, int is_bf16, const void* ptr, int cols, int rows, long long ld, int box_cols, int box_rows) {
  const unsigned long long dims[2] = {static_cast<unsigned long long>(cols), static_cast<unsigned long long>(rows)};
  const unsigned long long strides[1] = {static_cast<unsigned long long>(ld) * 2};
  const unsigned int box[2] = {static_cast<unsigned>(box_cols), static_cast<unsigned>(box_rows)};
  return encode_tiled(m, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, ptr, dims,
                      strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int run_linear(const void* A, long long lda, int a_mn, const void* B, long long ldb, int b_mn, LinArgs p,
               cudaStream_t stream) {
  const Plan pl = plan(p.M, p.N, p.K, sm_count());
  p.bn = pl.bn;
  p.splits = pl.splits;
  p.m_blocks = (p.M + BM - 1) / BM;
  p.n_blocks = (p.N + p.bn - 1) / p.bn;
  p.k_blocks = (p.K + BK - 1) / BK;
  p.raster_rows = static_cast<long long>(p.N) * p.K * 2 > kRasterBytes ? kRasterRows : 1;
  int rc = error_record_ptr(&p.ctx.rec);
  if (rc) return rc;
  p.ctx.limit_ns = wait_limit_ns();
  const int b_rows = pl.form == kPair ? p.bn / 2 : p.bn;
  CUtensorMap ma, mb;
  rc = a_mn ? map_2d(&ma, p.is_bf16, A, p.M, p.K, lda, 64, BK) : map_2d(&ma, p.is_bf16, A, p.K, p.M, lda, BK, BM);
  if (rc) return rc;
  rc = b_mn ? map_2d(&mb, p.is_bf16, B, p.N, p.K, ldb, 64, BK) : map_2d(&mb, p.is_bf16, B, p.K, p.N, ldb, BK, b_rows);
  if (rc) return rc;
  auto go = [&](auto form) {
    constexpr int F = decltype(form)::value;
    if (a_mn) return launch<F, true, true>(ma, mb, p, stream);
    if (b_mn) return launch<F, false, true>(ma, mb, p, stream);
    return launch<F, false, false>(ma, mb, p, stream);
  };
  if (pl.form == kPair) return go(std::integral_constant<int, kPair>{});
  if (pl.form == kSplit) return go(std::integral_constant<int, kSplit>{});
  return go(std::integral_constant<int, kSingle>{});
}

int check_operand(const void* p, long long ld, long long cols) {
  if (p == nullptr) return WDIT_ERR_ARG;
  if (ld < cols) return WDIT_ERR_SHAPE;
  if (!aligned16(p) || ld % 8 != 0) return WDIT_ERR_ALIGN;
  return WDIT_OK;
}

}  // namespace
}  // namespace wdit

using namespace wdit;

extern "C" {

int wdit_linear_act_residual(const void* A, long long lda, int a_mn, const void* B, long long ldb, int b_mn, int M,
                             int N, int K, int dtype, const void* bias, int bias_dtype, int act, const void* res,
                             long long ldr, void* out, long long ldo, void* pre_out, long long ldp, void* stream) {
  if (M < 0 || N < 0 || K < 0 || N % 8 != 0) return WDIT_ERR_SHAPE;
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

long long wdit_act_backward_workspace_bytes(int M, int N) {
  if (M <= 0 || N <= 0) return 0;
  return 4ll * ((M + kBackRows - 1) / kBackRows) * N;
}

int wdit_act_backward(const void* dout, long long ldd, const void* pre, long long ldp, int act, int dtype, int M, int N,
                      void* dpre, long long ldq, void* dbias, int dbias_dtype, void* workspace,
                      long long workspace_bytes, void* stream) {
  if (M < 0 || N < 0 || N % 8 != 0) return WDIT_ERR_SHAPE;
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
  if (dbias != nullptr) {
    if (workspace == nullptr || workspace_bytes < wdit_act_backward_workspace_bytes(M, N)) return WDIT_ERR_WORKSPACE;
    if (!aligned16(workspace)) return WDIT_ERR_ALIGN;
  }
  if (chunks > 65535) return WDIT_ERR_SHAPE;
  float* part = dbias != nullptr ? static_cast<float*>(workspace) : nullptr;
  const dim3 grid((N + kBackCols - 1) / kBackCols, chunks);
  const uint16_t* g = static_cast<const uint16_t*>(dout);
  const uint16_t* x = static_cast<const uint16_t*>(pre);
  uint16_t* d = static_cast<uint16_t*>(dpre);
  if (dtype == 1)
    act_backward_kernel<true><<<grid, 256, 0, st>>>(g, ldd, x, ldp, act, d, ldq, part, M, N);
  else
    act_backward_kernel<false><<<grid, 256, 0, st>>>(g, ldd, x, ldp, act, d, ldq, part, M, N);
  rc = launch_error(cudaGetLastError());
  if (rc || part == nullptr) return rc;
  col_sum_kernel<<<(N + 31) / 32, 256, 0, st>>>(part, chunks, N, dbias, dbias_dtype);
  return launch_error(cudaGetLastError());
}

}  // extern "C"
