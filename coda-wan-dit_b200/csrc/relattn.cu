// Attention that reads a learned relative position bias from its table.
//
//   S = scale q k^T + table[bucket(j - i - q_offset), h],  key j visible for j < k_lens[b] (and
//   j <= i + q_offset when causal),  P = softmax(S) over the visible keys,  O = P v
//   (a row that sees no key gives 0 and lse = -inf).
//
// Backward, with delta = rowsum(P dP) and lse kept by the forward:
//   dV = P^T dO,  dP = dO v^T,  dS = P (dP - delta),  dQ = scale dS k,  dK = scale dS^T q,
//   dtable[bucket, h] = the sum of dS over its cells.
//
// The bias is a function of the diagonal d = key - query and constant from the last bound on, so
// the CTA looks every diagonal up to it up once. A warp's tile of 32 rows then copies its 31 +
// columns values into a short line of its own (a thread's row reads consecutive entries, free of
// bank conflicts), or uses one value when the whole tile lies past the last bound, as it does away
// from the diagonal.
//
// All products run on the tensor cores (tcgen05, operands by TMA with the 128-byte swizzle,
// accumulators in TMEM); the score tile is read from TMEM one row per thread, transformed in
// registers and written back to TMEM in 16 bits as the A operand of the next product, so nothing
// of size Lq x Lk leaves the SM.
//
// delta is rowsum(dO O) too, but O holds its own rounding and that of P to 16 bits; the error goes into
// every cell of a row with one sign, and so into the table's sums, whose cells cancel, undiminished
// (table gradient off by, relative, bf16: 5 x 2 heads x 1870 queries x 2 keys x 128 3.9e-2, with O kept
// in 32 bits still 1.5e-2, and 6e-3 at 2 heads x 2000 x 280 x 128; its own rounding alone is 1.7e-3).
// So delta is formed from P and dP as dS is, in fp32, in a first pass over the keys: 15 of
// attn_dq_kernel's 58 us at 2 x 64 heads x 512 x 512 x 64, 33 of 92 at 74 x 512 x 2048.
//
//   attn_fwd_kernel  CTA = 128 query rows of one head; key tiles of 64; one or two warps load and
//                    issue MMAs, four are the softmax (one row per thread). With few CTAs the
//                    keys are split over several, whose parts attn_combine_kernel joins.
//   attn_dq_kernel   same rows, twice over the keys: first delta, then dQ and the table's partial
//                    sums. No atomics.
//   attn_dkv_kernel  CTA = 128 keys; runs over query tiles of 64 with the scores transposed, so
//                    P^T and dS^T are the A operands; dK and dV stay in TMEM.
//
// Measured (bf16): forward, 12 heads x 8192 x 8192 x 128 causal 187 - 205 us by the card's power, 1.0 -
// 1.1 PFLOP/s, tensor pipe and exponentials 55% busy each; 2 x 64 heads x 512 x 512 x 64 with lengths
// 512 and 227 22.4 us, of which a CTA's start and end are 4; one query over 8 x 12 heads x 8191 keys x
// 128 66 us, 6.1 TB/s. Backward at 2 x 64 heads x 512 x 512 x 64: dQ 58 us (fp16 63), dK and dV 46. What
// bounds the tiles is latency: a score tile passes from the MMAs to a warp and back over two barriers, about
// 200 clocks each behind the other warps' exponentials, besides its TMEM reads; more CTAs per SM,
// scores read ahead and polynomial exponentials were all slower.
//
// Keys past k_lens, and under a causal mask past the last query, may hold anything (NaN included):
// their scores are replaced, and their rows of an operand that is summed over are overwritten with
// zeros in shared memory.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "ptx.cuh"
#include "relpos.cuh"
#include "tmap.h"
#include "wdit_internal.h"

namespace wdit {

int launch_rel_table_sum(const float* part, int parts, int buckets, int H, void* out, int dtype, void* stream);

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_huge_valf();
constexpr int kRows = 128;  // accumulator rows of a CTA
constexpr int kCols = 64;   // columns of a score tile
constexpr int kMaxSplits = 64;
enum : unsigned int { kSiteAttn = 16, kSiteAttnDq = 32, kSiteAttnDkv = 48 };

struct AttnArgs {
  int B, H, Lq, Lk;
  int causal, q_offset;
  float scale;
  const int* k_lens;   // [B] or nullptr
  const void* table;   // [buckets, H]
  int table_dtype;
  RelBuckets rb;
  void* out;           // [B, Lq, H, D] contiguous
  float* lse;          // [B, H, Lq], log2 units; nullable
  int splits;          // forward: key splits; > 1 writes part_o / part_lse instead
  float* part_o;       // [splits][B * H * Lq][D]
  float* part_lse;     // [splits][B * H * Lq]
  // backward
  float* delta;        // [B, H, Lq]
  unsigned* tops;      // [B, H][4 q tiles], fp16: bounds of |dS| by 32 rows, as the bits of a float >= 0
  float* table_part;   // [H][B * q tiles][buckets]
  WaitCtx ctx;
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (BF16) return pack_bf16x2(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
  if constexpr (BF16) return unpack_bf16x2(w);
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float table_value(const AttnArgs& p, int b, int h) {
  const long long i = static_cast<long long>(b) * p.H + h;
  if (p.table_dtype == 0) return static_cast<const float*>(p.table)[i];
  if (p.table_dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16*>(p.table)[i]);
  return __half2float(static_cast<const __half*>(p.table)[i]);
}

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int h, int l,
                                            int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(h), "r"(l), "r"(b)
      : "memory");
}

__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int x, int h, int l, int b) {
  asm volatile(
      "cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(src)), "r"(x), "r"(h), "r"(l), "r"(b)
      : "memory");
}

// D[tmem] (+)= A[tmem, 16-bit, two K elements per column] * B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st32f(uint32_t taddr, const float* v) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(v[i]);
  tmem_st16(taddr, r);
  tmem_st16(taddr + 16, r + 16);
}

__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
      "[%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// The wait names the registers, so that no use of them is moved before it.
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}

// 32 columns from each of two places with one wait: both loads are in flight together.
__device__ __forceinline__ void tmem_ld32x2(uint32_t a, float* v, uint32_t b, float* w) {
  uint32_t r[32], q[32];
  tmem_ld32_nowait(a, r);
  tmem_ld32_nowait(b, q);
  tmem_wait_ld(r);
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(q[i]));
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    v[i] = __uint_as_float(r[i]);
    w[i] = __uint_as_float(q[i]);
  }
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// MN-major operand tile of ROWS K indices: rows of 64 elements (128 B) along M or N, one row per K
// index; pieces of 64 elements are ROWS x 128 B apart.
template <int ROWS>
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>((ROWS * 128u) >> 4) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}

__host__ __device__ constexpr uint32_t idesc16(int m, int n, bool bf16, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// Score product of a 128-row tile and a COLS-row tile, both K-major over D (pieces of 64 columns,
// 128 bytes a row).
template <int D, int COLS>
__device__ __forceinline__ void issue_scores(uint32_t d_tmem, uint32_t a128, uint32_t b_tile, uint32_t idesc) {
  const uint64_t a = smem_desc_sw128(a128), b = smem_desc_sw128(b_tile);
#pragma unroll
  for (int k = 0; k < D / 16; ++k)
    mma_bf16(d_tmem, a + (k >> 2) * (kRows * 8) + (k & 3) * 2, b + (k >> 2) * (COLS * 8) + (k & 3) * 2, idesc,
             k != 0 ? 1u : 0u);
}

// acc[128, D] (+)= A[128 x COLS, TMEM] * B[COLS x D, shared memory rows]. The two halves of A's
// columns are written by different warps, each over the scores it read: COLS / 2 TMEM columns apart.
template <int COLS>
__device__ __forceinline__ void issue_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_tile, uint32_t idesc,
                                         bool accum) {
  const uint64_t b = smem_desc_mn<COLS>(b_tile);
  constexpr int H = COLS / 32;  // MMAs of 16 K indices in a half
#pragma unroll
  for (int k = 0; k < COLS / 16; ++k)
    mma_ts(d_tmem, a_tmem + (k / H) * (COLS / 2) + (k % H) * 8, b + 128 * k, idesc, accum || k != 0 ? 1u : 0u);
}

// Zero rows [first, ROWS) of a tile (whole 128-byte rows: the swizzle stays inside a row).
template <int D, int ROWS>
__device__ __forceinline__ void zero_tail(uint8_t* tile, int first, int lane) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
    for (int x = first * 8 + lane; x < ROWS * 8; x += 32)
      *reinterpret_cast<uint4*>(tile + c * (ROWS * 128) + x * 16) = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  __syncwarp();
}

// The head's bias by diagonal: the table's values (bias_log2) and buckets of d = -reach .. reach,
// constant past both ends, in shared memory. reach is the last bound, at most kReach: a table with
// longer ones is searched per diagonal instead.
constexpr int kReach = 1024;

// A bias in units of log2 e. Finite ones end at 2^14 on either side: a table may hold its type's lowest
// value (or -1e9) as a mask, and a row that sees nothing but such keys still has to tell their scores
// apart, in fp32, in its maximum and its log-sum (half a step there is 2^-10). Next to any other
// key the weight of such a one is 0 as before, unless their scores are more than 11356 apart.
constexpr float kBiasMost = 16384.f;
__device__ __forceinline__ float bias_log2(float v) {
  float x = v * kLog2e;  // infinities and NaN stay
  if (x < -kBiasMost && v > -kInf) x = -kBiasMost;
  if (x > kBiasMost && v < kInf) x = kBiasMost;
  return x;
}

struct BiasLine {
  const int* bounds;
  const float* col;    // [buckets] bias_log2 of the table's column
  const float* value;  // [2 reach + 1] unless searched
  int n_bounds, bidirectional, reach;
  bool searched;

  __device__ __forceinline__ int bucket(int d) const { return rel_bucket(bounds, n_bounds, bidirectional, d); }
  __device__ __forceinline__ float at(int d) const {
    if (searched) return col[bucket(d)];
    return value[min(max(d, -reach), reach) + reach];
  }
  // One bucket each: d <= -reach, and d >= ahead() (past the last bound, or ahead of the query in
  // one direction).
  __device__ __forceinline__ int ahead() const { return bidirectional ? reach : 0; }
};

__host__ __device__ inline int bias_reach(const RelBuckets& rb) { return rb.bounds[rb.n_bounds - 1]; }

// Shared memory of load_bias in bytes (16-byte multiples).
inline int bias_smem(const RelBuckets& rb) {
  const int buckets = rel_num_buckets(rb.n_bounds, rb.bidirectional);
  const int reach = bias_reach(rb);
  return (1024 + buckets * 4 + (reach <= kReach ? (2 * reach + 1) * 4 : 0) + 15) / 16 * 16;
}

__device__ __forceinline__ BiasLine load_bias(const AttnArgs& p, int h, void* mem, int threads) {
  int* bounds = static_cast<int*>(mem);
  float* col = reinterpret_cast<float*>(bounds + 256);
  const int buckets = rel_num_buckets(p.rb.n_bounds, p.rb.bidirectional);
  BiasLine l;
  l.bounds = bounds;
  l.col = col;
  l.n_bounds = p.rb.n_bounds;
  l.bidirectional = p.rb.bidirectional;
  l.reach = bias_reach(p.rb);
  l.value = col + buckets;
  l.searched = l.reach > kReach;
  for (int t = threadIdx.x; t < p.rb.n_bounds; t += threads) bounds[t] = p.rb.bounds[t];
  for (int t = threadIdx.x; t < buckets; t += threads) col[t] = bias_log2(table_value(p, t, h));
  if (!l.searched) {
    __syncthreads();
    for (int t = threadIdx.x; t < 2 * l.reach + 1; t += threads) col[buckets + t] = col[l.bucket(t - l.reach)];
  }
  return l;
}

__device__ __forceinline__ int sample_len(const AttnArgs& p, int b) {
  if (p.k_lens == nullptr) return p.Lk;
  const int n = p.k_lens[b];
  return n < 0 ? 0 : (n > p.Lk ? p.Lk : n);
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
// Four softmax warps, one row per thread: warp w reads TMEM lanes [32 (w % 4), + 32). NB = 2: two CTAs
// per SM with two score buffers each; the scores of t + 1 are computed while those of t are
// exponentiated, so the softmax never waits for a product. One more warp loads, another issues
// MMAs. NB = 1 (D = 64): four CTAs per SM with one buffer each (128 TMEM columns, 96 registers a
// thread) and one warp that loads and issues; a CTA's products and softmax take turns, and the
// CTAs fill each other's gaps, starts and ends.
//
// The maximum in use is that of the row's first tile (bf16: 2^kHeadroom above it). Later tiles are
// exponentiated against it without looking for theirs; only when a tile's sum passes kSumLimit is
// the maximum taken anew, O rescaled and the tile done again. What bounds the two:
//   fp16  P up to 2^15 of its 65504; P v is then far inside fp32.
//   bf16  v may be as large as fp32 goes, so the row's sum of P stays below 1: at most 2^22 tiles of
//         at most 2^-22 each. The largest P of a tile whose maximum was taken is 2^-40: P may rise by
//         2^18 in one key, 2^12 in all 64 of a tile, before it is taken anew. P keeps its relative
//         precision down to 2^-86 of the largest, and O that of |v| from 2^-86 on.
template <bool BF16>
struct SoftmaxRange {
  static constexpr float kHeadroom = BF16 ? 40.f : 0.f;                // log2
  static constexpr float kSumLimit = BF16 ? 2.3841858e-07f : 32768.f;  // 2^-22, 2^15
};

template <int D, int NB>
struct Fwd {
  static constexpr int kCtas = NB == 1 ? 4 : 2;     // per SM
  static constexpr int kControl = NB == 1 ? 1 : 2;  // warps that load and issue
  static constexpr int kStages = D == 64 && NB == 2 ? 4 : 2;
  static constexpr int kThreads = 32 * (kControl + 4);
  static constexpr uint32_t kQ = kRows * D * 2;
  static constexpr uint32_t kTile = kCols * D * 2;
  static constexpr uint32_t kTmem = NB == 1 ? 128 : 256;  // score buffers of 64 columns, then O
  static constexpr int kLine = 96;        // per-warp bias line (31 + 64 diagonals)
  static int smem(const RelBuckets& rb) { return 1024 + kQ + kStages * 2 * kTile + 256 + 4 * kLine * 4 + bias_smem(rb); }
};

// Linear block index -> (query tile, split, head, sample). Under a causal mask the last query rows
// see most keys: all heads' last tiles go first, so that the short ones fill the end. Otherwise
// the query tile is fastest: its CTAs share K and V in L2.
struct FwdPlace {
  int qt, split, h, b;
};
__device__ __forceinline__ FwdPlace fwd_place(const AttnArgs& p, int q_tiles) {
  unsigned x = blockIdx.x;
  FwdPlace f;
  if (p.causal) {
    f.h = x % p.H;
    x /= p.H;
    f.b = x % p.B;
    x /= p.B;
    f.split = x % p.splits;
    f.qt = q_tiles - 1 - static_cast<int>(x / p.splits);
  } else {
    f.qt = x % q_tiles;
    x /= q_tiles;
    f.split = x % p.splits;
    x /= p.splits;
    f.h = x % p.H;
    f.b = x / p.H;
  }
  return f;
}

template <int D, bool BF16, int NB>
__global__ void __launch_bounds__(Fwd<D, NB>::kThreads, Fwd<D, NB>::kCtas)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmOut,
                    const __grid_constant__ AttnArgs p) {
  using C = Fwd<D, NB>;
  constexpr int ST = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + C::kQ;
  uint8_t* sV = sK + ST * C::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + ST * C::kTile);
  uint64_t* k_full = bars;
  uint64_t* k_empty = bars + ST;
  uint64_t* v_full = bars + 2 * ST;
  uint64_t* v_empty = bars + 3 * ST;
  uint64_t* q_full = bars + 4 * ST;
  uint64_t* s_full = q_full + 1;   // 2
  uint64_t* p_ready = s_full + 2;  // 2: a warp may finish its rows of t + 1 before another's of t
  uint64_t* pv_done = p_ready + 2;
  uint64_t* last = pv_done + 1;  // every product is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(last + 1);
  float* lines = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 256);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_tiles = (p.Lq + kRows - 1) / kRows;
  const FwdPlace at = fwd_place(p, q_tiles);
  const int h = at.h, b = at.b, split = at.split;
  const int i0 = at.qt * kRows;
  const int klen = sample_len(p, b);
  int visible = klen;  // keys any row of the tile sees
  if (p.causal) visible = min(visible, min(i0 + kRows, p.Lq) + p.q_offset);
  int t0 = 0, t1 = (visible + kCols - 1) / kCols;
  if (p.splits > 1) {
    const int tiles = (klen + kCols - 1) / kCols;
    const int per = (tiles + p.splits - 1) / p.splits;
    t0 = split * per;
    t1 = min(t1, t0 + per);
  }
  const int n = max(0, t1 - t0);

  auto load_k = [&](int t) {
    const int st = t % ST;
    mbar_arrive_expect_tx(&k_full[st], C::kTile);
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      tma_load_4d(sK + st * C::kTile + c * 8192, &tmK, &k_full[st], c * 64, h, (t0 + t) * kCols, b);
  };
  auto load_v = [&](int t) {
    const int st = t % ST;
    mbar_arrive_expect_tx(&v_full[st], C::kTile);
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
      tma_load_4d(sV + st * C::kTile + c * 8192, &tmV, &v_full[st], c * 64, h, (t0 + t) * kCols, b);
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
    }
    mbar_init(pv_done, 1);
    mbar_init(last, 1);
    fence_mbar_init();
    // the first loads run under the rest of the set-up
    if (n > 0) {
      mbar_arrive_expect_tx(q_full, C::kQ);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) tma_load_4d(sQ + c * 16384, &tmQ, q_full, c * 64, h, i0, b);
      for (int t = 0; t < min(n, ST); ++t) {
        load_k(t);
        load_v(t);
      }
    }
  }
  __syncwarp();
  if (warp == C::kControl - 1) {
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  const BiasLine bias = load_bias(p, h, lines + 4 * C::kLine, C::kThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_o = tmem + NB * kCols;

  if (NB == 2 && warp == 0) {
    if (elect_one() && n > 0) {
      int k_loaded = min(n, ST), v_loaded = k_loaded;
      for (int t = ST; t < n; ++t) {
        const uint32_t ph = (t / ST) & 1;
        if (!wait_parity(&k_empty[t % ST], ph ^ 1u, kSiteAttn, p.ctx)) break;
        load_k(t);
        k_loaded = t + 1;
        if (!wait_parity(&v_empty[t % ST], ph ^ 1u, kSiteAttn + 1, p.ctx)) break;
        load_v(t);
        v_loaded = t + 1;
      }
      // Do not leave while a copy into this CTA's shared memory is in flight.
      wait_parity(q_full, 0, kSiteAttn + 2, p.ctx);
      for (int t = max(0, k_loaded - ST); t < k_loaded; ++t)
        wait_parity(&k_full[t % ST], (t / ST) & 1, kSiteAttn + 2, p.ctx);
      for (int t = max(0, v_loaded - ST); t < v_loaded; ++t)
        wait_parity(&v_full[t % ST], (t / ST) & 1, kSiteAttn + 2, p.ctx);
    }
    __syncwarp();
  } else if (warp == C::kControl - 1) {
    constexpr uint32_t id_s = idesc16(kRows, kCols, BF16, false);
    constexpr uint32_t id_o = idesc16(kRows, D, BF16, true);
    auto scores = [&](int t) {
      const int st = t % ST;
      const bool ok = wait_parity(&k_full[st], (t / ST) & 1, kSiteAttn + 3, p.ctx);
      if (!__all_sync(0xffffffffu, ok)) return false;
      tc_fence_after();
      if (elect_one()) {
        issue_scores<D, kCols>(tmem + (t % NB) * kCols, smem_u32(sQ), smem_u32(sK + st * C::kTile), id_s);
        if (NB == 2) mma_commit(&k_empty[st]);
        mma_commit(&s_full[t % NB]);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    int loaded = min(n, ST);
    if (n > 0) {
      ok = wait_parity(q_full, 0, kSiteAttn + 4, p.ctx);
      ok = __all_sync(0xffffffffu, ok) && scores(0);
    }
    for (int t = 0; t < n && ok; ++t) {
      if (NB == 2 && t + 1 < n) {
        // scores(t + 1) overwrite the buffer whose P the product of t - 1 reads: products into
        // different accumulators are ordered by their completion only
        if (t > 0) ok = __all_sync(0xffffffffu, wait_parity(pv_done, (t - 1) & 1, kSiteAttn + 10, p.ctx));
        if (!ok || !scores(t + 1)) break;
      }
      const int st = t % ST;
      ok = wait_parity(&v_full[st], (t / ST) & 1, kSiteAttn + 5, p.ctx);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      const int j0 = (t0 + t) * kCols;
      // rows past the keys that any query of the tile sees would enter O as 0 * anything
      if (j0 + kCols > visible) zero_tail<D, kCols>(sV + st * C::kTile, visible - j0, lane);
      ok = wait_parity(&p_ready[t % NB], (t / NB) & 1, kSiteAttn + 6, p.ctx);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      if (elect_one()) {
        issue_ts<kCols>(tmem_o, tmem + (t % NB) * kCols, smem_u32(sV + st * C::kTile), id_o, t > 0);
        if (NB == 2) mma_commit(&v_empty[st]);
        mma_commit(pv_done);
        if (t + 1 == n) mma_commit(last);
      }
      __syncwarp();
      if (NB == 1 && t + 1 < n) {
        // the next scores take the place of the P that this product reads; its tiles are free too
        ok = __all_sync(0xffffffffu, wait_parity(pv_done, t & 1, kSiteAttn + 10, p.ctx));
        if (!ok || !scores(t + 1)) break;
        if (t + ST < n) {
          if (elect_one()) {
            load_k(t + ST);
            load_v(t + ST);
          }
          __syncwarp();
          loaded = t + ST + 1;
        }
      }
    }
    // Do not leave while a copy into this CTA's shared memory is in flight: all that was loaded has
    // been waited for unless a wait ran out.
    if (NB == 1 && !ok) {
      wait_parity(q_full, 0, kSiteAttn + 2, p.ctx);
      for (int t = max(0, loaded - ST); t < loaded; ++t) {
        wait_parity(&k_full[t % ST], (t / ST) & 1, kSiteAttn + 2, p.ctx);
        wait_parity(&v_full[t % ST], (t / ST) & 1, kSiteAttn + 2, p.ctx);
      }
    }
  } else {
    const int wq = warp & 3;
    const int i = i0 + wq * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    float* line = lines + wq * C::kLine;
    const uint64_t scale2 = f2_pack(p.scale * kLog2e, p.scale * kLog2e);
    const int row_end = p.causal ? min(klen, i + p.q_offset + 1) : klen;  // keys this row sees
    const int warp_first = i0 + wq * 32 + p.q_offset;                      // the warp's first position
    using Range = SoftmaxRange<BF16>;
    float m_used = -kInf, l = 0.f;
    bool ok = true;
    // Few query rows (one token): a warp without any leaves its rows of P as they are; they only
    // reach its own rows of O, which are not stored.
    const bool idle = i0 + wq * 32 >= p.Lq;
    // The warp's tiles by kind: bias of the last bucket on the left before t_left and on the right
    // from t_right on, some rows' keys ending inside from t_mask on (row_end rises with the lane).
    const int first_key = t0 * kCols;
    const int t_left = (warp_first - bias.reach - (kCols - 1) - first_key + kCols) / kCols;
    const int t_right = (warp_first + 31 + bias.ahead() - first_key + kCols - 1) / kCols;
    const int t_mask = (__shfl_sync(0xffffffffu, row_end, 0) - first_key) / kCols;
    const float c_left = bias.at(-bias.reach), c_right = bias.at(bias.reach);
    for (int t = 0; t < n; ++t) {
      const int j0 = (t0 + t) * kCols;
      const uint32_t ts = tmem + lane_off + (t % NB) * kCols;
      const bool masked = t >= t_mask;
      const bool flat = !masked && (t < t_left || t >= t_right);
      const float flat_c = t < t_left ? c_left : c_right;
      const int keep = row_end - j0;
      if (!flat && !idle) {
        const int d_lo = j0 - warp_first - 31;  // a line over the tile's 31 + 64 diagonals
        __syncwarp();                           // the previous tile's reads are done
#pragma unroll
        for (int q = 0; q < 3; ++q) line[lane + 32 * q] = bias.at(d_lo + lane + 32 * q);
        __syncwarp();
      }
      const float* ln = line + 31 - lane;
      ok = wait_parity(&s_full[t % NB], (t / NB) & 1, kSiteAttn + 7, p.ctx);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      if (idle) {
        if (lane == 0) mbar_arrive(&p_ready[t % NB]);
        continue;
      }
      tc_fence_after();
      uint32_t w[32];
      float sum = 0.f;
      // P of the tile against the maximum in use: 16-bit pairs in w, their sum before rounding in
      // `sum`. One instance for each kind of tile, so that nothing is decided per element.
      auto exponentiate = [&](auto is_flat, auto is_masked) {
        const float m = m_used == -kInf ? 0.f : m_used;
        const uint64_t sub = decltype(is_flat)::value ? f2_pack(flat_c - m, flat_c - m) : f2_pack(-m, -m);
        uint64_t s2[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
        // two CTAs per SM leave the registers to load both halves at once
        constexpr int HELD = NB == 2 ? 2 : 1;
        uint32_t raw[HELD][32];
        if constexpr (HELD == 2) {
          tmem_ld32_nowait(ts, raw[0]);
          tmem_ld32_nowait(ts + 32, raw[1]);
          tmem_wait_ld(raw[0]);
#pragma unroll
          for (int e = 0; e < 32; ++e) asm volatile("" : "+r"(raw[1][e]));
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if constexpr (HELD == 1) {
            tmem_ld32_nowait(ts + c * 32, raw[0]);
            tmem_wait_ld(raw[0]);
          }
          uint32_t* r = raw[c % HELD];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            uint64_t add = sub;
            if constexpr (!decltype(is_flat)::value)
              add = fadd2(f2_pack(ln[c * 32 + 2 * e], ln[c * 32 + 2 * e + 1]), sub);
            float x, y;
            f2_unpack(ffma2(f2_pack(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), scale2, add),
                      x, y);
            if constexpr (decltype(is_masked)::value) {
              x = c * 32 + 2 * e < keep ? x : -kInf;
              y = c * 32 + 2 * e + 1 < keep ? y : -kInf;
            }
            x = exp2_approx(x);
            y = exp2_approx(y);
            s2[e & 1] = fadd2(s2[e & 1], f2_pack(x, y));
            w[c * 16 + e] = pack16<BF16>(x, y);
          }
        }
        float x, y;
        f2_unpack(fadd2(s2[0], s2[1]), x, y);
        sum = x + y;
      };
      const std::true_type yes;
      const std::false_type no;
      bool settled = false;
      for (bool first = t == 0;; first = false) {
        if (!first) {
          if (masked)
            exponentiate(no, yes);  // the line serves flat tiles too
          else if (flat)
            exponentiate(yes, no);
          else
            exponentiate(no, no);
          if (settled || !__any_sync(0xffffffffu, m_used == -kInf || sum > Range::kSumLimit)) break;
        }
        // The row's maximum anew; everything before is rescaled to it, once the product of t - 1
        // has left O at rest.
        float m_tile = -kInf;
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          float z[32];
          tmem_ld32(ts + c * 32, z);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float x = fmaf(z[e], p.scale * kLog2e, flat ? flat_c : ln[c * 32 + e]);
            m_tile = fmaxf(m_tile, c * 32 + e < keep ? x : -kInf);
          }
        }
        const float m_new = fmaxf(m_used, m_tile + Range::kHeadroom);
        if (t > 0) {
          ok = wait_parity(pv_done, (t - 1) & 1, kSiteAttn + 8, p.ctx);
          if (!(ok = __all_sync(0xffffffffu, ok))) break;
          tc_fence_after();
          const float f = m_new == -kInf ? 1.f : exp2_approx(m_used - m_new);
          l *= f;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tmem_ld32(tmem_o + lane_off + c * 32, o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= f;
            tmem_st32f(tmem_o + lane_off + c * 32, o);
          }
        }
        m_used = m_new;
        settled = true;
      }
      if (!ok) break;
      l += sum;
      tmem_st16(ts, w);
      tmem_st16(ts + 32, w + 16);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[t % NB]);
    }
    if (ok && n > 0) {
      ok = wait_parity(last, 0, kSiteAttn + 9, p.ctx);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    const bool any = l > 0.f || l != l;
    const float inv = any ? 1.f / l : 0.f;
    const float lse = any ? m_used + log2f(l) : -kInf;
    const long long hrow = (static_cast<long long>(b) * p.H + h) * p.Lq + i;
    const long long slot = static_cast<long long>(split) * p.B * p.H * p.Lq + hrow;
    if (i < p.Lq) {
      if (p.splits > 1) {
        p.part_lse[slot] = lse;
      } else if (p.lse != nullptr) {
        p.lse[hrow] = lse;
      }
    }
    // The rows go out through the query tile's shared memory (every product that reads it is
    // done), 32 rows x 128 bytes a TMA store and warp: rows past Lq are left out by the map.
    uint8_t* stage = sQ + wq * 32 * 128;
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      float o[32];
      if (n > 0 && ok) {
        tmem_ld32(tmem_o + lane_off + c * 32, o);
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0.f;
      }
      // a row without keys is 0 whatever its accumulator holds
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = any ? o[e] * inv : 0.f;
      if (p.splits > 1) {
        if (i >= p.Lq) continue;
        float4* po = reinterpret_cast<float4*>(p.part_o + slot * D + c * 32);
#pragma unroll
        for (int q = 0; q < 8; ++q) po[q] = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        continue;
      }
      const uint32_t row = smem_u32(stage + (c >> 1) * 16384) + lane * 128;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        st_shared_v4(row + ((((c & 1) * 4 + q) ^ (lane & 7)) << 4), pack16<BF16>(o[8 * q], o[8 * q + 1]),
                     pack16<BF16>(o[8 * q + 2], o[8 * q + 3]), pack16<BF16>(o[8 * q + 4], o[8 * q + 5]),
                     pack16<BF16>(o[8 * q + 6], o[8 * q + 7]));
    }
    if (p.splits == 1) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (i0 + wq * 32 < p.Lq) {
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_store_4d(&tmOut, stage + c * 16384, c * 64, h, i0 + wq * 32, b);
        }
        bulk_commit();
        bulk_wait_read<0>();  // the stores have read shared memory
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::kControl - 1) tmem_dealloc(tmem, C::kTmem);
}

// out = sum_s 2^(lse_s - lse) part_o[s], lse = log2 sum_s 2^lse_s: one warp per row.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) attn_combine_kernel(const __grid_constant__ AttnArgs p) {
  const long long rows = static_cast<long long>(p.B) * p.H * p.Lq;
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  constexpr int V = D / 32;  // columns per lane
  constexpr int kAhead = 4;  // parts in flight: the first ones are loaded together with the sums
  const float* src = p.part_o + row * D + lane * V;
  float part[kAhead][V];
  auto load = [&](int base) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int q = 0; q < V; ++q) part[s][q] = base + s < p.splits ? src[(base + s) * rows * D + q] : 0.f;
  };
  load(0);
  static_assert(kMaxSplits == 64, "two parts a lane");
  const float lse0 = lane < p.splits ? p.part_lse[lane * rows + row] : -kInf;
  const float lse1 = lane + 32 < p.splits ? p.part_lse[(lane + 32) * rows + row] : -kInf;
  float m = fmaxf(lse0, lse1);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float ms = m == -kInf ? 0.f : m;
  float w0 = exp2f(lse0 - ms), w1 = exp2f(lse1 - ms);
  float total = w0 + w1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  // weights that add up to 1: a sum of parts near the type's largest value stays inside it
  const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
  w0 *= inv;
  w1 *= inv;
  float acc[V];
#pragma unroll
  for (int q = 0; q < V; ++q) acc[q] = 0.f;
  for (int base = 0; base < p.splits; base += kAhead) {
    float now[kAhead][V];
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int q = 0; q < V; ++q) now[s][q] = part[s][q];
    load(base + kAhead);
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {  // (weights past the last part are 0)
      const float w = __shfl_sync(0xffffffffu, base < 32 ? w0 : w1, (base + s) & 31);
#pragma unroll
      for (int q = 0; q < V; ++q) acc[q] = w == 0.f ? acc[q] : fmaf(w, now[s][q], acc[q]);
    }
  }
  const int i = static_cast<int>(row % p.Lq);
  const int h = static_cast<int>(row / p.Lq % p.H);
  const long long b = row / p.Lq / p.H;
  uint16_t* dst = static_cast<uint16_t*>(p.out) + ((b * p.Lq + i) * p.H + h) * D + lane * V;
#pragma unroll
  for (int q = 0; q < V; q += 2)
    *reinterpret_cast<uint32_t*>(dst + q) = pack16<BF16>(acc[q], acc[q + 1]);
  if (lane == 0 && p.lse != nullptr) p.lse[row] = inv == 0.f ? -kInf : ms + log2f(total);
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
// Eight compute warps: warp w reads TMEM lanes [32 (w % 4), + 32), warps 2-5 columns 0-31 of a
// score tile, warps 6-9 columns 32-63. D = 64: two CTAs per SM overlap each other; D = 128: one
// CTA per SM with two score buffers.
constexpr int kSumReach = 256;  // the table's gradient is summed by diagonal up to this last bound

// fp16 only: P and dS enter their products times a power of two. P is normalised (1 / Lk of flat
// scores) and dS as small as the loss's scale makes it; below 2^-14 fp16 loses their bits one by one,
// above 65504 it ends. P is taken times 2^14. dS is taken up to a bound of its size, 2^14 at most: for dQ
// the row's max |P dP| + |delta|, which the first pass over the keys gives; for dK, whose sums run over the
// rows, the largest of these of the head. So what a cell may lose is 2^-38 of that bound. A bound of 0,
// infinity or NaN takes none; past 2^60 the gradients are below fp16 whatever their factor, and |dP| of fp16
// operands stays below 2^39. The row's maximum and the factor cost attn_dq_kernel 5 of 63 us at 2 x 64
// heads x 512 x 512 x 64 (99 against 91 at 74 x 512 x 2048), attn_dkv_kernel 1 of 46.
constexpr int kPScale = 14;
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((127 + e) << 23); }  // -126 .. 127
__device__ __forceinline__ int grad_scale(unsigned bound_bits) {                          // log2 of dS's factor
  const int e = static_cast<int>(bound_bits >> 23) - 127;  // bound < 2^(e + 1)
  return bound_bits == 0 || e == 128 ? 0 : max(min(13 - e, 60), -60);
}
template <int D>
struct Bwd {
  static constexpr int kThreads = 320;
  static constexpr int kCtas = D == 64 ? 2 : 1;
  static constexpr int kBuf = D == 64 ? 1 : 2;
  static constexpr int kStages = 2;
  static constexpr uint32_t kTmem = D == 64 ? 256 : 512;
  static constexpr uint32_t kBig = kRows * D * 2;
  static constexpr uint32_t kTile = kCols * D * 2;
  static constexpr int kWarp = 64 + 96 + 64;  // floats per warp: bias line, diagonals, row values
  static int smem(const RelBuckets& rb) {
    return 1024 + 2 * kBig + kStages * 2 * kTile + 256 + 8 * kWarp * 4 + 8 * 4 * grad_sums(rb) + 4 * kRows * 4 +
           bias_smem(rb);
  }
  // Floats of a warp's sums of the table's gradient: by diagonal, or by bucket.
  __host__ __device__ static int grad_sums(const RelBuckets& rb) {
    const int reach = bias_reach(rb);
    const int n = reach <= kSumReach ? reach + (rb.bidirectional ? reach : 0) + 1
                                     : rel_num_buckets(rb.n_bounds, rb.bidirectional);
    return (n + 3) / 4 * 4;
  }
};

// 32 rows of a warp's accumulator, 64 columns from `tmem` on, times `mult`, through shared memory (32
// rows of 128 bytes, swizzled) out by TMA. zero: the rows of lanes without a result.
template <bool BF16>
__device__ __forceinline__ void store_rows64(const CUtensorMap* map, uint8_t* stage, uint32_t tmem, bool has, bool zero,
                                             float mult, int lane, int x, int h, int l, int b, bool inside) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float o[32];
    if (has) {
      tmem_ld32(tmem + c * 32, o);
    } else {
#pragma unroll
      for (int e = 0; e < 32; ++e) o[e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 32; ++e) o[e] = zero ? 0.f : o[e] * mult;
    const uint32_t row = smem_u32(stage) + lane * 128;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      st_shared_v4(row + (((c * 4 + q) ^ (lane & 7)) << 4), pack16<BF16>(o[8 * q], o[8 * q + 1]),
                   pack16<BF16>(o[8 * q + 2], o[8 * q + 3]), pack16<BF16>(o[8 * q + 4], o[8 * q + 5]),
                   pack16<BF16>(o[8 * q + 6], o[8 * q + 7]));
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    if (inside) tma_store_4d(map, stage, x, h, l, b);
    bulk_commit();
  }
}

__device__ __forceinline__ uint64_t exp2_2(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return f2_pack(exp2_approx(a), exp2_approx(b));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(Bwd<D>::kThreads, Bwd<D>::kCtas)
    attn_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                   const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ AttnArgs p) {
  using C = Bwd<D>;
  constexpr int ST = C::kStages;
  constexpr int NB = C::kBuf;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sO = sQ + C::kBig;  // dO
  uint8_t* sK = sO + C::kBig;
  uint8_t* sV = sK + ST * C::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + ST * C::kTile);
  uint64_t* full = bars;          // K and V of a stage
  uint64_t* empty = bars + ST;
  uint64_t* q_full = bars + 2 * ST;
  uint64_t* s_full = q_full + 1;  // NB
  uint64_t* ds_ready = s_full + 2;  // NB
  uint64_t* done = ds_ready + 2;
  uint64_t* last = done + 1;  // every product is done
  uint64_t* delta_ready = last + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(delta_ready + 1);
  float* warps = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 256);
  const int reach = bias_reach(p.rb);
  const bool by_diag = reach <= kSumReach;
  const int nsum = C::grad_sums(p.rb);
  float* sums = warps + 8 * C::kWarp;  // [8][nsum]
  float* sdelta = sums + 8 * nsum;     // [2][128]
  float* stop = sdelta + 2 * kRows;    // [2][128]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_tiles = (p.Lq + kRows - 1) / kRows;
  int x = blockIdx.x;
  const int qt = q_tiles - 1 - x % q_tiles;
  x /= q_tiles;
  const int h = x % p.H;
  const int b = x / p.H;
  const int i0 = qt * kRows;

  const int klen = sample_len(p, b);
  int visible = klen;
  if (p.causal) visible = min(visible, min(i0 + kRows, p.Lq) + p.q_offset);
  const int n = (visible + kCols - 1) / kCols;
  // A first pass over the key tiles forms delta; the steps of both passes count through.
  const int steps = 2 * n;
  auto tile = [&](int step) { return step < n ? step : step - n; };

  auto load_kv = [&](int step) {
    const int st = step % ST, t = tile(step);
    mbar_arrive_expect_tx(&full[st], 2 * C::kTile);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      tma_load_4d(sK + st * C::kTile + c * 8192, &tmK, &full[st], c * 64, h, t * kCols, b);
      tma_load_4d(sV + st * C::kTile + c * 8192, &tmV, &full[st], c * 64, h, t * kCols, b);
    }
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&ds_ready[i], 8);
    }
    mbar_init(done, 1);
    mbar_init(last, 1);
    mbar_init(delta_ready, 8);
    fence_mbar_init();
  }
  if (threadIdx.x == 0 && n > 0) {  // the first loads run under the rest of the set-up
    mbar_arrive_expect_tx(q_full, 2 * C::kBig);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      tma_load_4d(sQ + c * 16384, &tmQ, q_full, c * 64, h, i0, b);
      tma_load_4d(sO + c * 16384, &tmO, q_full, c * 64, h, i0, b);
    }
    for (int t = 0; t < min(steps, ST); ++t) load_kv(t);
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  for (int t = threadIdx.x; t < 8 * nsum; t += C::kThreads) sums[t] = 0.f;
  // this compute thread's row: its lse, loaded under the set-up too
  float lse = kInf;
  {
    const int i = i0 + (warp & 3) * 32 + lane;
    if (warp >= 2 && i < p.Lq) lse = p.lse[(static_cast<long long>(b) * p.H + h) * p.Lq + i];
    if (lse == -kInf) lse = kInf;  // no keys: every P is 0
  }
  const BiasLine bias = load_bias(p, h, stop + 2 * kRows, C::kThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_acc = tmem + NB * 2 * kCols;  // buffers of (scores, dP), then dQ

  if (warp == 0) {
    if (elect_one() && n > 0) {
      int loaded = min(steps, ST);
      for (int t = ST; t < steps; ++t) {
        if (!wait_parity(&empty[t % ST], ((t / ST) & 1) ^ 1u, kSiteAttnDq, p.ctx)) break;
        load_kv(t);
        loaded = t + 1;
      }
      wait_parity(q_full, 0, kSiteAttnDq + 1, p.ctx);
      for (int t = max(0, loaded - ST); t < loaded; ++t) wait_parity(&full[t % ST], (t / ST) & 1, kSiteAttnDq + 1, p.ctx);
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t id_s = idesc16(kRows, kCols, BF16, false);
    constexpr uint32_t id_acc = idesc16(kRows, D, BF16, true);
    auto scores = [&](int step) {
      const int st = step % ST, j0 = tile(step) * kCols;
      const bool ok = wait_parity(&full[st], (step / ST) & 1, kSiteAttnDq + 2, p.ctx);
      if (!__all_sync(0xffffffffu, ok)) return false;
      // rows past the keys that any query of the tile sees would enter dQ as 0 * anything
      if (j0 + kCols > visible) zero_tail<D, kCols>(sK + st * C::kTile, visible - j0, lane);
      tc_fence_after();
      if (elect_one()) {
        const uint32_t d = tmem + (step % NB) * 2 * kCols;
        issue_scores<D, kCols>(d, smem_u32(sQ), smem_u32(sK + st * C::kTile), id_s);
        issue_scores<D, kCols>(d + kCols, smem_u32(sO), smem_u32(sV + st * C::kTile), id_s);
        mma_commit(&s_full[step % NB]);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    if (n > 0) {
      ok = wait_parity(q_full, 0, kSiteAttnDq + 3, p.ctx);
      ok = __all_sync(0xffffffffu, ok) && scores(0);
    }
    for (int t = 0; t < steps && ok; ++t) {
      if (NB == 2 && t + 1 < steps) {
        // the buffer's previous content is still read until the product of t - 1 is done (first pass:
        // it has been read)
        if (t > n) ok = __all_sync(0xffffffffu, wait_parity(done, (t - 1 - n) & 1, kSiteAttnDq + 7, p.ctx));
        if (!ok || !scores(t + 1)) break;
      }
      ok = wait_parity(&ds_ready[t % NB], (t / NB) & 1, kSiteAttnDq + 4, p.ctx);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      const int st = t % ST;
      if (elect_one()) {
        if (t >= n)
          issue_ts<kCols>(tmem_acc, tmem + (t % NB) * 2 * kCols, smem_u32(sK + st * C::kTile), id_acc, t > n);
        mma_commit(&empty[st]);
        if (t >= n) mma_commit(done);
        if (t + 1 == steps) mma_commit(last);
      }
      __syncwarp();
      if (NB == 1 && t + 1 < steps) {
        if (t >= n) ok = __all_sync(0xffffffffu, wait_parity(done, (t - n) & 1, kSiteAttnDq + 7, p.ctx));
        ok = ok && scores(t + 1);
      }
    }
  } else {
    const int wq = warp & 3;
    const int half = (warp - 2) >> 2;
    const int r = wq * 32 + lane;
    const int i = i0 + r;
    const bool row_ok = i < p.Lq;
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    float* line = warps + (warp - 2) * C::kWarp;
    float* diag = line + 64;
    float* mine = sums + (warp - 2) * nsum;
    float left = 0.f, right = 0.f;  // this row's share of the table's gradient past the last bounds
    const int row_end = !row_ok ? 0 : (p.causal ? min(klen, i + p.q_offset + 1) : klen);
    const int warp_first = i0 + wq * 32 + p.q_offset;
    const uint64_t scale2 = f2_pack(p.scale * kLog2e, p.scale * kLog2e);
    uint64_t neg_delta = f2_pack(0.f, 0.f);
    float p_dp = 0.f;  // this row's sum of P dP over the warp's columns
    float top = 0.f;   // fp16: its largest |P dP|
    float ds_mult = 1.f, ds_back = 1.f;  // the row's factor, and 1 / it
    // The warp's tiles by kind, as in the forward kernel, for its 32 columns of each tile.
    const int t_left = (warp_first - bias.reach - 31 - half * 32 + kCols) / kCols;
    const int t_right = (warp_first + 31 + bias.ahead() - half * 32 + kCols - 1) / kCols;
    const int t_mask = ((__reduce_min_sync(0xffffffffu, row_end) - half * 32 - 32) >> 6) + 1;
    static_assert(kCols == 64, "shift above");
    const float c_left = bias.at(-bias.reach), c_right = bias.at(bias.reach);
    bool ok = true;
    for (int step = 0; step < steps; ++step) {
      const int t = tile(step);
      if (step == n) {  // the other half's columns are another warp's
        sdelta[half * kRows + r] = p_dp;
        if constexpr (!BF16) stop[half * kRows + r] = top;
        __syncwarp();
        if (lane == 0) mbar_arrive(delta_ready);
        ok = wait_parity(delta_ready, 0, kSiteAttnDq + 8, p.ctx);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        const float delta = sdelta[r] + sdelta[kRows + r];
        neg_delta = f2_pack(-delta, -delta);
        if (half == 0 && row_ok) p.delta[(static_cast<long long>(b) * p.H + h) * p.Lq + i] = delta;
        if constexpr (!BF16) {
          const unsigned bound = __float_as_uint(fmaxf(stop[r], stop[kRows + r]) + fabsf(delta));
          ds_mult = exp2_int(grad_scale(bound));
          ds_back = exp2_int(-grad_scale(bound));
          const unsigned all = __reduce_max_sync(0xffffffffu, bound);
          if (half == 0 && lane == 0)
            p.tops[((static_cast<long long>(b) * p.H + h) * q_tiles + qt) * 4 + wq] = all;
        }
      }
      const int j0 = t * kCols + half * 32;
      const int d_lo = j0 - warp_first - 31;
      const bool masked = t >= t_mask;
      const bool flat = !masked && (t < t_left || t >= t_right);
      if (!flat) {
        __syncwarp();
        line[lane] = bias.at(d_lo + lane);
        line[lane + 32] = bias.at(d_lo + lane + 32);
        __syncwarp();
      }
      const float* ln = line + 31 - lane;
      ok = wait_parity(&s_full[step % NB], (step / NB) & 1, kSiteAttnDq + 5, p.ctx);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      const uint32_t ts = tmem + lane_off + (step % NB) * 2 * kCols + half * 32;
      float s[32], g[32];
      tmem_ld32x2(ts, s, ts + kCols, g);
      if (step < n) {  // nothing is written back: the next scores may take their place
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_ready[step % NB]);
      }
      // dS in s (first pass: P dP)
      if (flat) {
        const float c = (t < t_left ? c_left : c_right) - lse;
        const uint64_t c2 = f2_pack(c, c);
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          f2_unpack(fmul2(exp2_2(ffma2(f2_pack(s[e], s[e + 1]), scale2, c2)), fadd2(f2_pack(g[e], g[e + 1]), neg_delta)),
                    s[e], s[e + 1]);
      } else {
        const uint64_t neg_lse = f2_pack(-lse, -lse);
#pragma unroll
        for (int e = 0; e < 32; e += 2)
          f2_unpack(fmul2(exp2_2(ffma2(f2_pack(s[e], s[e + 1]), scale2, fadd2(f2_pack(ln[e], ln[e + 1]), neg_lse))),
                          fadd2(f2_pack(g[e], g[e + 1]), neg_delta)),
                    s[e], s[e + 1]);
        if (masked) {
          const int keep = row_end - j0;
#pragma unroll
          for (int e = 0; e < 32; ++e) s[e] = e < keep ? s[e] : 0.f;
        }
      }
      if (step < n) {
        uint64_t a2 = f2_pack(s[0], s[1]), b2 = f2_pack(s[2], s[3]);
#pragma unroll
        for (int e = 4; e < 32; e += 4) {
          a2 = fadd2(a2, f2_pack(s[e], s[e + 1]));
          b2 = fadd2(b2, f2_pack(s[e + 2], s[e + 3]));
        }
        float x0, x1;
        f2_unpack(fadd2(a2, b2), x0, x1);
        p_dp += x0 + x1;
        if constexpr (!BF16) {
          float most[4] = {top, 0.f, 0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 32; ++e) most[e & 3] = fmaxf(most[e & 3], fabsf(s[e]));
          top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
        }
        continue;
      }
      uint32_t w[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        float x = s[2 * e], y = s[2 * e + 1];
        if constexpr (!BF16) f2_unpack(fmul2(f2_pack(x, y), f2_pack(ds_mult, ds_mult)), x, y);
        w[e] = pack16<BF16>(x, y);
      }
      tmem_st16(ts, w);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_ready[step % NB]);
      // The table's gradient: the sum of dS by diagonal (the products run meanwhile).
      if (flat) {
        uint64_t a2 = f2_pack(s[0], s[1]), b2 = f2_pack(s[2], s[3]);
#pragma unroll
        for (int e = 4; e < 32; e += 4) {
          a2 = fadd2(a2, f2_pack(s[e], s[e + 1]));
          b2 = fadd2(b2, f2_pack(s[e + 2], s[e + 3]));
        }
        float x0, x1;
        f2_unpack(fadd2(a2, b2), x0, x1);
        if (t < t_left) {
          left += x0 + x1;
        } else {
          right += x0 + x1;
        }
      } else {
        // From a column to the next a diagonal moves one lane up, so a running sum passed from lane
        // to lane follows it. Two chains of 16 columns; entry d + 31 of a chain.
        float a[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            a[c] = __shfl_up_sync(0xffffffffu, a[c], 1);
            a[c] = (lane == 0 ? 0.f : a[c]) + s[16 * c + e];
            if (lane == 31) diag[48 * c + e] = a[c];
          }
        }
        if (lane < 31) {
          diag[46 - lane] = a[0];
          diag[48 + 46 - lane] = a[1];
        }
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int idx = lane + 32 * q;
          const float v = (idx < 47 ? diag[idx] : 0.f) + (idx >= 16 && idx < 63 ? diag[48 + idx - 16] : 0.f);
          const int d = d_lo + idx;
          if (!by_diag) {
            add_buckets(mine, idx < 63 ? bias.bucket(d) : -1 - lane, v, lane);
          } else if (idx < 63) {
            if (d <= -reach) {
              left += v;
            } else if (d >= bias.ahead()) {
              right += v;
            } else {
              mine[d + reach] += v;  // one lane per diagonal
            }
          }
        }
        __syncwarp();
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      left += __shfl_xor_sync(0xffffffffu, left, o);
      right += __shfl_xor_sync(0xffffffffu, right, o);
    }
    if (lane == 0) {
      if (by_diag) {
        mine[0] += left;
        mine[reach + bias.ahead()] += right;
      } else {
        mine[bias.bucket(-reach)] += left;
        mine[bias.bucket(bias.ahead())] += right;
      }
    }
    if (ok && n > 0) {
      ok = wait_parity(last, 0, kSiteAttnDq + 6, p.ctx);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    // dQ through the query tile's shared memory: warps 2-5 write columns 0-63, 6-9 64-127.
    if (half < D / 64) {
      store_rows64<BF16>(&tmOut, sQ + half * 16384 + wq * 4096, tmem_acc + lane_off + half * 64, n > 0 && ok, false,
                         p.scale * ds_back, lane, half * 64, h, i0 + wq * 32, b, i0 + wq * 32 < p.Lq);
      if (lane == 0) bulk_wait_read<0>();
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::kTmem);
  for (int t = threadIdx.x; t < nsum; t += C::kThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w * nsum + t];
    sums[t] = s;  // (column t is this thread's)
  }
  __syncthreads();
  const int buckets = rel_num_buckets(p.rb.n_bounds, p.rb.bidirectional);
  for (int t = threadIdx.x; t < buckets; t += C::kThreads)
    p.table_part[(static_cast<long long>(h) * p.B * q_tiles + static_cast<long long>(b) * q_tiles + qt) * buckets + t] =
        by_diag ? rel_bucket_sum(sums, reach, bias.bounds, p.rb.n_bounds, t) : sums[t];
}

template <int D, bool BF16>
__global__ void __launch_bounds__(Bwd<D>::kThreads, Bwd<D>::kCtas)
    attn_dkv_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmO,
                    const __grid_constant__ CUtensorMap tmDk, const __grid_constant__ CUtensorMap tmDv,
                    const __grid_constant__ AttnArgs p) {
  using C = Bwd<D>;
  constexpr int ST = C::kStages;
  constexpr int NB = C::kBuf;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem =
      reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + C::kBig;
  uint8_t* sQ = sV + C::kBig;
  uint8_t* sO = sQ + ST * C::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sO + ST * C::kTile);
  uint64_t* full = bars;
  uint64_t* empty = bars + ST;
  uint64_t* k_full = bars + 2 * ST;
  uint64_t* s_full = k_full + 1;
  uint64_t* ds_ready = s_full + 2;  // NB
  uint64_t* done = ds_ready + 2;
  uint64_t* last = done + 1;  // every product is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(last + 1);
  float* warps = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 256);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k_tiles = (p.Lk + kRows - 1) / kRows;
  int x = blockIdx.x;
  const int kt = x % k_tiles;
  x /= k_tiles;
  const int h = x % p.H;
  const int b = x / p.H;
  const int j0 = kt * kRows;
  // query tiles with a row that sees one of these keys
  const int q_tiles = (p.Lq + kCols - 1) / kCols;
  const int first = p.causal ? max(0, j0 - p.q_offset) / kCols : 0;
  unsigned top = 0;
  if constexpr (!BF16) {  // (not looked at where the sample has no keys, and the bounds no values)
    const int n_tops = (p.Lq + kRows - 1) / kRows * 4;
    const unsigned* src = p.tops + (static_cast<long long>(b) * p.H + h) * n_tops;
    for (int t = threadIdx.x; t < n_tops; t += C::kThreads) top = max(top, src[t]);
  }

  auto load_q = [&](int t) {
    const int st = t % ST;
    mbar_arrive_expect_tx(&full[st], 2 * C::kTile);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      tma_load_4d(sQ + st * C::kTile + c * 8192, &tmQ, &full[st], c * 64, h, (first + t) * kCols, b);
      tma_load_4d(sO + st * C::kTile + c * 8192, &tmO, &full[st], c * 64, h, (first + t) * kCols, b);
    }
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(k_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&ds_ready[i], 8);
    }
    mbar_init(done, 1);
    mbar_init(last, 1);
    fence_mbar_init();
  }
  const int klen = sample_len(p, b);
  const int n = j0 < klen ? max(0, q_tiles - first) : 0;
  if (threadIdx.x == 0 && n > 0) {  // the first loads run under the rest of the set-up
    mbar_arrive_expect_tx(k_full, 2 * C::kBig);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      tma_load_4d(sK + c * 16384, &tmK, k_full, c * 64, h, j0, b);
      tma_load_4d(sV + c * 16384, &tmV, k_full, c * 64, h, j0, b);
    }
    for (int t = 0; t < min(n, ST); ++t) load_q(t);
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  unsigned* tops = reinterpret_cast<unsigned*>(warps + 8 * C::kWarp);  // fp16: a bound of |dS| per warp
  if constexpr (!BF16) {
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
  }
  const BiasLine bias = load_bias(p, h, tops + 16, C::kThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_dv = tmem + NB * 2 * kCols;
  const uint32_t tmem_dk = tmem_dv + D;

  if (warp == 0) {
    if (elect_one() && n > 0) {
      int loaded = min(n, ST);
      for (int t = ST; t < n; ++t) {
        if (!wait_parity(&empty[t % ST], ((t / ST) & 1) ^ 1u, kSiteAttnDkv, p.ctx)) break;
        load_q(t);
        loaded = t + 1;
      }
      wait_parity(k_full, 0, kSiteAttnDkv + 1, p.ctx);
      for (int t = max(0, loaded - ST); t < loaded; ++t) wait_parity(&full[t % ST], (t / ST) & 1, kSiteAttnDkv + 1, p.ctx);
    }
    __syncwarp();
  } else if (warp == 1) {
    constexpr uint32_t id_s = idesc16(kRows, kCols, BF16, false);
    constexpr uint32_t id_acc = idesc16(kRows, D, BF16, true);
    auto scores = [&](int t) {
      const int st = t % ST;
      const bool ok = wait_parity(&full[st], (t / ST) & 1, kSiteAttnDkv + 2, p.ctx);
      if (!__all_sync(0xffffffffu, ok)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t d = tmem + (t % NB) * 2 * kCols;
        issue_scores<D, kCols>(d, smem_u32(sK), smem_u32(sQ + st * C::kTile), id_s);
        issue_scores<D, kCols>(d + kCols, smem_u32(sV), smem_u32(sO + st * C::kTile), id_s);
        mma_commit(&s_full[t % NB]);
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    if (n > 0) {
      ok = wait_parity(k_full, 0, kSiteAttnDkv + 3, p.ctx);
      ok = __all_sync(0xffffffffu, ok) && scores(0);
    }
    for (int t = 0; t < n && ok; ++t) {
      if (NB == 2 && t + 1 < n) {
        // the buffer's previous content is still read until the products of t - 1 are done
        if (t > 0) ok = __all_sync(0xffffffffu, wait_parity(done, (t - 1) & 1, kSiteAttnDkv + 7, p.ctx));
        if (!ok || !scores(t + 1)) break;
      }
      ok = wait_parity(&ds_ready[t % NB], (t / NB) & 1, kSiteAttnDkv + 4, p.ctx);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      const int st = t % ST;
      if (elect_one()) {
        const uint32_t d = tmem + (t % NB) * 2 * kCols;
        issue_ts<kCols>(tmem_dv, d, smem_u32(sO + st * C::kTile), id_acc, t > 0);
        issue_ts<kCols>(tmem_dk, d + kCols, smem_u32(sQ + st * C::kTile), id_acc, t > 0);
        mma_commit(&empty[st]);
        mma_commit(done);
        if (t + 1 == n) mma_commit(last);
      }
      __syncwarp();
      if (NB == 1 && t + 1 < n)
        ok = __all_sync(0xffffffffu, wait_parity(done, t & 1, kSiteAttnDkv + 7, p.ctx)) && scores(t + 1);
    }
  } else {
    const int wq = warp & 3;
    const int half = (warp - 2) >> 2;
    const int jw = j0 + wq * 32;  // the warp's first key
    const int j = jw + lane;      // this thread's key
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    float* line = warps + (warp - 2) * C::kWarp;
    float* rowv = line + 160;  // -lse and -delta of the half tile's 32 query rows
    const uint64_t scale2 = f2_pack(p.scale * kLog2e, p.scale * kLog2e);
    const bool key_ok = j < klen;
    const unsigned head = static_cast<unsigned>(b) * p.H + h;
    // Row values of tile t for this lane: loaded a tile ahead, looked at when their tile begins.
    // -inf: no such row, or one without keys; every P is 0.
    float next_lse = -kInf, next_delta = 0.f;
    auto load_rows = [&](int t) {
      const int i = (first + t) * kCols + half * 32 + lane;
      next_lse = -kInf;
      if (t < n && i < p.Lq) {
        next_lse = p.lse[static_cast<long long>(head) * p.Lq + i];
        next_delta = p.delta[static_cast<long long>(head) * p.Lq + i];
      }
    };
    load_rows(0);
    // Tile kinds: positions pos .. pos + 31 of the half tile's rows, pos = pos0 + t * kCols. Keys
    // jw .. jw + 31 lie past the last bound on the left from t_left on, on the right before t_right.
    const int pos0 = first * kCols + half * 32 + p.q_offset;
    const int t_left = (jw + 31 + bias.reach - pos0 + kCols - 1) / kCols;
    const int t_right = (jw - 31 - bias.ahead() - pos0 + kCols) / kCols;
    // masked: rows past Lq, keys past klen, or (causal) a row before one of the keys
    const int t_causal = p.causal ? (jw + 31 - pos0 + kCols - 1) / kCols : 0;
    const bool all_keys = jw + 32 <= klen;
    if (lane == 0) {  // (in shared memory: registers are short)
      line[64] = bias.at(-bias.reach);
      line[65] = bias.at(bias.reach);
    }
    auto ds_scale = [&] {  // fp16: log2 of dS's factor
      return grad_scale(__reduce_max_sync(0xffffffffu, lane < C::kThreads / 32 ? tops[lane] : 0u));
    };
    const float ds_mult = BF16 ? 1.f : exp2_int(ds_scale() - kPScale);  // (P carries the rest)
    bool ok = true;
    for (int t = 0; t < n; ++t) {
      const int pos = pos0 + t * kCols;
      const int i_half = pos - p.q_offset;
      const bool masked = !all_keys || t < t_causal || i_half + 32 > p.Lq;
      const bool flat = !masked && (t >= t_left || t < t_right);
      __syncwarp();
      rowv[lane] = next_lse == -kInf ? -kInf : BF16 ? -next_lse : kPScale - next_lse;
      rowv[32 + lane] = BF16 ? -next_delta : -next_delta * ds_mult;
      if (!flat) {
        // diagonal of (key lane, query e): d_lo + 31 + lane - e
        const int d_lo = jw - pos - 31;
        line[lane] = bias.at(d_lo + lane);
        line[lane + 32] = bias.at(d_lo + lane + 32);
      }
      __syncwarp();
      load_rows(t + 1);
      ok = wait_parity(&s_full[t % NB], (t / NB) & 1, kSiteAttnDkv + 5, p.ctx);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      const uint32_t ts = tmem + lane_off + (t % NB) * 2 * kCols + half * 32;
      float s[32], g[32];
      tmem_ld32x2(ts, s, ts + kCols, g);
      uint32_t wp[16], wd[16];
      auto transform = [&](auto is_flat, auto is_masked) {
        const float c = line[t >= t_left ? 64 : 65];
        const uint64_t c2 = f2_pack(c, c);
        const float* ln = line + 31 + lane;
        const int from = !key_ok ? 32 : (p.causal ? j - pos : 0), to = p.Lq - i_half;
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          const float4 l4 = *reinterpret_cast<const float4*>(rowv + e);
          const float4 d4 = *reinterpret_cast<const float4*>(rowv + 32 + e);
          const uint64_t nl[2] = {f2_pack(l4.x, l4.y), f2_pack(l4.z, l4.w)};
          const uint64_t nd[2] = {f2_pack(d4.x, d4.y), f2_pack(d4.z, d4.w)};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int q = e + 2 * u;
            uint64_t add;
            if constexpr (decltype(is_flat)::value) {
              add = fadd2(c2, nl[u]);
            } else {
              add = fadd2(f2_pack(ln[-q], ln[-q - 1]), nl[u]);
            }
            uint64_t pr = exp2_2(ffma2(f2_pack(s[q], s[q + 1]), scale2, add));
            const uint64_t g2 = f2_pack(g[q], g[q + 1]);
            uint64_t ds = fmul2(pr, BF16 ? fadd2(g2, nd[u]) : ffma2(g2, f2_pack(ds_mult, ds_mult), nd[u]));
            float p0, p1, d0, d1;
            f2_unpack(pr, p0, p1);
            f2_unpack(ds, d0, d1);
            if constexpr (decltype(is_masked)::value) {
              const bool a = q >= from && q < to, bb = q + 1 >= from && q + 1 < to;
              p0 = a ? p0 : 0.f;
              d0 = a ? d0 : 0.f;
              p1 = bb ? p1 : 0.f;
              d1 = bb ? d1 : 0.f;
            }
            wp[q >> 1] = pack16<BF16>(p0, p1);
            wd[q >> 1] = pack16<BF16>(d0, d1);
          }
        }
      };
      if (masked) {
        transform(std::false_type{}, std::true_type{});
      } else if (flat) {
        transform(std::true_type{}, std::false_type{});
      } else {
        transform(std::false_type{}, std::false_type{});
      }
      tmem_st16(ts, wp);
      tmem_st16(ts + kCols, wd);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_ready[t % NB]);
    }
    if (ok && n > 0) {
      ok = wait_parity(last, 0, kSiteAttnDkv + 6, p.ctx);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    // Warps 2-5 write dV, warps 6-9 dK (through the tiles' shared memory); keys past the sample's
    // length get 0.
    const float mult =
        half == 0 ? (BF16 ? 1.f : exp2_int(-kPScale)) : (BF16 ? p.scale : p.scale * exp2_int(-ds_scale()));
#pragma unroll 1
    for (int c = 0; c < D / 64; ++c)
      store_rows64<BF16>(half == 0 ? &tmDv : &tmDk, (half == 0 ? sV : sK) + c * 16384 + wq * 4096,
                         (half == 0 ? tmem_dv : tmem_dk) + lane_off + c * 64, n > 0 && ok, !key_ok,
                         mult, lane, c * 64, h, jw, b, jw < p.Lk);
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, C::kTmem);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int cuda_rc(cudaError_t e) {
  if (e == cudaSuccess) return WDIT_OK;
  cudaGetLastError();  // reported here, not by the next launch too
  return WDIT_ERR_CUDA_BASE + static_cast<int>(e);
}

// Key splits of the forward: with fewer CTAs than two per SM (a few query rows of a few heads)
// one CTA would walk a long cache alone, so the keys are divided until the SMs are full, at least
// four tiles a part (one query row, bf16, us with at least 1 / 4 / 16 tiles a part and undivided: 12
// heads x 8191 keys x 128 17.3 / 17.2 / 21.2 / 97, 12 x 1000 x 64 11.0 / 11.9 / 18.2 / 18.1, 8 x 12 x
// 8191 x 128 66 / 66 / 66 / 115, with lengths from 8191 down to 3291 57.6 / 57.6 / 57.6 / 113).
int attn_splits(int B, int H, int Lq, int Lk) {
  const long long ctas = static_cast<long long>(B) * H * ((Lq + kRows - 1) / kRows);
  const int tiles = (Lk + kCols - 1) / kCols;
  if (ctas <= 0) return 1;
  long long s = 2ll * sm_count() / ctas;
  if (s > tiles / 4) s = tiles / 4;
  return s < 1 ? 1 : (s > kMaxSplits ? kMaxSplits : static_cast<int>(s));
}

// Which forward of D = 64: four CTAs per SM with one score buffer each, or two with two. Four win
// where the CTAs outnumber two per SM and a CTA's start and end weigh (us, two / four per SM, 64
// heads bidirectional: 2 x 512 x 512 29.7 / 27.0, 8 x 512 x 512 97 / 86; causal 8 x 512 x 512 81.6 /
// 64.8; 80 x 12 heads x 77 x 77 29.9 / 23.0; 148 heads x 512 x 2048 72.6 / 70.6). Two win where
// there are no more CTAs than that (74 heads x 512 x 512 16.2 / 19.6) and on long keys, whose one
// CTA then walks twice as fast (12 heads x 8192 x 8192 337 / 355, causal 4096 x 4096 61 / 81).
bool four_per_sm(const AttnArgs& p) {
  const long long ctas = static_cast<long long>(p.B) * p.H * ((p.Lq + kRows - 1) / kRows);
  return ctas > 2ll * sm_count() && p.Lk <= 2048;
}

struct Strides {
  long long b, l, h;
};

// [B, L, H, D] with element strides, unit along D; box of 64 columns x rows of one head
int map_heads(CUtensorMap* m, bool bf16, const void* ptr, int B, int L, int H, int D, Strides s, int rows) {
  const unsigned long long dims[4] = {static_cast<unsigned long long>(D), static_cast<unsigned long long>(H),
                                      static_cast<unsigned long long>(L), static_cast<unsigned long long>(B)};
  const unsigned long long st[3] = {static_cast<unsigned long long>(s.h) * 2, static_cast<unsigned long long>(s.l) * 2,
                                    static_cast<unsigned long long>(s.b) * 2};
  const unsigned int box[4] = {64, 1, static_cast<unsigned>(rows), 1};
  return encode_tiled(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, ptr, dims, st,
                      box, CU_TENSOR_MAP_SWIZZLE_128B);
}

int check_attn(const int* bounds, int n_bounds, int B, int H, int Lq, int Lk, int D, int dtype, int table_dtype,
               int q_offset, const void* table) {
  if (bounds == nullptr || table == nullptr) return WDIT_ERR_ARG;
  if (dtype != 1 && dtype != 2) return WDIT_ERR_ARG;
  if (table_dtype < 0 || table_dtype > 2) return WDIT_ERR_ARG;
  if (n_bounds < 1 || n_bounds > kMaxRelBounds) return WDIT_ERR_SHAPE;
  if (B < 0 || H < 1 || H > 65535 || Lq < 0 || Lk < 0 || (D != 64 && D != 128)) return WDIT_ERR_SHAPE;
  if (q_offset < 0 || static_cast<long long>(q_offset) + Lq > (1ll << 30) || Lq > (1 << 28) || Lk > (1 << 28))
    return WDIT_ERR_SHAPE;
  return WDIT_OK;
}

int check_heads(const void* p, const long long* s) {
  if (p == nullptr || s == nullptr) return WDIT_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(p) & 15) != 0) return WDIT_ERR_ALIGN;
  for (int i = 0; i < 3; ++i) {
    if (s[i] <= 0) return WDIT_ERR_SHAPE;
    if (s[i] % 8 != 0) return WDIT_ERR_ALIGN;
  }
  return WDIT_OK;
}

// The kernels' limit is raised once to what any table needs (always the same value, so that calls at
// the same time do no harm).
constexpr int kSmemMost = 176 * 1024;

template <typename K>
int set_smem(K kernel, int bytes, bool (&done)[64]) {
  if (bytes > kSmemMost) return WDIT_ERR_SHAPE;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_rc(e);
  if (!done[dev & 63]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMost);
    if (e != cudaSuccess) return cuda_rc(e);
    done[dev & 63] = true;
  }
  return WDIT_OK;
}

template <int D, bool BF16, int NB>
int run_fwd(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& o,
            const AttnArgs& p, cudaStream_t st) {
  static bool done[64] = {};
  const int smem = Fwd<D, NB>::smem(p.rb);
  int rc = set_smem(attn_fwd_kernel<D, BF16, NB>, smem, done);
  if (rc) return rc;
  const long long grid = static_cast<long long>((p.Lq + kRows - 1) / kRows) * p.splits * p.H * p.B;
  if (grid > 0x7fffffffll) return WDIT_ERR_SHAPE;
  attn_fwd_kernel<D, BF16, NB><<<static_cast<unsigned>(grid), Fwd<D, NB>::kThreads, smem, st>>>(q, k, v, o, p);
  rc = cuda_rc(cudaGetLastError());
  if (rc || p.splits == 1) return rc;
  const long long rows = static_cast<long long>(p.B) * p.H * p.Lq;
  attn_combine_kernel<D, BF16><<<static_cast<unsigned>((rows + 7) / 8), 256, 0, st>>>(p);
  return cuda_rc(cudaGetLastError());
}

template <int D, bool BF16>
int run_bwd(const CUtensorMap (&big)[4], const CUtensorMap (&small)[4], const CUtensorMap (&out)[3], const AttnArgs& p,
            int buckets, void* dtable, int dtable_dtype, cudaStream_t st) {
  // order of the maps: q, k, v, dO; dq, dk, dv
  static bool done_q[64] = {}, done_kv[64] = {};
  const int smem = Bwd<D>::smem(p.rb);
  int rc = set_smem(attn_dq_kernel<D, BF16>, smem, done_q);
  if (rc) return rc;
  if ((rc = set_smem(attn_dkv_kernel<D, BF16>, smem, done_kv))) return rc;
  const int q_tiles = (p.Lq + kRows - 1) / kRows;
  const long long gq = static_cast<long long>(q_tiles) * p.H * p.B;
  const long long gk = static_cast<long long>((p.Lk + kRows - 1) / kRows) * p.H * p.B;
  if (gq > 0x7fffffffll || gk > 0x7fffffffll) return WDIT_ERR_SHAPE;
  attn_dq_kernel<D, BF16><<<static_cast<unsigned>(gq), Bwd<D>::kThreads, smem, st>>>(big[0], small[1], small[2],
                                                                                    big[3], out[0], p);
  if ((rc = cuda_rc(cudaGetLastError()))) return rc;
  attn_dkv_kernel<D, BF16><<<static_cast<unsigned>(gk), Bwd<D>::kThreads, smem, st>>>(big[1], big[2], small[0],
                                                                                     small[3], out[1], out[2], p);
  if ((rc = cuda_rc(cudaGetLastError()))) return rc;
  return launch_rel_table_sum(p.table_part, p.B * q_tiles, buckets, p.H, dtable, dtable_dtype, st);
}

long long align16(long long x) { return (x + 15) / 16 * 16; }

}  // namespace
}  // namespace wdit

using namespace wdit;

extern "C" {

long long wdit_rel_attention_workspace_bytes(int B, int H, int Lq, int Lk, int D) {
  if (B <= 0 || H <= 0 || Lq <= 0 || Lk <= 0 || D <= 0) return 0;
  const int s = attn_splits(B, H, Lq, Lk);
  return s == 1 ? 0 : 4ll * s * B * H * Lq * (D + 1);
}

int wdit_rel_attention(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
                       const void* v, const long long* v_strides, int B, int H, int Lq, int Lk, int D, int dtype,
                       const int* k_lens, const void* table, int table_dtype, const int* bounds, int n_bounds,
                       int bidirectional, int causal, int q_offset, float scale, void* out, float* lse,
                       void* workspace, long long workspace_bytes, void* stream) {
  int rc = check_attn(bounds, n_bounds, B, H, Lq, Lk, D, dtype, table_dtype, q_offset, table);
  if (rc) return rc;
  if (B == 0 || Lq == 0) return WDIT_OK;
  if (out == nullptr) return WDIT_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(out) & 15) != 0) return WDIT_ERR_ALIGN;
  if (Lk == 0) return WDIT_ERR_SHAPE;  // the caller knows the answer: zeros
  if ((rc = check_heads(q, q_strides)) || (rc = check_heads(k, k_strides)) || (rc = check_heads(v, v_strides)))
    return rc;
  AttnArgs p = {};
  p.B = B;
  p.H = H;
  p.Lq = Lq;
  p.Lk = Lk;
  p.causal = causal != 0;
  p.q_offset = q_offset;
  p.scale = scale;
  p.k_lens = k_lens;
  p.table = table;
  p.table_dtype = table_dtype;
  if (!rel_fill(&p.rb, bounds, n_bounds, bidirectional)) return WDIT_ERR_ARG;
  p.out = out;
  p.lse = lse;
  p.splits = attn_splits(B, H, Lq, Lk);
  if (p.splits > 1) {
    if (workspace == nullptr || workspace_bytes < wdit_rel_attention_workspace_bytes(B, H, Lq, Lk, D))
      return WDIT_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return WDIT_ERR_ALIGN;
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + static_cast<long long>(p.splits) * B * H * Lq * D;
  }
  if ((rc = error_record_ptr(&p.ctx.rec))) return rc;
  p.ctx.limit_ns = wait_limit_ns();
  const bool bf16 = dtype == 1;
  CUtensorMap mq, mk, mv, mo;
  if ((rc = map_heads(&mq, bf16, q, B, Lq, H, D, {q_strides[0], q_strides[1], q_strides[2]}, kRows)) ||
      (rc = map_heads(&mk, bf16, k, B, Lk, H, D, {k_strides[0], k_strides[1], k_strides[2]}, kCols)) ||
      (rc = map_heads(&mv, bf16, v, B, Lk, H, D, {v_strides[0], v_strides[1], v_strides[2]}, kCols)) ||
      (rc = map_heads(&mo, bf16, out, B, Lq, H, D, {1ll * Lq * H * D, 1ll * H * D, D}, 32)))
    return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto run) { return run(mq, mk, mv, mo, p, st); };
  if (D == 128) return bf16 ? go(run_fwd<128, true, 2>) : go(run_fwd<128, false, 2>);
  if (four_per_sm(p)) return bf16 ? go(run_fwd<64, true, 1>) : go(run_fwd<64, false, 1>);
  return bf16 ? go(run_fwd<64, true, 2>) : go(run_fwd<64, false, 2>);
}

long long wdit_rel_attention_backward_workspace_bytes(int B, int H, int Lq, int n_bounds, int bidirectional) {
  if (B <= 0 || H <= 0 || Lq <= 0 || n_bounds < 1) return 0;
  const long long q_tiles = (Lq + kRows - 1) / kRows;
  return align16(4ll * B * H * Lq) + 16ll * H * B * q_tiles +
         4ll * H * B * q_tiles * rel_num_buckets(n_bounds, bidirectional);
}

int wdit_rel_attention_backward(const void* q, const long long* q_strides, const void* k, const long long* k_strides,
                                const void* v, const long long* v_strides, const void* dout,
                                const long long* dout_strides, const float* lse, int B, int H, int Lq, int Lk, int D,
                                int dtype, const int* k_lens, const void* table, int table_dtype, const int* bounds,
                                int n_bounds, int bidirectional, int causal, int q_offset, float scale, void* dq,
                                void* dk, void* dv, void* dtable, int dtable_dtype, void* workspace,
                                long long workspace_bytes, void* stream) {
  int rc = check_attn(bounds, n_bounds, B, H, Lq, Lk, D, dtype, table_dtype, q_offset, table);
  if (rc) return rc;
  if (B == 0 || Lq == 0 || Lk == 0) return WDIT_ERR_SHAPE;  // the caller knows the answer: zeros
  if (lse == nullptr || dq == nullptr || dk == nullptr || dv == nullptr || dtable == nullptr || dtable_dtype < 0 ||
      dtable_dtype > 2)
    return WDIT_ERR_ARG;
  for (const void* t : {dq, dk, dv})
    if ((reinterpret_cast<uintptr_t>(t) & 15) != 0) return WDIT_ERR_ALIGN;
  if ((rc = check_heads(q, q_strides)) || (rc = check_heads(k, k_strides)) || (rc = check_heads(v, v_strides)) ||
      (rc = check_heads(dout, dout_strides)))
    return rc;
  if (workspace == nullptr ||
      workspace_bytes < wdit_rel_attention_backward_workspace_bytes(B, H, Lq, n_bounds, bidirectional))
    return WDIT_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return WDIT_ERR_ALIGN;
  AttnArgs p = {};
  p.B = B;
  p.H = H;
  p.Lq = Lq;
  p.Lk = Lk;
  p.causal = causal != 0;
  p.q_offset = q_offset;
  p.scale = scale;
  p.k_lens = k_lens;
  p.table = table;
  p.table_dtype = table_dtype;
  if (!rel_fill(&p.rb, bounds, n_bounds, bidirectional)) return WDIT_ERR_ARG;
  p.lse = const_cast<float*>(lse);
  p.splits = 1;
  p.delta = static_cast<float*>(workspace);
  p.tops = reinterpret_cast<unsigned*>(static_cast<char*>(workspace) + align16(4ll * B * H * Lq));
  p.table_part = reinterpret_cast<float*>(p.tops + 4ll * B * H * ((Lq + kRows - 1) / kRows));
  if ((rc = error_record_ptr(&p.ctx.rec))) return rc;
  p.ctx.limit_ns = wait_limit_ns();
  const bool bf16 = dtype == 1;
  CUtensorMap big[4], small[4], outs[3];
  const void* ptrs[4] = {q, k, v, dout};
  const long long* strides[4] = {q_strides, k_strides, v_strides, dout_strides};
  for (int i = 0; i < 4; ++i) {
    const int L = i == 1 || i == 2 ? Lk : Lq;
    const Strides s = {strides[i][0], strides[i][1], strides[i][2]};
    if ((rc = map_heads(&big[i], bf16, ptrs[i], B, L, H, D, s, kRows)) ||
        (rc = map_heads(&small[i], bf16, ptrs[i], B, L, H, D, s, kCols)))
      return rc;
  }
  void* const grads[3] = {dq, dk, dv};
  for (int i = 0; i < 3; ++i) {
    const int L = i == 0 ? Lq : Lk;
    if ((rc = map_heads(&outs[i], bf16, grads[i], B, L, H, D, {1ll * L * H * D, 1ll * H * D, D}, 32))) return rc;
  }
  const int buckets = rel_num_buckets(n_bounds, p.rb.bidirectional);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (D == 64)
    return bf16 ? run_bwd<64, true>(big, small, outs, p, buckets, dtable, dtable_dtype, st)
                : run_bwd<64, false>(big, small, outs, p, buckets, dtable, dtable_dtype, st);
  return bf16 ? run_bwd<128, true>(big, small, outs, p, buckets, dtable, dtable_dtype, st)
              : run_bwd<128, false>(big, small, outs, p, buckets, dtable, dtable_dtype, st);
}

}  // extern "C"
