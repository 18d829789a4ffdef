// Learned relative position bias by buckets: the bias tensor and the gradient of its table.
//
//   out[h, i, j]   = table[bucket(j - (i + q_offset)), h]
//   dtable[b, h]   = sum over batch, i, j with bucket(j - (i + q_offset)) = b of dbias[., h, i, j]
//
// Both depend on a cell through its diagonal d = j - i only, and both are bound by HBM: the
// forward writes every cell once, the gradient reads every cell once.
//
// Forward (rel_bias_kernel). A CTA takes a tile of rows x columns of one head, looks the bucket of
// each of the tile's rows + columns - 1 diagonals up once, keeps the table's values for them in
// shared memory, and writes every row as a shifted window of that line with 16-byte stores. The
// line is kept as 32-bit words (16-bit types: one copy per element parity) with a word of padding
// every 32, so that lanes four words apart read different banks. 64 heads x 512 x 512 bf16: 8.1 us,
// 4.1 TB/s (launch, look-up and the first stores take half of it); 12 heads x 1 x 4097 fp32 4.7 us.
//
// Gradient (rel_bias_grad_kernel). A warp takes some rows of a strip of columns, and a lane's
// accumulators are diagonals, never looked up per cell:
//   rows on 16-byte boundaries: a rectangle of 256 columns, 8 per lane, 8 rows at a time. Row u adds
//     its column e to the lane's sum e - u; after 8 rows the sums move 8 columns on, to the next
//     lane (one shuffle per row of the block), and those of the last lane leave the strip.
//   other rows: a parallelogram of 256 diagonals; the columns read move one on per row, so each
//     lane stays on its 8 diagonals. The rows come by 16-byte asynchronous copies of the aligned
//     blocks that hold them, eight rows ahead, and are read from shared memory at any offset.
// The diagonal sums then go to the warp's sums per diagonal, which reach from the last bound on
// one side to the other; what lies past them goes into one sum per side. Buckets are formed once
// per CTA. (A table whose last bound is above 512 has no room for that; its strips are added bucket
// by bucket.) Sums are fp32, the order is fixed (no atomics), and a second small kernel adds the
// CTAs' partial buckets (2 us). Aligned: 40 heads x 2048 x 2048 fp32 100 us, 6.7 TB/s; 2 x 64 heads
// x 512 x 512 bf16 14 us, 4.7 TB/s (by the other form 148 and 38). Unaligned: 40 heads x 2047 x 2049
// fp32 120 us, 5.6 TB/s: a seventh of its cells lie in strips that leave the row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "relpos.cuh"
#include "wdit_internal.h"

namespace wdit {
namespace {

constexpr int kRelThreads = 256;
constexpr int kRelWarps = kRelThreads / 32;
constexpr int kBiasRows = 32;    // rows of a forward tile
constexpr int kBiasCols = 2048;  // columns of a forward tile
constexpr int kGradRowsMin = 32;  // rows of a gradient strip: 32, 64 or 128
constexpr int kGradRowsMax = 128;
constexpr int kGradCols = 256;   // columns of a gradient strip (8 per lane)
constexpr int kGradReach = 512;  // sums per diagonal are kept up to this last bound

constexpr int kRing = 8;  // rows of a parallelogram strip in flight per warp

// Shared memory of the gradient kernel: sums and bounds, then (unaligned rows) the warps' rings of
// 256 columns and one more 16-byte block a row.
__host__ __device__ constexpr int grad_fixed_bytes(int sums) {
  return (kRelWarps * sums * 4 + kMaxRelBounds * 4 + 15) / 16 * 16;
}
__host__ __device__ constexpr int grad_row_bytes(int esize) { return kGradCols * esize + 16; }

// Strips of a gradient chunk of `rows` rows: 256 columns each, or 256 of its Lk + rows - 1 diagonals.
__host__ __device__ inline int grad_strips(int Lk, int rows, bool vec) {
  return ((vec ? Lk : Lk + rows - 1) + kGradCols - 1) / kGradCols;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
  return __half2float(v);
}

template <typename T>
__global__ void __launch_bounds__(kRelThreads)
    rel_bias_kernel(const T* __restrict__ table, const __grid_constant__ RelBuckets rb, int H, int Lq, int Lk,
                    int q_offset, int rows, T* __restrict__ out) {
  constexpr int E = 4 / static_cast<int>(sizeof(T));  // elements of a word
  constexpr int V = 4 * E;                            // elements of a 16-byte store
  constexpr int kWords = (kBiasCols + kBiasRows) / E + 16;
  __shared__ uint32_t line[E][kWords + kWords / 32 + 1];
  __shared__ int bounds[kMaxRelBounds];
  auto slot = [](int w) { return w + (w >> 5); };
  const int col_tiles = (Lk + kBiasCols - 1) / kBiasCols;
  const int row_tile = static_cast<int>(blockIdx.x) / col_tiles;
  const int h = blockIdx.y;
  const int i0 = row_tile * rows;
  const int i1 = min(i0 + rows, Lq);
  const int j0 = (static_cast<int>(blockIdx.x) - row_tile * col_tiles) * kBiasCols;
  const int j1 = min(j0 + kBiasCols, Lk);
  for (int t = threadIdx.x; t < rb.n_bounds; t += kRelThreads) bounds[t] = rb.bounds[t];
  __syncthreads();
  const int d0 = j0 - (i1 - 1) - q_offset;  // the tile's first diagonal
  const int nd = (j1 - j0) + (i1 - i0) - 1;
  for (int t = threadIdx.x; t < nd; t += kRelThreads) {
    const T v = table[static_cast<size_t>(rel_bucket(bounds, rb.n_bounds, rb.bidirectional, d0 + t)) * H + h];
    if constexpr (E == 1) {
      line[0][slot(t)] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      reinterpret_cast<T*>(&line[0][slot(t >> 1)])[t & 1] = v;
      if (t > 0) reinterpret_cast<T*>(&line[E - 1][slot((t - 1) >> 1)])[(t - 1) & 1] = v;
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // few rows: the warps share a row's pieces instead of taking rows
  const int by_row = i1 - i0 >= kRelWarps ? 1 : 0;
  const int w0 = by_row ? 0 : warp, wstep = by_row ? 1 : kRelWarps;
  for (int i = i0 + (by_row ? warp : 0); i < i1; i += by_row ? kRelWarps : 1) {
    T* row = out + (static_cast<size_t>(h) * Lq + i) * Lk;
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row + j0) & 15) / sizeof(T));
    const int shift = i1 - 1 - i - j0;  // column j of this row is diagonal j + shift of the line
    for (int j = j0 - mis + (w0 * 32 + lane) * V; j < j1; j += wstep * 32 * V) {  // 16-byte aligned
      const int s = j + shift;
      if (j >= j0 && j + V <= j1) {
        const uint32_t* src = line[E == 2 ? s & 1 : 0];
        const int w = E == 2 ? s >> 1 : s;
        *reinterpret_cast<uint4*>(row + j) =
            make_uint4(src[slot(w)], src[slot(w + 1)], src[slot(w + 2)], src[slot(w + 3)]);
      } else {
        for (int q = 0; q < V; ++q)
          if (j + q >= j0 && j + q < j1) {
            const int e = s + q;
            if constexpr (E == 1)
              row[j + q] = *reinterpret_cast<const T*>(&line[0][slot(e)]);
            else
              row[j + q] = reinterpret_cast<const T*>(&line[0][slot(e >> 1)])[e & 1];
          }
      }
    }
  }
}

// Eight neighbouring elements as fp32 from loaded words.
template <typename T>
__device__ __forceinline__ void widen8(const uint32_t* w, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(w[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = to_f32<T>(reinterpret_cast<const T*>(w)[e]);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kRelThreads, VEC ? 2 : 3)
    rel_bias_grad_kernel(const T* __restrict__ db, const __grid_constant__ RelBuckets rb, int B, int Lq, int Lk,
                         int q_offset, long long stride_b, long long stride_h, long long stride_i, int buckets,
                         int rows, float* __restrict__ part) {
  extern __shared__ float sm[];
  // per warp: sums of the diagonals -reach .. reach (the ends hold all beyond), or of the buckets
  const int reach = rb.bounds[rb.n_bounds - 1];
  const bool by_diag = reach <= kGradReach;
  const int ahead = rb.bidirectional ? reach : 0;  // from here on one bucket
  const int sums = by_diag ? reach + ahead + 1 : buckets;
  float* acc_b = sm;  // [warps][sums]
  int* bounds = reinterpret_cast<int*>(sm + kRelWarps * sums);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kRowBytes = grad_row_bytes(sizeof(T));
  uint8_t* const rows_smem =
      reinterpret_cast<uint8_t*>(sm) + grad_fixed_bytes(sums) + (VEC ? 0 : warp * kRing * kRowBytes);
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(rows_smem));
  const int h = blockIdx.y;
  for (int t = threadIdx.x; t < rb.n_bounds; t += kRelThreads) bounds[t] = rb.bounds[t];
  for (int t = threadIdx.x; t < kRelWarps * sums; t += kRelThreads) acc_b[t] = 0.f;
  __syncthreads();
  float* mine = acc_b + warp * sums;
  float left = 0.f, right = 0.f;  // this lane's share of the cells past the ends
  // One value per lane, of 32 different diagonals.
  auto add_diag = [&](int d, float val) {
    if (by_diag) {
      if (d <= -reach) {
        left += val;
      } else if (d >= ahead) {
        right += val;
      } else {
        mine[d + reach] += val;
      }
      __syncwarp();
    } else {
      add_buckets(mine, rel_bucket(bounds, rb.n_bounds, rb.bidirectional, d), val, lane);
    }
  };
  const int chunks = (Lq + rows - 1) / rows;
  const int strips = grad_strips(Lk, rows, VEC);
  // (2^31 strips would be more cells than any memory holds: the entry point refuses them)
  const unsigned items = static_cast<unsigned>(B) * chunks * strips;
  for (unsigned it = blockIdx.x * kRelWarps + warp; it < items; it += gridDim.x * kRelWarps) {
    const unsigned r = it / strips;
    const int strip = static_cast<int>(it - r * strips);
    const unsigned smp = r / chunks;
    const int i0 = static_cast<int>(r - smp * chunks) * rows;
    const int i1 = min(i0 + rows, Lq);
    const T* src = db + smp * stride_b + h * stride_h + i0 * stride_i;
    if constexpr (VEC) {
      constexpr int kW = static_cast<int>(sizeof(T)) * 2;  // loaded words of a lane and row
      const int j = strip * kGradCols + 8 * lane;            // the lane's first column
      float acc[15];  // acc[7 + s]: the diagonal of column s of the block's first row
#pragma unroll
      for (int e = 0; e < 15; ++e) acc[e] = 0.f;
      for (int i = i0; i < i1; i += 8, src += 8 * stride_i) {
        uint32_t raw[8][kW];
        const T* p = src + j;
        if (i + 8 <= i1 && j + 8 <= Lk) {
#pragma unroll
          for (int u = 0; u < 8; ++u, p += stride_i) {
#pragma unroll
            for (int q = 0; q < kW; q += 4) {
              const uint4 w = __ldcs(reinterpret_cast<const uint4*>(p) + q / 4);
              raw[u][q] = w.x, raw[u][q + 1] = w.y, raw[u][q + 2] = w.z, raw[u][q + 3] = w.w;
            }
          }
        } else {
          // past the last row, or the row's end inside this lane's eight columns or before them
#pragma unroll
          for (int u = 0; u < 8; ++u, p += stride_i) {
            T e8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) e8[e] = i + u < i1 && j + e < Lk ? p[e] : T(0.f);
#pragma unroll
            for (int q = 0; q < kW; ++q) raw[u][q] = reinterpret_cast<const uint32_t*>(e8)[q];
          }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          float v[8];
          widen8<T>(raw[u], v);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[7 + e - u] += v[e];
        }
        // Eight columns on: sums 0 .. 7 belong to the next lane, -7 .. -1 stay as 1 .. 7. The last
        // lane's leave the strip, one after the other from one lane.
        const int d = j - i - q_offset;
        float up[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          up[e] = __shfl_up_sync(0xffffffffu, acc[7 + e], 1);
          if (lane == 0) up[e] = 0.f;
        }
        float leaving = 0.f;  // lane e < 8 takes sum e of the last lane
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __shfl_sync(0xffffffffu, acc[7 + e], 31);
          if (lane == e) leaving = x;
        }
        add_diag(__shfl_sync(0xffffffffu, d, 31) + lane, leaving);
#pragma unroll
        for (int e = 7; e > 0; --e) acc[7 + e] = acc[e - 1] + up[e];
        acc[7] = up[0];
#pragma unroll
        for (int e = 0; e < 7; ++e) acc[e] = 0.f;
      }
      const int rows8 = (i1 - i0 + 7) / 8 * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) add_diag(j + e - (i0 + rows8) - q_offset, acc[7 + e]);
    } else {
      const int dw = strip * kGradCols - (i1 - 1);  // the strip's first diagonal (j - i)
      const int d0 = dw + lane;
      float acc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
      // rows with a column of the strip
      const int r0 = max(i0, -(dw + kGradCols - 1)), r1 = min(i1, Lk - dw);
      const bool inside = dw + r0 >= 0 && dw + r1 - 1 + kGradCols <= Lk;  // all 256 of every row
      const uint64_t step = static_cast<uint64_t>((stride_i + 1) * static_cast<int>(sizeof(T)));
      // address of the strip's first column in the next row to load and in the next row to read
      uint64_t load_at = reinterpret_cast<uint64_t>(src) +
                         static_cast<uint64_t>(((r0 - i0) * stride_i + dw + r0) * static_cast<int>(sizeof(T)));
      uint32_t read_at = static_cast<uint32_t>(load_at);
      const uint32_t lane_to = ring + lane * 16;
      // An aligned 16-byte block is loaded when it holds an element of the strip and of the row.
      auto fetch = [&](int i, int slot) {
        const uint64_t block = (load_at & ~15ull) + lane * 16;
        const uint32_t to = lane_to + slot * kRowBytes;
        if (inside || (dw + i >= 0 && dw + i + kGradCols <= Lk)) {
#pragma unroll
          for (int c = 0; c < kGradCols * static_cast<int>(sizeof(T)); c += 512)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + c), "l"(block + c) : "memory");
          if (lane == 0 && (load_at & 15) != 0)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + kRowBytes - 16),
                         "l"(block + kRowBytes - 16)
                         : "memory");
        } else {
          // byte positions of the row's columns 0 and Lk from the strip's first block
          const int off = static_cast<int>(load_at & 15) - (dw + i) * static_cast<int>(sizeof(T));
          const int end = off + Lk * static_cast<int>(sizeof(T));
#pragma unroll
          for (int c = 0; c < kRowBytes; c += 512) {
            const int at = c + lane * 16;
            if (at < kRowBytes && at + 16 > off && at < end)
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + c), "l"(block + c) : "memory");
          }
        }
        load_at += step;
      };
      auto consume = [&](int k, int slot) {
        const T* line = reinterpret_cast<const T*>(rows_smem + slot * kRowBytes + (read_at & 15u)) + lane;
        if (inside || (dw + k >= 0 && dw + k + kGradCols <= Lk)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] += to_f32<T>(line[32 * e]);
        } else {
          const int j = d0 + k;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (static_cast<unsigned>(j + 32 * e) < static_cast<unsigned>(Lk)) acc[e] += to_f32<T>(line[32 * e]);
        }
        read_at += static_cast<uint32_t>(step);
      };
      for (int base = r0; base < r1 + kRing - 1; base += kRing) {
#pragma unroll
        for (int u = 0; u < kRing; ++u) {
          const int i = base + u, k = i - (kRing - 1);  // the rows loaded and read now
          if (i < r1) fetch(i, u);
          asm volatile("cp.async.commit_group;" ::: "memory");
          if (k >= r0 && k < r1) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 1) : "memory");
            __syncwarp();
            consume(k, (u + 1) % kRing);
            __syncwarp();  // the slot is loaded anew in the next turn
          }
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
      for (int e = 0; e < 8; ++e) add_diag(d0 + 32 * e - q_offset, acc[e]);
    }
  }
  if (by_diag) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      left += __shfl_xor_sync(0xffffffffu, left, o);
      right += __shfl_xor_sync(0xffffffffu, right, o);
    }
    if (lane == 0) {
      mine[0] += left;
      mine[reach + ahead] += right;
    }
  }
  __syncthreads();
  for (int t = threadIdx.x; t < sums; t += kRelThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kRelWarps; ++w) s += acc_b[w * sums + t];
    acc_b[t] = s;  // (row 0 is read by this thread only)
  }
  __syncthreads();
  for (int b = threadIdx.x; b < buckets; b += kRelThreads) {
    const float s = by_diag ? rel_bucket_sum(acc_b, reach, bounds, rb.n_bounds, b) : acc_b[b];
    part[(static_cast<size_t>(h) * gridDim.x + blockIdx.x) * buckets + b] = s;
  }
}

// dtable[b, h] = sum over the CTAs' partial buckets, rounded once to dtype. A warp takes a bucket of
// a head: lane l adds parts l, l + 32, ..., then the lanes are added (a fixed order).
__global__ void __launch_bounds__(256)
    rel_table_sum_kernel(const float* __restrict__ part, int parts, int buckets, int H, void* __restrict__ out,
                         int dtype) {
  const int b = blockIdx.x * 8 + (threadIdx.x >> 5), h = blockIdx.y, lane = threadIdx.x & 31;
  if (b >= buckets) return;
  const float* p = part + static_cast<size_t>(h) * parts * buckets + b;
  float s = 0.f;
  for (int x = lane; x < parts; x += 32) s += p[static_cast<size_t>(x) * buckets];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane != 0) return;
  const size_t at = static_cast<size_t>(b) * H + h;
  if (dtype == 0) {
    static_cast<float*>(out)[at] = s;
  } else if (dtype == 1) {
    static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(s);
  } else {
    static_cast<__half*>(out)[at] = __float2half_rn(s);
  }
}

int cuda_rc(cudaError_t e) {
  if (e == cudaSuccess) return WDIT_OK;
  cudaGetLastError();  // reported here, not by the next launch too
  return WDIT_ERR_CUDA_BASE + static_cast<int>(e);
}

// At most 34 KB, and 65 KB of rings.
int grad_smem(const RelBuckets& rb, int buckets, bool vec, int esize) {
  const int reach = rb.bounds[rb.n_bounds - 1];
  const int sums = reach <= kGradReach ? reach + (rb.bidirectional ? reach : 0) + 1 : buckets;
  return grad_fixed_bytes(sums) + (vec ? 0 : kRelWarps * kRing * grad_row_bytes(esize));
}

// Rows of a strip and CTAs per head of the gradient. All CTAs run at once (per_sm of them), a head's
// warps share its strips. Aligned rows: the rows whose rounds of strips cost least, a strip costing
// its rows and 24 more for its ends (us with 32 / 64 / 128 rows, bf16: 64 heads x 512 x 512 9.6 /
// 10.9 / 15.4, twice that batch 15.9 / 15.4 / 21.3, eight times 51.5 / 49.9 / 48.7). Unaligned rows:
// 32 (40 heads x 2047 x 2049 fp32 122 / 164 / 164, 12 heads x 333 x 333 fp16 18 / 30 / 54).
struct GradPlan {
  int rows, parts;
};
GradPlan grad_plan(int B, int H, int Lq, int Lk, bool vec, int per_sm, int sms) {
  const long long most = sms * per_sm / H > 0 ? sms * per_sm / H : 1;
  GradPlan best = {kGradRowsMin, 1};
  long long best_cost = -1;
  for (int rows = kGradRowsMin; rows <= (vec ? kGradRowsMax : kGradRowsMin); rows *= 2) {
    const long long items = static_cast<long long>(B) * ((Lq + rows - 1) / rows) * grad_strips(Lk, rows, vec);
    const long long rounds = (items + most * kRelWarps - 1) / (most * kRelWarps);
    const long long cost = rounds * (rows + 24);
    if (best_cost < 0 || cost < best_cost) {
      best_cost = cost;
      best = {rows, static_cast<int>((items + rounds * kRelWarps - 1) / (rounds * kRelWarps))};
    }
  }
  return best;
}

template <typename T>
int launch_bias(const void* table, const RelBuckets& rb, int H, int Lq, int Lk, int q_offset, void* out,
                cudaStream_t st) {
  const int rows = Lq < kBiasRows ? Lq : kBiasRows;
  const long long tiles = static_cast<long long>((Lk + kBiasCols - 1) / kBiasCols) * ((Lq + rows - 1) / rows);
  if (tiles > 0x7fffffffll) return WDIT_ERR_SHAPE;  // (more cells than any memory holds)
  const dim3 grid(static_cast<unsigned>(tiles), H);
  rel_bias_kernel<T><<<grid, kRelThreads, 0, st>>>(static_cast<const T*>(table), rb, H, Lq, Lk, q_offset, rows,
                                                   static_cast<T*>(out));
  return cuda_rc(cudaGetLastError());
}

template <typename T>
int launch_grad(const void* db, const RelBuckets& rb, int B, int H, int Lq, int Lk, int q_offset, long long sb,
                long long sh, long long si, int buckets, bool vec, GradPlan plan, float* part, cudaStream_t st) {
  const int rows = plan.rows;
  const size_t smem = grad_smem(rb, buckets, vec, static_cast<int>(sizeof(T)));
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(rel_bias_grad_kernel<T, false>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024);
    if (e != cudaSuccess) return cuda_rc(e);
  }
  const dim3 grid(plan.parts, H);
  const T* p = static_cast<const T*>(db);
  if (vec)
    rel_bias_grad_kernel<T, true><<<grid, kRelThreads, smem, st>>>(p, rb, B, Lq, Lk, q_offset, sb, sh, si, buckets,
                                                                  rows, part);
  else
    rel_bias_grad_kernel<T, false><<<grid, kRelThreads, smem, st>>>(p, rb, B, Lq, Lk, q_offset, sb, sh, si, buckets,
                                                                   rows, part);
  return cuda_rc(cudaGetLastError());
}

int check_rel(const int* bounds, int n_bounds, int H, int Lq, int Lk, int q_offset, int dtype) {
  if (bounds == nullptr) return WDIT_ERR_ARG;
  if (n_bounds < 1 || n_bounds > kMaxRelBounds || H < 1 || H > 65535 || Lq < 0 || Lk < 0) return WDIT_ERR_SHAPE;
  // positions up to 2^30, rows up to 2^28 cells (byte offsets in a row stay inside 32 bits)
  if (q_offset < 0 || static_cast<long long>(q_offset) + Lq > (1ll << 30) || Lq > (1 << 28) || Lk > (1 << 28))
    return WDIT_ERR_SHAPE;
  if (dtype < 0 || dtype > 2) return WDIT_ERR_ARG;
  return WDIT_OK;
}

}  // namespace

int launch_rel_table_sum(const float* part, int parts, int buckets, int H, void* out, int dtype, void* stream) {
  rel_table_sum_kernel<<<dim3((buckets + 7) / 8, H), 256, 0, static_cast<cudaStream_t>(stream)>>>(part, parts, buckets,
                                                                                                 H, out, dtype);
  return cuda_rc(cudaGetLastError());
}

}  // namespace wdit

using namespace wdit;

extern "C" {

int wdit_rel_pos_bias(const void* table, int dtype, const int* bounds, int n_bounds, int bidirectional, int H, int Lq,
                      int Lk, int q_offset, void* out, void* stream) {
  const int rc = check_rel(bounds, n_bounds, H, Lq, Lk, q_offset, dtype);
  if (rc) return rc;
  if (Lq == 0 || Lk == 0) return WDIT_OK;
  if (table == nullptr || out == nullptr) return WDIT_ERR_ARG;
  if ((reinterpret_cast<uintptr_t>(out) & 15) != 0 || (reinterpret_cast<uintptr_t>(table) & (dtype == 0 ? 3 : 1)) != 0)
    return WDIT_ERR_ALIGN;
  RelBuckets rb;
  if (!rel_fill(&rb, bounds, n_bounds, bidirectional)) return WDIT_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == 0) return launch_bias<float>(table, rb, H, Lq, Lk, q_offset, out, st);
  if (dtype == 1) return launch_bias<__nv_bfloat16>(table, rb, H, Lq, Lk, q_offset, out, st);
  return launch_bias<__half>(table, rb, H, Lq, Lk, q_offset, out, st);
}

long long wdit_rel_pos_bias_grad_workspace_bytes(int B, int H, int Lq, int Lk, int n_bounds, int bidirectional) {
  if (B <= 0 || H <= 0 || Lq <= 0 || Lk <= 0 || n_bounds < 1) return 0;
  // (the rows' alignment and the last bound are not known here: enough for any)
  const int sms = sm_count();
  int parts = grad_plan(B, H, Lq, Lk, true, 2, sms).parts;
  for (int per_sm = 2; per_sm <= 3; ++per_sm) {
    const int n = grad_plan(B, H, Lq, Lk, false, per_sm, sms).parts;
    parts = n > parts ? n : parts;
  }
  return 4ll * parts * H * rel_num_buckets(n_bounds, bidirectional);
}

int wdit_rel_pos_bias_grad(const void* dbias, int dtype, int B, int H, int Lq, int Lk, long long stride_b,
                           long long stride_h, long long stride_i, const int* bounds, int n_bounds, int bidirectional,
                           int q_offset, void* dtable, int dtable_dtype, void* workspace, long long workspace_bytes,
                           void* stream) {
  int rc = check_rel(bounds, n_bounds, H, Lq, Lk, q_offset, dtype);
  if (rc) return rc;
  if (B < 0) return WDIT_ERR_SHAPE;
  if (dtable == nullptr || dtable_dtype < 0 || dtable_dtype > 2) return WDIT_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int buckets = rel_num_buckets(n_bounds, bidirectional);
  if (B == 0 || Lq == 0 || Lk == 0) {  // no cells: a zero gradient
    return cuda_rc(cudaMemsetAsync(dtable, 0, static_cast<size_t>(buckets) * H * (dtable_dtype == 0 ? 4 : 2), st));
  }
  if (dbias == nullptr) return WDIT_ERR_ARG;
  if (stride_b < 0 || stride_h < 0 || stride_i < 0) return WDIT_ERR_SHAPE;
  if (static_cast<long long>(B) * ((Lq + kGradRowsMin - 1) / kGradRowsMin) * grad_strips(Lk, kGradRowsMin, false) >= 1ll << 31)
    return WDIT_ERR_SHAPE;
  if (workspace == nullptr ||
      workspace_bytes < wdit_rel_pos_bias_grad_workspace_bytes(B, H, Lq, Lk, n_bounds, bidirectional))
    return WDIT_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return WDIT_ERR_ALIGN;
  RelBuckets rb;
  if (!rel_fill(&rb, bounds, n_bounds, bidirectional)) return WDIT_ERR_ARG;
  const long long V = dtype == 0 ? 4 : 8;
  const bool vec =
      (reinterpret_cast<uintptr_t>(dbias) & 15) == 0 && stride_b % V == 0 && stride_h % V == 0 && stride_i % V == 0;
  // three CTAs per SM where their shared memory fits, two of the aligned form by its registers
  const int smem = grad_smem(rb, buckets, vec, dtype == 0 ? 4 : 2);
  const GradPlan plan = grad_plan(B, H, Lq, Lk, vec, !vec && 3 * (smem + 1024) <= 228 * 1024 ? 3 : 2, sm_count());
  float* part = static_cast<float*>(workspace);
  auto go = [&](auto* type) {
    return launch_grad<std::remove_pointer_t<decltype(type)>>(dbias, rb, B, H, Lq, Lk, q_offset, stride_b, stride_h,
                                                              stride_i, buckets, vec, plan, part, st);
  };
  rc = dtype == 0 ? go(static_cast<float*>(nullptr))
                  : (dtype == 1 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<__half*>(nullptr)));
  if (rc) return rc;
  return launch_rel_table_sum(part, plan.parts, buckets, H, dtable, dtable_dtype, stream);
}

}  // extern "C"
