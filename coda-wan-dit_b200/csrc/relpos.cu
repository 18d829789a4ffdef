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
// shared memory, and writes every row as a shifted window of that line with 16-byte stores.
//
// Gradient (rel_bias_grad_kernel). A warp walks down a strip of 256 columns; a lane's accumulators
// follow the diagonals: from a row to the next every diagonal moves one column to the right, so
// the accumulators shift by one column (a register renaming, plus one shuffle per lane boundary)
// instead of being looked up. Only the diagonal that leaves the strip is stored per row. At the
// strip's end each warp adds its 256 + rows diagonal sums into the buckets. Sums are fp32, the
// order is fixed (no atomics), and a second small kernel adds the CTAs' partial buckets.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "relpos.cuh"
#include "wdit_internal.h"

namespace wdit {
namespace {

constexpr int kRelThreads = 256;
constexpr int kRelWarps = kRelThreads / 32;
constexpr int kBiasRows = 32;    // rows of a forward tile
constexpr int kBiasCols = 2048;  // columns of a forward tile
constexpr int kGradRows = 64;    // rows of a gradient strip
constexpr int kGradCols = 256;   // columns of a gradient strip (8 per lane)

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

// Lines of table values per element parity, so that a 16-byte piece of 2-byte elements that
// starts at an odd diagonal is still read as aligned 32-bit words.
template <typename T>
__global__ void __launch_bounds__(kRelThreads)
    rel_bias_kernel(const T* __restrict__ table, const __grid_constant__ RelBuckets rb, int H, int Lq, int Lk,
                    int q_offset, int rows, T* __restrict__ out) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  constexpr int kCopies = sizeof(T) == 2 ? 2 : 1;
  constexpr int kLine = kBiasCols + kBiasRows + 16;
  __shared__ __align__(16) T line[kCopies][kLine];
  __shared__ int bounds[kMaxRelBounds];
  const int h = blockIdx.z;
  const int i0 = static_cast<int>(blockIdx.y) * rows;
  const int i1 = min(i0 + rows, Lq);
  const int j0 = static_cast<int>(blockIdx.x) * kBiasCols;
  const int j1 = min(j0 + kBiasCols, Lk);
  for (int t = threadIdx.x; t < rb.n_bounds; t += kRelThreads) bounds[t] = rb.bounds[t];
  __syncthreads();
  const int d0 = j0 - (i1 - 1) - q_offset;  // the tile's first diagonal
  const int nd = (j1 - j0) + (i1 - i0) - 1;
  for (int t = threadIdx.x; t < nd; t += kRelThreads) {
    const T v = table[static_cast<size_t>(rel_bucket(bounds, rb.n_bounds, rb.bidirectional, d0 + t)) * H + h];
    line[0][t] = v;
    if (kCopies == 2 && t > 0) line[kCopies - 1][t - 1] = v;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int segs = (j1 - j0 + V - 1 + 32 * V - 1) / (32 * V);  // warp-wide pieces of a row, any alignment
  for (int it = warp; it < segs * (i1 - i0); it += kRelWarps) {
    const int i = i0 + it / segs;
    T* row = out + (static_cast<size_t>(h) * Lq + i) * Lk;
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row + j0) & 15) / sizeof(T));
    const int j = j0 - mis + ((it % segs) * 32 + lane) * V;  // 16-byte aligned in memory
    const int s = j - j0 + (i1 - 1 - i);                      // its diagonal in the line
    if (j >= j0 && j + V <= j1) {
      uint32_t w[4];
      if constexpr (sizeof(T) == 2) {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(&line[s & (kCopies - 1)][s & ~1]);
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = src[q];
      } else {
        const uint32_t* src = reinterpret_cast<const uint32_t*>(&line[0][s]);
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = src[q];
      }
      *reinterpret_cast<uint4*>(row + j) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int q = 0; q < V; ++q)
        if (j + q >= j0 && j + q < j1) row[j + q] = line[0][s + q];
    }
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
    const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = to_f32<T>(e[q]);
  }
}

// VEC: rows start on 16-byte boundaries and lane l holds columns 8 l .. 8 l + 7 of the strip;
// otherwise lane l holds columns l + 32 e (coalesced single elements).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRelThreads)
    rel_bias_grad_kernel(const T* __restrict__ db, const __grid_constant__ RelBuckets rb, int B, int Lq, int Lk,
                         int q_offset, long long stride_b, long long stride_h, long long stride_i, int buckets,
                         float* __restrict__ part) {
  extern __shared__ float sm[];
  constexpr int kDiag = kGradCols + kGradRows;
  float* acc_b = sm;                                   // [warps][buckets]
  float* diag_all = sm + kRelWarps * buckets;          // [warps][kDiag]
  int* bounds = reinterpret_cast<int*>(diag_all + kRelWarps * kDiag);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y;
  for (int t = threadIdx.x; t < rb.n_bounds; t += kRelThreads) bounds[t] = rb.bounds[t];
  for (int t = threadIdx.x; t < kRelWarps * buckets; t += kRelThreads) acc_b[t] = 0.f;
  __syncthreads();
  float* mine = acc_b + warp * buckets;
  float* diag = diag_all + warp * kDiag;
  const int chunks = (Lq + kGradRows - 1) / kGradRows;
  const int strips = (Lk + kGradCols - 1) / kGradCols;
  const long long items = static_cast<long long>(B) * chunks * strips;
  for (long long it = static_cast<long long>(blockIdx.x) * kRelWarps + warp; it < items;
       it += static_cast<long long>(gridDim.x) * kRelWarps) {
    const int strip = static_cast<int>(it % strips);
    const long long r = it / strips;
    const int i0 = static_cast<int>(r % chunks) * kGradRows;
    const int i1 = min(i0 + kGradRows, Lq);
    const int j0 = strip * kGradCols;
    const T* src = db + (r / chunks) * stride_b + h * stride_h + j0;
    float acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    // diag[t] holds the sum of diagonal d = j - i (row-relative) = t - (kGradRows - 1)
    constexpr int kStep = VEC ? 8 : 4;  // rows whose loads are in flight together
    for (int i = i0; i < i1; i += kStep) {
      float v[kStep][8];
#pragma unroll
      for (int u = 0; u < kStep; ++u) {
        const T* p = src + static_cast<long long>(i + u) * stride_i;
        const bool row_ok = i + u < i1;
        if constexpr (VEC) {
          // rows are a multiple of 16 bytes long, so 8 columns are all inside or (past the row's
          // end: at most one 16-byte piece of fp32 inside) checked one by one
          if (row_ok && j0 + 8 * lane + 8 <= Lk) {
            load8<T>(p + 8 * lane, v[u]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              v[u][e] = row_ok && j0 + 8 * lane + e < Lk ? to_f32<T>(p[8 * lane + e]) : 0.f;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            v[u][e] = row_ok && j0 + lane + 32 * e < Lk ? to_f32<T>(p[lane + 32 * e]) : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < kStep; ++u) {
        if (i + u >= i1) break;
        if (i + u > i0) {
          // next row: every diagonal moves one column right; the strip's last one leaves
          const float out = acc[7];
          if (lane == 31) diag[kGradCols - 1 - (i + u - 1 - i0) + kGradRows - 1] = out;
          if constexpr (VEC) {
            float in = __shfl_up_sync(0xffffffffu, acc[7], 1);
            if (lane == 0) in = 0.f;
#pragma unroll
            for (int e = 7; e > 0; --e) acc[e] = acc[e - 1];
            acc[0] = in;
          } else {
            float rot[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) rot[e] = __shfl_sync(0xffffffffu, acc[e], (lane + 31) & 31);
#pragma unroll
            for (int e = 7; e > 0; --e) acc[e] = lane == 0 ? rot[e - 1] : rot[e];
            acc[0] = lane == 0 ? 0.f : rot[0];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += v[u][e];
      }
    }
    // the diagonals still in the strip at its last row
    const int last = i1 - 1 - i0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = VEC ? 8 * lane + e : lane + 32 * e;
      diag[c - last + kGradRows - 1] = acc[e];
    }
    __syncwarp();
    // Diagonals -last .. 255 into the buckets, 32 at a time: equal buckets are neighbours, so a
    // piece usually has one or a few; each is summed over its lanes in a fixed order.
    const int base = kGradRows - 1 - last;
    const int nd = kGradCols + last;
    const int d_first = j0 - (i0 + last) - q_offset;
    for (int t0 = 0; t0 < nd; t0 += 32) {
      const int t = t0 + lane;
      const float val = t < nd ? diag[base + t] : 0.f;
      const int b = t < nd ? rel_bucket(bounds, rb.n_bounds, rb.bidirectional, d_first + t) : -1 - lane;
      add_buckets(mine, b, val, lane);
    }
    __syncwarp();  // diag and mine are reused by the next strip
  }
  __syncthreads();
  for (int b = threadIdx.x; b < buckets; b += kRelThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kRelWarps; ++w) s += acc_b[w * buckets + b];
    part[(static_cast<size_t>(h) * gridDim.x + blockIdx.x) * buckets + b] = s;
  }
}

// dtable[b, h] = sum over the CTAs' partial buckets, one thread each (a fixed order).
__global__ void rel_table_sum_kernel(const float* __restrict__ part, int parts, int buckets, int H,
                                     float* __restrict__ out) {
  const int h = blockIdx.x;
  for (int b = threadIdx.x; b < buckets; b += blockDim.x) {
    const float* p = part + static_cast<size_t>(h) * parts * buckets + b;
    float s = 0.f;
    for (int x = 0; x < parts; ++x) s += p[static_cast<size_t>(x) * buckets];
    out[static_cast<size_t>(b) * H + h] = s;
  }
}

int rel_cta_target() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148 * 4;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148 * 4;
  return n * 4;
}

// CTAs per head of the gradient: about four per SM over all heads, at least one strip per warp.
int grad_parts(int B, int H, int Lq, int Lk, int target) {
  const long long items = static_cast<long long>(B) * ((Lq + kGradRows - 1) / kGradRows) *
                          ((Lk + kGradCols - 1) / kGradCols);
  long long x = (target + H - 1) / H;
  const long long most = (items + kRelWarps - 1) / kRelWarps;
  if (x > most) x = most;
  return x < 1 ? 1 : static_cast<int>(x);
}

template <typename T>
int launch_bias(const void* table, const RelBuckets& rb, int H, int Lq, int Lk, int q_offset, void* out,
                cudaStream_t st) {
  const int rows = Lq < kBiasRows ? Lq : kBiasRows;
  const dim3 grid((Lk + kBiasCols - 1) / kBiasCols, (Lq + rows - 1) / rows, H);
  rel_bias_kernel<T><<<grid, kRelThreads, 0, st>>>(static_cast<const T*>(table), rb, H, Lq, Lk, q_offset, rows,
                                                   static_cast<T*>(out));
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? WDIT_OK : WDIT_ERR_CUDA_BASE + static_cast<int>(e);
}

template <typename T>
int launch_grad(const void* db, const RelBuckets& rb, int B, int H, int Lq, int Lk, int q_offset, long long sb,
                long long sh, long long si, int buckets, int parts, float* part, cudaStream_t st) {
  constexpr long long V = 16 / static_cast<long long>(sizeof(T));
  const bool vec = (reinterpret_cast<uintptr_t>(db) & 15) == 0 && sb % V == 0 && sh % V == 0 && si % V == 0;
  const size_t smem = (static_cast<size_t>(kRelWarps) * (buckets + kGradCols + kGradRows) + kMaxRelBounds) * 4;
  const dim3 grid(parts, H);
  const T* p = static_cast<const T*>(db);
  if (vec)
    rel_bias_grad_kernel<T, true><<<grid, kRelThreads, smem, st>>>(p, rb, B, Lq, Lk, q_offset, sb, sh, si, buckets,
                                                                  part);
  else
    rel_bias_grad_kernel<T, false><<<grid, kRelThreads, smem, st>>>(p, rb, B, Lq, Lk, q_offset, sb, sh, si, buckets,
                                                                   part);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? WDIT_OK : WDIT_ERR_CUDA_BASE + static_cast<int>(e);
}

int check_rel(const int* bounds, int n_bounds, int H, int Lq, int Lk, int q_offset, int dtype) {
  if (bounds == nullptr) return WDIT_ERR_ARG;
  if (n_bounds < 1 || n_bounds > kMaxRelBounds || H < 1 || H > 65535 || Lq < 0 || Lk < 0) return WDIT_ERR_SHAPE;
  if (q_offset < 0 || static_cast<long long>(q_offset) + Lq > (1ll << 30) || Lk > (1 << 30)) return WDIT_ERR_SHAPE;
  if (dtype < 0 || dtype > 2) return WDIT_ERR_ARG;
  return WDIT_OK;
}

}  // namespace

int launch_rel_table_sum(const float* part, int parts, int buckets, int H, float* out, void* stream) {
  rel_table_sum_kernel<<<H, 128, 0, static_cast<cudaStream_t>(stream)>>>(part, parts, buckets, H, out);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? WDIT_OK : WDIT_ERR_CUDA_BASE + static_cast<int>(e);
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
  if ((Lq + kBiasRows - 1) / kBiasRows > 65535) return WDIT_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(out) & 15) != 0 || (reinterpret_cast<uintptr_t>(table) & 3) != 0)
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
  return 4ll * grad_parts(B, H, Lq, Lk, rel_cta_target()) * H * rel_num_buckets(n_bounds, bidirectional);
}

int wdit_rel_pos_bias_grad(const void* dbias, int dtype, int B, int H, int Lq, int Lk, long long stride_b,
                           long long stride_h, long long stride_i, const int* bounds, int n_bounds, int bidirectional,
                           int q_offset, float* dtable, void* workspace, long long workspace_bytes, void* stream) {
  int rc = check_rel(bounds, n_bounds, H, Lq, Lk, q_offset, dtype);
  if (rc) return rc;
  if (B < 0) return WDIT_ERR_SHAPE;
  if (dtable == nullptr) return WDIT_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int buckets = rel_num_buckets(n_bounds, bidirectional);
  if (B == 0 || Lq == 0 || Lk == 0) {  // no cells: a zero gradient
    const cudaError_t e = cudaMemsetAsync(dtable, 0, static_cast<size_t>(buckets) * H * 4, st);
    return e == cudaSuccess ? WDIT_OK : WDIT_ERR_CUDA_BASE + static_cast<int>(e);
  }
  if (dbias == nullptr) return WDIT_ERR_ARG;
  if (stride_b < 0 || stride_h < 0 || stride_i < 0) return WDIT_ERR_SHAPE;
  if (workspace == nullptr ||
      workspace_bytes < wdit_rel_pos_bias_grad_workspace_bytes(B, H, Lq, Lk, n_bounds, bidirectional))
    return WDIT_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return WDIT_ERR_ALIGN;
  RelBuckets rb;
  if (!rel_fill(&rb, bounds, n_bounds, bidirectional)) return WDIT_ERR_ARG;
  const int parts = grad_parts(B, H, Lq, Lk, rel_cta_target());
  float* part = static_cast<float*>(workspace);
  if (dtype == 0)
    rc = launch_grad<float>(dbias, rb, B, H, Lq, Lk, q_offset, stride_b, stride_h, stride_i, buckets, parts, part, st);
  else if (dtype == 1)
    rc = launch_grad<__nv_bfloat16>(dbias, rb, B, H, Lq, Lk, q_offset, stride_b, stride_h, stride_i, buckets, parts,
                                    part, st);
  else
    rc = launch_grad<__half>(dbias, rb, B, H, Lq, Lk, q_offset, stride_b, stride_h, stride_i, buckets, parts, part,
                             st);
  if (rc) return rc;
  return launch_rel_table_sum(part, parts, buckets, H, dtable, stream);
}

}  // extern "C"
