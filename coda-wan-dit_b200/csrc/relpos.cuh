// The bucket rule of the learned relative position bias, shared by the kernels that write the
// bias, reduce its gradient or read it inside attention.
//
// Relative position d = key - query. Distance n = |d| (bidirectional: keys ahead of the query
// use the upper half of the buckets) or max(-d, 0) (one direction). The bucket of n is the number
// of bounds <= n: the caller passes the distances at which the bucket steps up, so that the
// logarithmic part of the rule is decided in whole numbers on the host and a distance next to a
// border never depends on the rounding of a device logarithm.
#pragma once

namespace wdit {

constexpr int kMaxRelBounds = 255;

struct RelBuckets {
  int n_bounds;
  int bidirectional;
  int bounds[kMaxRelBounds];  // ascending, >= 1
};

// Number of bounds <= n by binary search (bounds in shared memory).
__device__ __forceinline__ int rel_bucket(const int* bounds, int n_bounds, int bidirectional, int d) {
  const int n = bidirectional ? (d < 0 ? -d : d) : (d < 0 ? -d : 0);
  int lo = 0, hi = n_bounds;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (bounds[mid] <= n) {
      lo = mid + 1;
    } else {
      hi = mid;
    }
  }
  return bidirectional && d > 0 ? lo + n_bounds + 1 : lo;
}

// Adds v into the warp's bucket sums: lanes with a bucket of their own directly, equal ones
// through a fixed-order sum over the lanes.
__device__ __forceinline__ void add_buckets(float* acc, int bucket, float v, int lane) {
  const unsigned same = __match_any_sync(0xffffffffu, bucket);
  const bool alone = same == (1u << lane);
  if (alone && bucket >= 0) acc[bucket] += v;
  unsigned todo = __ballot_sync(0xffffffffu, !alone && bucket >= 0);
  while (todo != 0) {
    const int bb = __shfl_sync(0xffffffffu, bucket, __ffs(todo) - 1);
    float s = bucket == bb ? v : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) acc[bb] += s;
    todo &= ~__ballot_sync(0xffffffffu, bucket == bb);
  }
  __syncwarp();
}

// Sum of bucket b from sums by diagonal: sums[reach + d] for -reach <= d <= reach (bidirectional) or
// <= 0, the ends holding everything past them; reach is the last bound.
__device__ __forceinline__ float rel_bucket_sum(const float* sums, int reach, const int* bounds, int n_bounds, int b) {
  const bool up = b > n_bounds;  // keys ahead of the query
  const int k = up ? b - n_bounds - 1 : b;
  const int lo = k == 0 ? 0 : bounds[k - 1];  // the bucket's distances
  const int hi = k == n_bounds ? reach : bounds[k] - 1;
  float s = 0.f;
  if (up) {
    for (int n = lo < 1 ? 1 : lo; n <= hi; ++n) s += sums[reach + n];
  } else {
    for (int n = lo; n <= hi; ++n) s += sums[reach - n];
  }
  return s;
}

__host__ __device__ inline int rel_num_buckets(int n_bounds, int bidirectional) { return (n_bounds + 1) * (bidirectional ? 2 : 1); }

// Host check and copy of the caller's bounds; false = not ascending distances in 1 .. 2^29 (positions
// go up to 2^30: their sums stay inside 32 bits).
inline bool rel_fill(RelBuckets* rb, const int* bounds, int n_bounds, int bidirectional) {
  rb->n_bounds = n_bounds;
  rb->bidirectional = bidirectional != 0 ? 1 : 0;
  for (int i = 0; i < n_bounds; ++i) {
    if (bounds[i] < 1 || bounds[i] > (1 << 29) || (i > 0 && bounds[i] < bounds[i - 1])) return false;
    rb->bounds[i] = bounds[i];
  }
  return true;
}

}  // namespace wdit
