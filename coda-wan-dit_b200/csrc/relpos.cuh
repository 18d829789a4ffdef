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

__host__ __device__ inline int rel_num_buckets(int n_bounds, int bidirectional) { return (n_bounds + 1) * (bidirectional ? 2 : 1); }

// Host check and copy of the caller's bounds; false = not ascending positive distances.
inline bool rel_fill(RelBuckets* rb, const int* bounds, int n_bounds, int bidirectional) {
  rb->n_bounds = n_bounds;
  rb->bidirectional = bidirectional != 0 ? 1 : 0;
  for (int i = 0; i < n_bounds; ++i) {
    if (bounds[i] < 1 || (i > 0 && bounds[i] < bounds[i - 1])) return false;
    rb->bounds[i] = bounds[i];
  }
  return true;
}

}  // namespace wdit
