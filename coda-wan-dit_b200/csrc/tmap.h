// Tensor-map encoding shared by the translation units that issue TMA (defined in gemm.cu).
#pragma once
#include <cuda.h>

namespace wdit {

// rank-`rank` tiled map over 2- or 4-byte elements. dims / box innermost first; strides_bytes[i] is
// the byte stride of dimension i + 1. Returns WDIT_OK / WDIT_ERR_*.
int encode_tiled(CUtensorMap* map, CUtensorMapDataType dt, int rank, const void* ptr, const unsigned long long* dims,
                 const unsigned long long* strides_bytes, const unsigned int* box, CUtensorMapSwizzle sw);

}  // namespace wdit
