// Tensor maps for tiled TMA loads, 128-byte swizzled, zeros outside.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

namespace lmc {

// `dims` and `box` innermost first; `strides` in elements for dimensions 1...
// (a dimension of one has no stride to keep to the rules).
inline bool encode_rows(CUtensorMap *map, bool bf16, const void *base, int rank,
                        const long long *dims, const long long *strides, const int *box) {
  using Encode = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                              const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault,
                                         &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      fn = nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  if (encode == nullptr) return false;
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], step[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i]);
    b[i] = static_cast<cuuint32_t>(box[i]);
    step[i] = 1;
    if (i > 0) s[i - 1] = static_cast<cuuint64_t>(dims[i] == 1 ? dims[0] * 2 : strides[i - 1] * 2);
  }
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                static_cast<cuuint32_t>(rank), const_cast<void *>(base), d, s, b, step,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace lmc
