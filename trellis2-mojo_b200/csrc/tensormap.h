// Tensor maps for tiled TMA loads, encoded on the host for each call.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/t2sc.h"

namespace t2sc {

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder (looked up once; the library does not link libcuda).
inline EncodeTiled tensormap_encoder() {
  static const EncodeTiled fn = []() -> EncodeTiled {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// A map over 16-bit elements: dims and box innermost first, strides[i] the
// bytes between elements of dimension i + 1. The box's rows are 128 bytes,
// stored with the 128-byte swizzle; what lies outside reads as zero.
inline int tensormap_16bit(CUtensorMap *map, int dtype, int rank, const void *base, const uint64_t *dims,
                           const uint64_t *strides, const uint32_t *box, std::string &err) {
  const EncodeTiled enc = tensormap_encoder();
  if (!enc) {
    err = "cuTensorMapEncodeTiled is not available";
    return T2SC_ERR_CUDA;
  }
  cuuint64_t d[5], s[5];
  cuuint32_t b[5], one[5];
  for (int i = 0; i < rank; i++) d[i] = dims[i], b[i] = box[i], one[i] = 1;
  for (int i = 0; i + 1 < rank; i++) s[i] = strides[i];
  const CUresult r = enc(map, dtype == T2SC_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         (cuuint32_t)rank, const_cast<void *>(base), d, s, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    err = "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")";
    return T2SC_ERR_CUDA;
  }
  return T2SC_OK;
}

}  // namespace t2sc
