// Host-side construction of TMA tensor maps (CUtensorMap) through the driver entry point, so the
// extension needs no link-time dependency on libcuda.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <ATen/core/Tensor.h>
#include <c10/util/Exception.h>

namespace snb_host {

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    TORCH_CHECK(e == cudaSuccess && q == cudaDriverEntryPointSuccess && p != nullptr,
                "cuTensorMapEncodeTiled entry point unavailable");
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

// Whether a matrix of 16-bit elements can be mapped as it is: contiguous rows on 16-byte boundaries that do not overlap.
inline bool is_mappable(const at::Tensor& x) {
  return x.stride(1) == 1 && x.stride(0) % 8 == 0 && x.stride(0) >= x.size(1) &&
         reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
}
// The matrix, or a copy that can be mapped. A clone, since contiguous() keeps what counts as contiguous already: a
// tensor off the boundaries, or a single row whatever its stride says.
inline at::Tensor mappable(const at::Tensor& x) {
  return is_mappable(x) ? x : x.clone(at::MemoryFormat::Contiguous);
}

// 2D tiled map over a row-major matrix: `inner` elements per row (contiguous), `outer` rows,
// `row_bytes` pitch. Box = box_inner x box_outer elements. Out-of-range elements read as zero.
inline CUtensorMap make_tmap_2d(const void* base, CUtensorMapDataType dt, uint64_t inner, uint64_t outer,
                                uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer,
                                CUtensorMapSwizzle swizzle) {
  TORCH_CHECK((reinterpret_cast<uintptr_t>(base) & 15) == 0, "TMA base must be 16-byte aligned");
  TORCH_CHECK(row_bytes % 16 == 0, "TMA row pitch must be a multiple of 16 bytes, got ", row_bytes);
  CUtensorMap m;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {row_bytes};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = encode_fn()(&m, dt, 2, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", (int)r);
  return m;
}

}  // namespace snb_host
