// Tensor maps of 16-bit tensors, made through the driver's entry point.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "pa_common.cuh"

namespace pa {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
                   ? (EncodeTiled)p : (EncodeTiled) nullptr;
    }();
    return fn;
}

// A map of 16-bit elements whose boxes are 64 elements wide and land 128-byte-swizzled; elements outside the tensor read as zero.
// sizes and box in elements, innermost first; strides in elements, of the dimensions behind the first.
inline bool make_map(CUtensorMap* map, int dtype, const void* base, int rank, const long long* sizes, const long long* strides, const int* box) {
    cuuint64_t dims[4], pitch[3];
    cuuint32_t b[4], one[4] = {1, 1, 1, 1};
    for (int i = 0; i < rank; ++i) { dims[i] = (cuuint64_t)sizes[i]; b[i] = (cuuint32_t)box[i]; }
    for (int i = 0; i + 1 < rank; ++i) pitch[i] = (cuuint64_t)strides[i] * 2;
    const EncodeTiled encode = encode_tiled();
    return encode && encode(map, dtype == PA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void*>(base),
                            dims, pitch, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace pa
