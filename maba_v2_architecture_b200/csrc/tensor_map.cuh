// Host side of the tensor-memory loads: tiled maps of 16-bit matrices with the 128-byte
// swizzle that the tcgen05 operand descriptors read.
#pragma once
#include "common.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

namespace maba {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_fn() {
    static EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) !=
                cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// rank-R tiled map of 16-bit (or float32) elements; strides in elements (R-1 of them).  The
// swizzle is the inner box's width, 128 or 64 bytes.
inline bool make_map(CUtensorMap* m, int dtype, const void* ptr, int rank, const int64_t* dims, const int64_t* strides,
                     const uint32_t* box) {
    EncodeTiled fn = encode_fn();
    if (fn == nullptr) return false;
    const int el = dtype == MABA_F32 ? 4 : 2;
    cuuint64_t gd[5], gs[4];
    cuuint32_t bx[5], es[5];
    for (int i = 0; i < rank; ++i) {
        gd[i] = (cuuint64_t)dims[i];
        bx[i] = box[i];
        es[i] = 1;
        if (i + 1 < rank) gs[i] = (cuuint64_t)strides[i] * el;
    }
    const CUresult r =
        fn(m,
           dtype == MABA_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
           : dtype == MABA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
           (cuuint32_t)rank, const_cast<void*>(ptr), gd, gs, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
           box[0] * el == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS;
}

inline bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool s16(int64_t stride_elems) { return ((stride_elems * 2) % 16) == 0 && stride_elems > 0; }

}  // namespace maba
