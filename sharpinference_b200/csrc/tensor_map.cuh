// Host-side creation of TMA tensor maps.  The driver's encoder is looked up through the runtime
// (cudaGetDriverEntryPoint), so the kernel libraries do not link against libcuda.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tmap {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(ptr);
    }
    return fn;
}

// bf16 tensor [d2, d1, d0] (d0 innermost and contiguous; d2 == 0 makes it two-dimensional), box
// [1, box1, box0] with box0 * 2 bytes == 128, 128-byte swizzle, out-of-range elements read as zero.
inline bool make_bf16_map(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint32_t box0,
                          uint32_t box1) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const bool three = d2 > 0;
    cuuint64_t dims[3] = {d0, d1, three ? d2 : 1};
    cuuint64_t strides[2] = {d0 * 2, d0 * d1 * 2};
    cuuint32_t box[3] = {box0, box1, 1};
    cuuint32_t elem[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, three ? 3 : 2, const_cast<void*>(base), dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// bf16 tensor [d2][d1][ld], of which the first d0 of every ld elements are read (ld a multiple of 8): boxes of [box2, 1, box0],
// 128-byte swizzle as above, out-of-range elements read as zero.
inline bool make_bf16_rows_map(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t ld, uint32_t box0,
                               uint32_t box2) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    cuuint64_t dims[3] = {d0, d1, d2};
    cuuint64_t strides[2] = {ld * 2, d1 * ld * 2};
    cuuint32_t box[3] = {box0, 1, box2};
    cuuint32_t elem[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 8-bit tensor [d2][d1][d0] with rows ld bytes apart (a multiple of 16) and d1 * ld between the outermost (d2 == 0 makes it
// two-dimensional): boxes of [1, box1, 128], 128-byte swizzle, out-of-range elements read as zero.
inline bool make_u8_map(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t ld, uint32_t box1) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const bool three = d2 > 0;
    cuuint64_t dims[3] = {d0, d1, three ? d2 : 1};
    cuuint64_t strides[2] = {ld, d1 * ld};
    cuuint32_t box[3] = {128, box1, 1};
    cuuint32_t elem[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, three ? 3 : 2, const_cast<void*>(base), dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace tmap
