// Host-side construction of TMA tensor maps.  cuTensorMapEncodeTiled is a
// driver entry point; it is resolved once through cudaGetDriverEntryPoint so the
// library does not link libcuda directly.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

#include "../../include/h3_b200.h"

namespace h3 {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

// The driver's call wants the device's context current.  A thread that has only allocated
// from a pool and not launched anything has none yet; choosing its device again binds it
// (which a stream capture allows).
template <typename... Args>
inline int encode_tiled(CUtensorMap *map, Args... args) {
    const EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return H3_ERR_DRIVER;
    CUresult r = fn(map, args...);
    if (r != CUDA_SUCCESS && r != CUDA_ERROR_INVALID_VALUE) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) {
            cudaGetLastError();
            return H3_ERR_DRIVER;
        }
        r = fn(map, args...);
    }
    return r == CUDA_SUCCESS ? H3_OK : r == CUDA_ERROR_INVALID_VALUE ? H3_ERR_BAD_LAYOUT : H3_ERR_DRIVER;
}

// BF16 tensor map with 128-byte swizzle.  dims/strides innermost first; strides
// in bytes for dims 1..rank-1; box innermost first.  Returns H3 status.
inline int make_tmap_bf16(CUtensorMap *map, void *base, int rank, const cuuint64_t *dims,
                          const cuuint64_t *strides_bytes, const cuuint32_t *box) {
    cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, base, dims, strides_bytes, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// The same for a matrix of bytes [rows, width] with rows `pitch` bytes apart.
inline int make_tmap_bytes(CUtensorMap *map, void *base, uint64_t width, uint64_t rows, uint64_t pitch,
                           uint32_t box_width, uint32_t box_rows) {
    const cuuint64_t dims[2] = {width, rows};
    const cuuint64_t strides[1] = {pitch};
    const cuuint32_t box[2] = {box_width, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Rows of `width` contiguous bytes (a multiple of 16), moved in boxes of box_bytes (at
// most 2048) x box_rows without swizzle.  Elements are 8 bytes: a box is at most 256 wide.
inline int make_tmap_words(CUtensorMap *map, const void *base, uint64_t width, uint64_t rows, uint32_t box_bytes,
                           uint32_t box_rows) {
    const cuuint64_t dims[2] = {width / 8, rows};
    const cuuint64_t strides[1] = {width};
    const cuuint32_t box[2] = {box_bytes / 8, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_INT64, 2, const_cast<void *>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

}  // namespace h3
