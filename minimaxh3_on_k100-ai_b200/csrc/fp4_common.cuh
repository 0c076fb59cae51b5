// Microscaled 4-bit floating point: formats, layout and block-scaled tcgen05 wrappers.
//
// A matrix [rows, cols] is held as
//   codes  [rows, ceil(cols/32)*16] bytes: e2m1 codes, element 2i in the low nibble of
//          byte i, 2i+1 in the high one; columns past `cols` are zero codes
//   scales [ceil(rows/128), ceil(blocks/4), 512] bytes, blocks = ceil(cols/BLOCK): the
//          scale of (row r, block b) is byte (r%32)*16 + (r%128)/32*4 + b%4 of chunk
//          [r/128][b/4].  A chunk is what one tcgen05.cp.32x128b.warpx4 moves to tensor
//          memory (row r%32 + 32j of the tile in lane r%32, column j), so the product
//          copies scales as they lie; blocks past the last one hold 0 and rows past the
//          last one are never read into a result.
// mxfp4: blocks of 32, scale 2^(byte-127) (byte 255: NaN).  nvfp4: blocks of 16, scale an
// unsigned e4m3 (byte 127: NaN) times one power of two of the whole tensor.
#pragma once

#include <cuda.h>
#include <stdint.h>

#include "h3_abi_util.h"
#include "sm100_ptx.cuh"

namespace h3 {
namespace fp4 {

constexpr int MX = H3_MXFP4, NV = H3_NVFP4;
constexpr int CHUNK = 512;                       // bytes of 128 rows x 4 blocks of scales
__host__ __device__ constexpr int block_of(int fmt) { return fmt == MX ? 32 : 16; }

inline int64_t code_pitch(int64_t cols) { return (cols + 31) / 32 * 16; }
inline int64_t scale_chunks(int fmt, int64_t cols) {
    const int64_t blocks = (cols + block_of(fmt) - 1) / block_of(fmt);
    return (blocks + 3) / 4;
}

// codes and scales of a [rows, cols] matrix in `fmt`
inline int check_held(const h3_tensor *codes, const h3_tensor *scales, int fmt, int64_t rows, int64_t cols) {
    H3_CHECK(check_desc(codes, H3_U8));
    H3_CHECK(check_desc(scales, H3_U8));
    if (fmt != MX && fmt != NV) return H3_ERR_UNSUPPORTED;
    if (codes->ndim != 2 || codes->shape[0] != rows || codes->shape[1] != code_pitch(cols)) return H3_ERR_BAD_SHAPE;
    if (scales->ndim != 3 || scales->shape[0] != (rows + 127) / 128 || scales->shape[1] != scale_chunks(fmt, cols) ||
        scales->shape[2] != CHUNK)
        return H3_ERR_BAD_SHAPE;
    if (rows == 0) return H3_OK;
    if (codes->strides[1] != 1 || !aligned16(codes->data) || !aligned16(scales->data)) return H3_ERR_BAD_LAYOUT;
    if (rows > 1 && (codes->strides[0] % 16 != 0 || codes->strides[0] < codes->shape[1])) return H3_ERR_BAD_LAYOUT;
    if (scales->strides[2] != 1 || (scales->shape[1] > 1 && scales->strides[1] != CHUNK) ||
        (scales->shape[0] > 1 && scales->strides[0] != CHUNK * scales->shape[1]))
        return H3_ERR_BAD_LAYOUT;
    return H3_OK;
}

// a power of two that keeps block scale times tensor scale a normal fp32 number
inline bool tensor_scale_ok(int fmt, float t) {
    uint32_t u;
    memcpy(&u, &t, 4);
    if (fmt == MX) return u == 0x3f800000u;
    return (u & 0x807fffffu) == 0 && t >= 0x1p-64f && t <= 0x1p64f;
}

}  // namespace fp4
}  // namespace h3
