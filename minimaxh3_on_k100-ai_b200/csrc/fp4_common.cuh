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
// unsigned e4m3 (byte 127: NaN) times one number of the whole tensor, a power of two where
// the quantisation is done here.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <string.h>

#include "h3_abi_util.h"
#include "h3_common.cuh"
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

// the scale of a matrix that is held: block scale times tensor scale is a normal fp32 number
inline bool held_scale_ok(int fmt, float t) { return fmt == MX ? t == 1.0f : t >= 0x1p-64f && t <= 0x1p64f; }
// of one that is quantised: a power of two
inline bool tensor_scale_ok(int fmt, float t) {
    uint32_t u;
    memcpy(&u, &t, 4);
    return held_scale_ok(fmt, t) && (u & 0x007fffffu) == 0;
}

// ---------------------------------------------------------------------------
// quantisation of 16 columns by one thread
// ---------------------------------------------------------------------------
constexpr int UNIT = 16;

struct TensorScale {
    float t, sixth;              // a power of two, and 1 / (6 t)
    __host__ static TensorScale make(float t) { return {t, 1.0f / (6.0f * t)}; }
};
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 columns of a row as packed BF16 pairs, zeros past the end
template <bool VEC>
__device__ __forceinline__ void load_unit(const __nv_bfloat16 *row, int col, int cols, uint32_t (&w)[8]) {
    if (VEC && col + UNIT <= cols) {
        const uint4 a = reinterpret_cast<const uint4 *>(row + col)[0];
        const uint4 b = reinterpret_cast<const uint4 *>(row + col)[1];
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
    } else {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t lo = col + 2 * i < cols ? p[col + 2 * i] : 0;
            const uint32_t hi = col + 2 * i + 1 < cols ? p[col + 2 * i + 1] : 0;
            w[i] = lo | (hi << 16);
        }
    }
}

// two e2m1 codes: `lo` in the low nibble
__device__ __forceinline__ uint32_t e2m1x2(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}"
        : "=r"(r)
        : "f"(hi), "f"(lo));
    return r;
}

// e4m3 of v >= 0, at most 448.  Through fp16: where v is the quotient of an 8-bit amax and
// 6 t, known to a few units of fp32, its 11 bits put a quotient that lies half way between
// two e4m3 numbers (5 significant bits) exactly there, and any other, at least 2^-8 of
// itself away, on its side.
__device__ __forceinline__ uint32_t e4m3(float v) {
    uint16_t r;
    asm("{\n\t.reg .b32 h;\n\tcvt.rn.f16x2.f32 h, %1, %2;\n\tcvt.rn.satfinite.e4m3x2.f16x2 %0, h;\n\t}"
        : "=h"(r)
        : "f"(0.f), "f"(fminf(v, 448.f)));
    return r & 0xffu;
}
__device__ __forceinline__ float from_e4m3(uint32_t b) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)b));
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffff)));
}

// Codes (8 bytes) and scale byte of a unit; an mxfp4 block is this lane's unit and its
// neighbour's (lane ^ 1), so all lanes of the warp take part.
template <int FMT>
__device__ __forceinline__ void quantize_unit(const uint32_t (&w)[8], const TensorScale &ts, uint32_t (&c)[2],
                                              uint32_t &byte) {
    // magnitudes order as integers; at 0x7f80 and above they are infinite or NaN
    uint32_t top2 = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top2 = __vmaxu2(top2, w[i] & 0x7fff7fffu);
    uint32_t top = max(top2 & 0xffffu, top2 >> 16);
    if (FMT == MX) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const bool bad = top >= 0x7f80u;
    c[0] = c[1] = 0;
    if (FMT == MX) {
        // the exponent field of amax is floor(log2 amax) + 127 (0 below the normals)
        const int e = (int)(top >> 7) - 2;
        byte = bad ? 255u : (uint32_t)max(e, 0);
        const float inv = __uint_as_float((254u - byte) << 23);      // 2^(127 - byte), exact
        if (!bad) {
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i >> 2] |= e2m1x2(blo(w[i]) * inv, bhi(w[i]) * inv) << (8 * (i & 3));
        }
    } else {
        const float amax = __uint_as_float(top << 16);
        byte = bad ? 127u : e4m3(amax * ts.sixth);
        if (!bad && byte != 0) {
            // x / scale lies on a border between two codes, a multiple of 1/4, or (x has 8
            // significant bits, the scale 4) at least 1/300 of it away.  Adding and taking
            // away 1.5 * 2^11 rounds the product with the (approximate) reciprocal to a multiple
            // of 2^-12, which puts the first kind exactly on its border and moves none across.
            const float r = rcp(from_e4m3(byte) * ts.t);
            constexpr float SNAP = 1.5f * 2048.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                c[i >> 2] |= e2m1x2(__fadd_rn(__fmaf_rn(blo(w[i]), r, SNAP), -SNAP),
                                    __fadd_rn(__fmaf_rn(bhi(w[i]), r, SNAP), -SNAP))
                             << (8 * (i & 3));
        }
    }
}

// The four scales of a chunk's word, gathered from the 4 (nvfp4) or 8 (mxfp4, each twice)
// lanes that hold them; valid in the first of those.
template <int FMT>
__device__ __forceinline__ uint32_t scale_word(uint32_t byte) {
    constexpr int STEP = FMT == MX ? 2 : 1;
    uint32_t word = byte | (__shfl_down_sync(0xffffffffu, byte, STEP) << 8);
    return word | __shfl_down_sync(0xffffffffu, word, 2 * STEP) << 16;
}

}  // namespace fp4
}  // namespace h3
