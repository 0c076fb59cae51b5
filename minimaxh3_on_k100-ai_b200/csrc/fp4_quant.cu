// Microscaled 4-bit quantisation of BF16 rows and its inverse (layout: fp4_common.cuh).
//
//   mxfp4  e = clamp(floor(log2 amax) - 2, -127, 127), scale 2^e   (block of 32)
//   nvfp4  s = e4m3(amax / (6 t)), scale s t                       (block of 16)
//   code   = e2m1 nearest-even of x / scale, at most 6 in magnitude
// A block that holds an infinity or a NaN gets the NaN scale, so what is wrong stays
// visible; a block whose scale rounds to zero gets zero codes.
//
// Every element is read once and written once: HBM-bound, 2 B in and 0.5 B + 1/block out
// per element.  A thread owns 16 consecutive columns of a row (two 16-byte loads, one
// 8-byte store of codes); an nvfp4 block is one thread's, an mxfp4 block two neighbours'.
// The four scales of a chunk word are gathered by shuffle and stored as one word.
#include <math.h>
#include <string.h>

#include "fp4_common.cuh"
#include "h3_common.cuh"

namespace h3 {
namespace fp4 {

constexpr int THREADS = 256;

struct Shape {
    int64_t rows;
    int cols, units;                     // units: 16-column pieces of a row, whole chunks
    int code_units;                      // 16-column pieces of the code pitch
    int log_tx;                          // threads along a row (power of two)
    int chunks;                          // scale chunks along a row
    int64_t ldx, ldc;                    // row strides: x in elements, codes in bytes
    TensorScale ts;
};

// Rows that 16-byte accesses do not fit (odd widths): the tx threads of a row move its
// segment of 16 tx elements between global and shared memory by neighbouring 4-byte words
// instead of each its own unit 32 bytes away from the next thread's (187 -> 21 us to read
// back 18944 x 1795).  The copy in shared memory starts at element `a` (0 or 1) of its
// space, so that its words are the row's words; n elements exist.
constexpr int SEG_PAD = 8;               // elements between the segments of a block's rows

__device__ __forceinline__ int odd_start(const void *p) { return (int)(reinterpret_cast<uintptr_t>(p) >> 1) & 1; }

__device__ __forceinline__ void load_segment(uint16_t *seg, const __nv_bfloat16 *src, int a, int n, int t, int tx) {
    const uint16_t *p = reinterpret_cast<const uint16_t *>(src);
    const uint32_t *words = reinterpret_cast<const uint32_t *>(p - a);      // word k: elements 2k - a, 2k - a + 1
    uint32_t *dst = reinterpret_cast<uint32_t *>(seg);
    uint32_t v[8];
    const int inside = (n + a) / 2;      // words [a, inside) lie within the row
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int k = t + i * tx;
        if (k >= a && k < inside) v[i] = words[k];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int k = t + i * tx;
        if (k >= a && k < inside) dst[k] = v[i];
    }
    if (t == 0) {
        if (a) seg[1] = p[0];
        if ((n + a) & 1) seg[n - 1 + a] = p[n - 1];
    }
}
// one thread's 16 elements of the copy
__device__ __forceinline__ void read_unit(const uint16_t *seg, int a, int t, uint32_t (&w)[8]) {
    const uint4 *at = reinterpret_cast<const uint4 *>(seg + t * UNIT);
    const uint4 x = at[0], y = at[1];
    const uint32_t v[9] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w, reinterpret_cast<const uint32_t *>(at + 2)[0]};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], 16 * a);
}
__device__ __forceinline__ void write_unit(uint16_t *seg, int a, int t, const uint32_t (&w)[8]) {
    if (a == 0) {
        uint4 *at = reinterpret_cast<uint4 *>(seg + t * UNIT);
        at[0] = make_uint4(w[0], w[1], w[2], w[3]);
        at[1] = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
        uint32_t *at = reinterpret_cast<uint32_t *>(seg + t * UNIT);
        seg[t * UNIT + 1] = (uint16_t)w[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) at[i] = __funnelshift_r(w[i - 1], w[i], 16);
        seg[t * UNIT + 16] = (uint16_t)(w[7] >> 16);
    }
}
__device__ __forceinline__ void store_segment(__nv_bfloat16 *dst, const uint16_t *seg, int a, int n, int t, int tx) {
    uint16_t *p = reinterpret_cast<uint16_t *>(dst);
    uint32_t *words = reinterpret_cast<uint32_t *>(p - a);
    const uint32_t *src = reinterpret_cast<const uint32_t *>(seg);
    const int inside = (n + a) / 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int k = t + i * tx;
        if (k >= a && k < inside) words[k] = src[k];
    }
    if (t == 0) {
        if (a) p[0] = seg[1];
        if ((n + a) & 1) p[n - 1] = seg[n - 1 + a];
    }
}

template <int FMT, bool VEC>
__global__ void __launch_bounds__(THREADS)
    quantize_kernel(const __nv_bfloat16 *x, uint8_t *codes, uint8_t *scales, Shape s) {
    // in this order: a product behind this kernel reads its weights ahead of the wait for x,
    // so nothing before this kernel may still be running when that product starts
    wait_for_previous();
    release_next();
    const int tx = 1 << s.log_tx;
    const int unit = (int)blockIdx.y * tx + (int)(threadIdx.x & (tx - 1));
    const int64_t row = (int64_t)blockIdx.x * (THREADS >> s.log_tx) + (threadIdx.x >> s.log_tx);
    const bool live = row < s.rows && unit < s.units;
    uint32_t w[8] = {};
    if (VEC) {
        if (live) load_unit<true>(x + row * s.ldx, unit * UNIT, s.cols, w);
    } else {
        __shared__ __align__(16) uint16_t seg[THREADS * (UNIT + 1)];
        const int t = threadIdx.x & (tx - 1), col0 = (int)blockIdx.y * tx * UNIT, n = min(tx * UNIT, s.cols - col0);
        uint16_t *mine = seg + (threadIdx.x >> s.log_tx) * (tx * UNIT + SEG_PAD);   // this row's segment
        const __nv_bfloat16 *src = x + row * s.ldx + col0;
        const int a = odd_start(src);
        if (row < s.rows && n > 0) load_segment(mine, src, a, n, t, tx);
        __syncthreads();
        read_unit(mine, a, t, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = t * UNIT + 2 * i;
            if (!live || e >= n) w[i] = 0;
            else if (e + 1 >= n) w[i] &= 0xffffu;
        }
    }

    uint32_t byte, c[2];
    quantize_unit<FMT>(w, s.ts, c, byte);
    if (live && unit < s.code_units)
        *reinterpret_cast<uint2 *>(codes + row * s.ldc + unit * (UNIT / 2)) = make_uint2(c[0], c[1]);

    const uint32_t word = scale_word<FMT>(byte);
    constexpr int STEP = FMT == MX ? 2 : 1;
    if (live && unit % (4 * STEP) == 0) {
        const int64_t chunk = (row >> 7) * s.chunks + unit / (4 * STEP);
        *reinterpret_cast<uint32_t *>(scales + chunk * CHUNK + (row & 31) * 16 + ((row >> 5) & 3) * 4) = word;
    }
}

// the values of a unit as packed BF16 pairs
template <int FMT>
__device__ __forceinline__ void value_unit(const uint8_t *codes, const uint8_t *scales, const Shape &s, int64_t row,
                                           int unit, uint32_t (&w)[8]) {
    const uint2 c = *reinterpret_cast<const uint2 *>(codes + row * s.ldc + unit * (UNIT / 2));
    const int block = FMT == MX ? unit >> 1 : unit;
    const uint32_t byte = scales[((row >> 7) * s.chunks + (block >> 2)) * CHUNK + (row & 31) * 16 +
                                 ((row >> 5) & 3) * 4 + (block & 3)];
    float scale;
    if (FMT == MX) scale = byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte == 0 ? 1u << 22 : byte << 23);
    else scale = from_e4m3(byte) * s.ts.t;      // cvt makes byte 127 a NaN
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = ((i < 4 ? c.x : c.y) >> (8 * (i & 3))) & 0xffu;
        uint32_t h;
        asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(b));
        const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&h));
        // 2 significant bits times 4: exact in BF16 where the tensor scale is a power of two
        w[i] = bf2u(__floats2bfloat162_rn(f.x * scale, f.y * scale));
    }
}

template <int FMT, bool VEC>
__global__ void __launch_bounds__(THREADS)
    dequantize_kernel(__nv_bfloat16 *y, const uint8_t *codes, const uint8_t *scales, Shape s) {
    const int tx = 1 << s.log_tx;
    const int unit = (int)blockIdx.y * tx + (int)(threadIdx.x & (tx - 1));
    const int64_t row = (int64_t)blockIdx.x * (THREADS >> s.log_tx) + (threadIdx.x >> s.log_tx);
    const int col = unit * UNIT;
    wait_for_previous();
    const bool live = row < s.rows && col < s.cols;
    if (VEC && !live) return;
    uint32_t w[8];
    if (live) value_unit<FMT>(codes, scales, s, row, unit, w);
    if (VEC) {
        __nv_bfloat16 *dst = y + row * s.ldx + col;
        if (col + UNIT <= s.cols) {
            reinterpret_cast<uint4 *>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4 *>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
            uint16_t *p = reinterpret_cast<uint16_t *>(dst);
#pragma unroll
            for (int i = 0; i < UNIT; ++i)
                if (col + i < s.cols) p[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        }
    } else {
        __shared__ __align__(16) uint16_t seg[THREADS * (UNIT + 1)];
        const int t = threadIdx.x & (tx - 1), col0 = (int)blockIdx.y * tx * UNIT, n = min(tx * UNIT, s.cols - col0);
        uint16_t *mine = seg + (threadIdx.x >> s.log_tx) * (tx * UNIT + SEG_PAD);
        __nv_bfloat16 *dst = y + row * s.ldx + col0;
        const int a = odd_start(dst);
        if (live) write_unit(mine, a, t, w);
        __syncthreads();
        if (row < s.rows && n > 0) store_segment(dst, mine, a, n, t, tx);
    }
}

// Shared checks and launch shape; `x` is the BF16 side.
int plan(const h3_tensor *x, const h3_tensor *codes, const h3_tensor *scales, int fmt, float tensor_scale, Shape *s,
         dim3 *grid, bool *vec) {
    H3_CHECK(check_bf16(x));
    if (x->ndim != 2 || x->shape[1] < 1) return H3_ERR_BAD_SHAPE;
    H3_CHECK(check_held(codes, scales, fmt, x->shape[0], x->shape[1]));
    if (!held_scale_ok(fmt, tensor_scale)) return H3_ERR_UNSUPPORTED;
    if (x->shape[0] > 0x7fffffffLL || x->shape[1] > (1 << 24)) return H3_ERR_UNSUPPORTED;
    if (x->shape[0] == 0) return H3_OK;
    if ((x->shape[1] > 1 && x->strides[1] != 1) || (x->shape[0] > 1 && x->strides[0] < 0)) return H3_ERR_BAD_LAYOUT;
    s->rows = x->shape[0];
    s->cols = (int)x->shape[1];
    s->chunks = (int)scales->shape[1];
    s->units = s->chunks * (fmt == MX ? 8 : 4);
    s->code_units = (int)codes->shape[1] / (UNIT / 2);
    s->ldx = x->shape[0] > 1 ? x->strides[0] : 0;
    s->ldc = x->shape[0] > 1 ? codes->strides[0] : 0;
    s->ts = TensorScale::make(tensor_scale);
    // threads along a row: enough for short rows, at most 64 so that long rows waste few
    s->log_tx = 3;
    while (s->log_tx < 6 && (1 << s->log_tx) < s->units) ++s->log_tx;
    const int ty = THREADS >> s->log_tx;
    *grid = dim3((unsigned)((s->rows + ty - 1) / ty), (unsigned)((s->units + (1 << s->log_tx) - 1) >> s->log_tx));
    *vec = aligned16(x->data) && s->ldx % 8 == 0;
    return H3_OK;
}

template <typename Kernel, typename... Args>
int launch(Kernel kernel, dim3 grid, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr = overlapped_launch();
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
        cudaGetLastError();
        return H3_ERR_LAUNCH;
    }
    return launch_status();
}

int quantize(const h3_tensor *codes, const h3_tensor *scales, const h3_tensor *x, int fmt, float tensor_scale,
             cudaStream_t stream) {
    Shape s{};
    dim3 grid;
    bool vec;
    H3_CHECK(plan(x, codes, scales, fmt, tensor_scale, &s, &grid, &vec));
    if (!tensor_scale_ok(fmt, tensor_scale)) return H3_ERR_UNSUPPORTED;
    if (x->shape[0] == 0) return H3_OK;
    auto kernel = fmt == MX ? (vec ? quantize_kernel<MX, true> : quantize_kernel<MX, false>)
                            : (vec ? quantize_kernel<NV, true> : quantize_kernel<NV, false>);
    return launch(kernel, grid, stream, static_cast<const __nv_bfloat16 *>(x->data),
                  static_cast<uint8_t *>(codes->data), static_cast<uint8_t *>(scales->data), s);
}

}  // namespace fp4
}  // namespace h3

using namespace h3;

extern "C" int h3_quantize_fp4(const h3_tensor *codes, const h3_tensor *scales, const h3_tensor *x, int32_t format,
                               float tensor_scale, void *stream) {
    return fp4::quantize(codes, scales, x, format, tensor_scale, (cudaStream_t)stream);
}

extern "C" int h3_dequantize_fp4(const h3_tensor *y, const h3_tensor *codes, const h3_tensor *scales, int32_t format,
                                 float tensor_scale, void *stream) {
    fp4::Shape s{};
    dim3 grid;
    bool vec;
    H3_CHECK(fp4::plan(y, codes, scales, format, tensor_scale, &s, &grid, &vec));
    if (y->shape[0] == 0) return H3_OK;
    if (y->shape[0] > 1 && y->strides[0] < y->shape[1]) return H3_ERR_BAD_LAYOUT;   // rows would overlap
    auto kernel = format == fp4::MX ? (vec ? fp4::dequantize_kernel<fp4::MX, true> : fp4::dequantize_kernel<fp4::MX, false>)
                                    : (vec ? fp4::dequantize_kernel<fp4::NV, true> : fp4::dequantize_kernel<fp4::NV, false>);
    return fp4::launch(kernel, grid, (cudaStream_t)stream, static_cast<__nv_bfloat16 *>(y->data),
                       static_cast<const uint8_t *>(codes->data), static_cast<const uint8_t *>(scales->data), s);
}
