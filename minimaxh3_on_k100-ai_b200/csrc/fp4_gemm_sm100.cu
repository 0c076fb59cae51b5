// Projections with microscaled 4-bit operands on tcgen05's block-scaled MMA (sm_100a):
//
//   y[m][n] = bf16( t * sum_k xq[m][k] wq[n][k] + bias[n] ),   fp32 accumulation,
//
// xq and wq in one format (layout: fp4_common.cuh), t the product of their tensor scales.
// The tensor core multiplies the codes, applies both block scales and adds in fp32, so
// nothing is widened in memory: a product reads K/2 + K/block bytes per row.
//
// swap form: the weight's rows are the M = 128 side of the MMA and BN rows of x the N
// side, so a few tokens cost N = 16 columns, not a 128-row tile.  A CTA owns one tile; a
// cluster of up to 8 CTAs splits K, each CTA leaves its fp32 tile in shared memory and
// sums its share of the columns over the cluster in rank order (fixed order, no atomics,
// no scratch in global memory).  Bound by reading the weights (HBM).
//
// For up to 8 rows the same kernel can quantise x itself: four more warps write this CTA's
// share of x to the ring, which saves a launch and the scratch.  nvfp4, back to back in a
// graph: 1 x 15360 x 5120 11.8 us against 12.8 with the quantisation before it, 4 rows 12.3
// against 12.6, 8 rows 13.1 against 12.8 (there it is the second launch's host time that is
// saved); 16 rows would take 16.9 against 13.0.
//
// tile form: persistent CTA pairs (cta_group::2), 256 x 256 output tiles, K in tiles of 256
// (one 128-byte swizzle span of codes) through a 5-slot TMA ring.  Each CTA loads its 128 x
// rows, half the tile's w rows, and the scales of its x rows and of all the w rows; the
// leader copies both CTAs' scales to tensor memory and issues the MMAs.  Two accumulators
// of 256 columns and the scales do not fit the 512 columns, so the accumulators share 128:
// the epilogue reads those first and then lets the next tile start, so all but that read
// overlaps the next tile's products.
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "fp4_common.cuh"
#include "h3_abi_util.h"
#include "h3_common.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.h"

namespace h3 {
namespace fp4 {

int quantize(const h3_tensor *codes, const h3_tensor *scales, const h3_tensor *x, int fmt, float tensor_scale,
             cudaStream_t stream);

constexpr int BK = 256;                          // columns per K tile: one 128-byte swizzle span
constexpr int KSTEP = 64;                        // columns per MMA
__host__ __device__ constexpr int tile_chunks(int fmt) { return fmt == MX ? 2 : 4; }   // scale chunks per K tile

struct Params {
    int M, N;                    // rows of x, rows of w
    int ktiles, chunks, ksteps;  // along K: tiles, scale chunks, MMAs
    const uint8_t *sx, *sw;      // scales
    __nv_bfloat16 *y;
    int64_t ldy;
    const __nv_bfloat16 *bias;   // may be null
    float t;
    int num_m, num_n;            // tiles
    int wide;                    // 4-column (8-byte) stores allowed; tile form: stores through TMA
    int dependent;               // launched behind the quantisation of x: w may be read before that ends
    // fused quantisation: x itself
    const __nv_bfloat16 *x;
    int64_t ldx;
    int cols, x_vec;             // x_vec: 16-byte loads of x allowed
    TensorScale x_scale;
};

template <int FMT, int BN>
struct Swap {
    static constexpr int CH = tile_chunks(FMT);
    static constexpr int A_BYTES = 128 * 128;                 // 128 weight rows
    static constexpr int B_BYTES = BN * 128;
    static constexpr int SF_BYTES = CH * CHUNK;
    static constexpr int STAGE = A_BYTES + B_BYTES + 2 * SF_BYTES;
    static constexpr int STAGE_PAD = (STAGE + 1023) / 1024 * 1024;
    static constexpr int RING_SPACE = 110 * 1024;                 // two CTAs per SM
    static constexpr int STAGES = RING_SPACE / STAGE_PAD;
    static constexpr int RED_BYTES = BN * 128 * 4;            // the fp32 tile, in the ring's place
    static constexpr int OFF_BAR = STAGES * STAGE_PAD > RED_BYTES ? STAGES * STAGE_PAD : RED_BYTES;
    static constexpr int SMEM = OFF_BAR + (2 * STAGES + 1) * 8 + 16 + 1024;
    static constexpr int SF_COLS = CH * 4;                    // tensor memory columns of one operand's scales
    static constexpr int SF_COL0 = BN < 32 ? 32 : BN;         // behind the accumulator
    static constexpr uint32_t TMEM = SF_COL0 + 4 * SF_COLS <= 128 ? 128 : 256;
    static_assert(SF_COL0 + 4 * SF_COLS <= (int)TMEM, "tensor memory");
    static_assert(STAGES >= 3, "ring");
};
constexpr int SWAP_THREADS = 128;
constexpr int QUANT_WARPS = 4;                   // of the fused form
constexpr int FUSED_TILE = 16, FUSED_ROWS = 8;   // of the fused form: x tile, and how many rows it takes

// 16 bytes from CTA `rank`'s shared memory at this CTA's address `addr`
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr, uint32_t rank) {
    float4 v;
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}
__device__ __forceinline__ void ld_shared_words(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_word(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_shared_words(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void st_shared_f32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// grid: x = cluster rank (K share), y = weight row tile, z = x row tile
template <int FMT, int BN, bool FUSED>
__global__ void __launch_bounds__(SWAP_THREADS + (FUSED ? QUANT_WARPS * 32 : 0), 2)
    swap_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw, Params p) {
    using C = Swap<FMT, BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
    uint64_t *empty = full + C::STAGES;
    uint64_t *done = empty + C::STAGES;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = (int)gridDim.x, rank = (int)blockIdx.x;   // the cluster spans grid x
    const int n0 = (int)blockIdx.y * 128, m0 = (int)blockIdx.z * BN;   // m0: a multiple of 128 (0 where BN is smaller)
    const int k_begin = (int)((int64_t)p.ktiles * rank / split), k_end = (int)((int64_t)p.ktiles * (rank + 1) / split);
    const int nk = k_end - k_begin;

    auto load_w = [&](int i) {
        const int slot = i % C::STAGES, kt = k_begin + i, ch = min(C::CH, p.chunks - kt * C::CH);
        uint8_t *st = smem + slot * C::STAGE_PAD;
        if (elect_one()) {
            mbar_expect_tx(&full[slot], C::A_BYTES + ch * CHUNK + (FUSED ? 0 : C::B_BYTES + ch * CHUNK));
            tma_load_2d(st, &tw, &full[slot], kt * 128, n0);
            bulk_load(st + C::A_BYTES + C::B_BYTES, p.sw + ((int64_t)blockIdx.y * p.chunks + kt * C::CH) * CHUNK,
                      ch * CHUNK, &full[slot]);
        }
        __syncwarp();
    };
    // Warp 0 fills the ring with weights before the rest is set up: behind the quantisation
    // of x at once (whatever ran before that kernel is done), else when the kernel before
    // this one has ended.
    const int head = min(nk, C::STAGES);
    if (warp == 0) {
        if (elect_one()) {
            for (int s = 0; s < C::STAGES; ++s) {
                mbar_init(&full[s], FUSED ? 2 : 1);
                mbar_init(&empty[s], 1);
            }
            mbar_init(done, 1);
            *abort_flag = 0;
            fence_mbar_init();
            fence_proxy_async_smem();   // the copies below come before any block barrier
        }
        __syncwarp();
        if (!p.dependent) wait_for_previous();
        for (int i = 0; i < head; ++i) load_w(i);
    } else if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    wait_for_previous();   // every warp: the bounded waits below must not count the previous kernel's time

    if (warp == 0) {
        auto load_x = [&](int i) {
            const int slot = i % C::STAGES, kt = k_begin + i, ch = min(C::CH, p.chunks - kt * C::CH);
            uint8_t *st = smem + slot * C::STAGE_PAD;
            if (FUSED) return;
            if (elect_one()) {
                tma_load_2d(st + C::A_BYTES, &tx, &full[slot], kt * 128, m0);
                bulk_load(st + C::A_BYTES + C::B_BYTES + C::SF_BYTES,
                          p.sx + ((int64_t)(m0 >> 7) * p.chunks + kt * C::CH) * CHUNK, ch * CHUNK, &full[slot]);
            }
            __syncwarp();
        };
        for (int i = 0; i < head; ++i) load_x(i);
        for (int i = head; i < nk; ++i) {
            if (!__all_sync(0xffffffffu, mbar_wait(&empty[i % C::STAGES], (i / C::STAGES - 1) & 1, abort_flag))) break;
            load_w(i);
            load_x(i);
        }
    } else if (warp == 1) {
        const uint32_t base = smem_u32(smem);
        bool ok = true;
        for (int i = 0; i < nk; ++i) {
            const int slot = i % C::STAGES, kt = k_begin + i;
            ok = mbar_wait(&full[slot], (i / C::STAGES) & 1, abort_flag);
            // two scale buffers: the MMAs of tile i - 2 must have read the one about to be overwritten
            if (ok && i >= 2) ok = mbar_wait(&empty[(i - 2) % C::STAGES], ((i - 2) / C::STAGES) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t sa = base + slot * C::STAGE_PAD, sb = sa + C::A_BYTES;
            const uint32_t ssa = sb + C::B_BYTES, ssb = ssa + C::SF_BYTES;
            const uint32_t ta = tmem + C::SF_COL0 + (i & 1) * 2 * C::SF_COLS, tb = ta + C::SF_COLS;
            const int ch = min(C::CH, p.chunks - kt * C::CH);
            const int steps = min(BK / KSTEP, p.ksteps - kt * (BK / KSTEP));
            if (elect_one()) {
#pragma unroll
                for (int c = 0; c < C::CH; ++c) {
                    if (c < ch) {
                        tmem_cp_scales<false>(ta + 4 * c, smem_desc_rows16(ssa + c * CHUNK));
                        tmem_cp_scales<false>(tb + 4 * c, smem_desc_rows16(ssb + c * CHUNK));
                    }
                }
#pragma unroll
                for (int s = 0; s < BK / KSTEP; ++s) {
                    const int c = FMT == MX ? s >> 1 : s;
                    if (s < steps)
                        umma_fp4<FMT == MX, false>(tmem, smem_desc_sw128(sa + s * 32, 16, 1024),
                                                   smem_desc_sw128(sb + s * 32, 16, 1024),
                                                   idesc_fp4(128, BN, FMT == MX, FMT == MX ? (s & 1) * 2 : 0),
                                                   ta + 4 * c, tb + 4 * c, (i > 0 || s > 0) ? 1u : 0u);
                }
                umma_commit(&empty[slot]);
                if (i == nk - 1) umma_commit(done);
            }
            __syncwarp();
        }
        if (!ok) drain_in_flight();
    } else if (FUSED && warp >= 4) {
        // This CTA's share of x in 4 bits, straight to the ring.  A warp takes every fourth K
        // tile whole, 16 lanes to a row; its next tile's columns load while it stores this
        // one's.  Every CTA of a column of tiles repeats this, so it is for a few rows: then
        // it costs less than a launch.
        constexpr int PER = FUSED_ROWS / 2;                  // pairs of rows
        const int half = lane >> 4, unit = lane & 15;
        uint32_t w[PER][8];
        auto load = [&](int i) {
            const int col = (k_begin + i) * BK + unit * UNIT;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const int r = 2 * j + half;
                if (2 * j >= p.M) break;
                if (r < p.M) {
                    const __nv_bfloat16 *row = p.x + (int64_t)r * p.ldx;
                    if (p.x_vec) load_unit<true>(row, col, p.cols, w[j]);
                    else load_unit<false>(row, col, p.cols, w[j]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[j][e] = 0;
                }
            }
        };
        const int first = warp - 4;
        if (first < nk) load(first);
        for (int i = first; i < nk; i += QUANT_WARPS) {
            const int slot = i % C::STAGES;
            uint32_t c[PER][2], word[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (2 * j >= p.M) break;                     // uniform
                uint32_t byte;
                quantize_unit<FMT>(w[j], p.x_scale, c[j], byte);
                word[j] = scale_word<FMT>(byte);
            }
            if (i + QUANT_WARPS < nk) load(i + QUANT_WARPS);
            if (i >= C::STAGES &&
                !__all_sync(0xffffffffu, mbar_wait(&empty[slot], (i / C::STAGES - 1) & 1, abort_flag)))
                break;
            const uint32_t sx = smem_u32(smem) + slot * C::STAGE_PAD + C::A_BYTES, ssx = sx + C::B_BYTES + C::SF_BYTES;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (2 * j >= p.M) break;
                const int r = 2 * j + half;
                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(sx + r * 128 + (((unit >> 1) ^ (r & 7)) << 4) +
                                                                      (unit & 1) * 8),
                             "r"(c[j][0]), "r"(c[j][1])
                             : "memory");
                constexpr int LANES = FMT == MX ? 8 : 4;     // units of a chunk
                if (unit % LANES == 0) st_shared_f32(ssx + unit / LANES * CHUNK + r * 16, word[j]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[slot]);
        }
    }
    __syncwarp();
    const bool ok = nk == 0 || __all_sync(0xffffffffu, mbar_wait(done, 0, abort_flag));
    tc_fence_after();
    // lane = weight row: column c of the tile becomes 128 consecutive floats
    const uint32_t red = smem_u32(smem);
    const int cols = min(BN, p.M - m0);
    if (ok && warp < 4) {
#pragma unroll 1
        for (int c0 = 0; c0 < cols; c0 += 16) {
            uint32_t v[16];
            if (nk > 0) {
                tmem_ld16(tmem + ((uint32_t)(warp * 32) << 16) + c0, v);
                tmem_ld_wait();
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                st_shared_f32(red + ((c0 + i) * 128 + warp * 32 + lane) * 4, nk > 0 ? v[i] : 0u);
        }
    }
    tc_fence_before();
    if (split > 1) cluster_sync();
    else __syncthreads();
    if (ok && warp < 4) {
        const int n = n0 + lane * 4;
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (p.bias) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < p.N) b[e] = __bfloat162float(p.bias[n + e]);
        }
        for (int c = rank * 4 + warp; c < cols; c += split * 4) {
            // all ranks' pieces are requested before the first is needed
            float4 part[8];
#pragma unroll
            for (int r = 0; r < 8; ++r)
                if (r < split) part[r] = ld_cluster_f4(red + (c * 128 + lane * 4) * 4, (uint32_t)r);
            float4 acc = part[0];
#pragma unroll
            for (int r = 1; r < 8; ++r)
                if (r < split) acc.x += part[r].x, acc.y += part[r].y, acc.z += part[r].z, acc.w += part[r].w;
            const float f[4] = {fmaf(acc.x, p.t, b[0]), fmaf(acc.y, p.t, b[1]), fmaf(acc.z, p.t, b[2]),
                                fmaf(acc.w, p.t, b[3])};
            __nv_bfloat16 *dst = p.y + (int64_t)(m0 + c) * p.ldy + n;
            if (p.wide && n + 4 <= p.N) {
                *reinterpret_cast<uint2 *>(dst) = pack4(f);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < p.N) dst[e] = __float2bfloat16_rn(f[e]);
            }
        }
    }
    if (split > 1) cluster_sync();   // no CTA leaves while another reads its tile
    else __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM);
    }
}

// K shares of `tiles` output tiles: as many as run in one wave and have a K tile each, the
// same for a fused product and for one of rows quantised beforehand.  0: cannot be told.
template <int FMT, int BN>
int swap_split(int64_t tiles, int ktiles) {
    using C = Swap<FMT, BN>;
    // Per device: how many clusters of 1..8 CTAs are resident at once.  A cluster stays
    // within one group of SMs, so 8-CTA clusters fill fewer SMs than their number suggests.
    static std::atomic<int> resident[64][9];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return 0;
    if (resident[dev][1].load() == 0) {
        auto plain = swap_kernel<FMT, BN, false>;
        if (cudaFuncSetAttribute(plain, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return 0;
        if constexpr (BN == FUSED_TILE) {
            auto fused = swap_kernel<FMT, BN, true>;
            if (cudaFuncSetAttribute(fused, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
                return 0;
        }
        for (int c = 8; c >= 1; --c) {
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = c;
            attr.val.clusterDim.y = 1;
            attr.val.clusterDim.z = 1;
            cfg.gridDim = dim3(c, 1024, 1);
            cfg.blockDim = dim3(SWAP_THREADS);
            cfg.dynamicSmemBytes = C::SMEM;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, plain, &cfg) != cudaSuccess || n < 1) return 0;
            resident[dev][c].store(n);
        }
    }
    int split = ktiles < 8 ? ktiles : 8;
    // The count takes one CTA per SM, as if each used all of tensor memory; two run (their
    // columns and shared memory fit).  Measured at 1 x 15360 x 5120 nvfp4: 13.3 us with a
    // split for one per SM, 11.8 for two.
    while (split > 1 && 2 * resident[dev][split].load() < tiles) --split;
    return split;
}

template <int FMT, int BN, bool FUSED>
int launch_swap(const h3_tensor *xc, const h3_tensor *wc, Params &p, cudaStream_t stream) {
    using C = Swap<FMT, BN>;
    CUtensorMap tx, tw;
    H3_CHECK(make_tmap_bytes(&tw, wc->data, wc->shape[1], wc->shape[0],
                             wc->shape[0] > 1 ? wc->strides[0] : wc->shape[1], 128, 128));
    if (FUSED) tx = tw;   // not used
    else
        H3_CHECK(make_tmap_bytes(&tx, xc->data, xc->shape[1], xc->shape[0],
                                 xc->shape[0] > 1 ? xc->strides[0] : xc->shape[1], 128, BN));
    p.num_m = (p.M + BN - 1) / BN;
    p.num_n = (p.N + 127) / 128;
    if (p.num_m > 65535 || p.num_n > 65535) return H3_ERR_UNSUPPORTED;
    const int split = swap_split<FMT, BN>((int64_t)p.num_m * p.num_n, p.ktiles);
    if (split < 1) return H3_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1] = overlapped_launch();
    cfg.gridDim = dim3(split, p.num_n, p.num_m);
    cfg.blockDim = dim3(SWAP_THREADS + (FUSED ? QUANT_WARPS * 32 : 0));
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, swap_kernel<FMT, BN, FUSED>, tx, tw, p) != cudaSuccess) {
        cudaGetLastError();
        return H3_ERR_LAUNCH;
    }
    return launch_status();
}

// ---------------------------------------------------------------------------
// tile form: persistent CTA pairs, 256 x 256 output tiles
// ---------------------------------------------------------------------------
constexpr int TILE = 256;                        // rows and columns of a pair's output tile
constexpr int EPI_WARPS = 8;                     // two per quarter of the rows, each every other 64 columns
constexpr int TILE_THREADS = (4 + EPI_WARPS) * 32;
// Column tiles per raster group.  Sustained at 18944 x 27648 x 5120 nvfp4, under the power cap:
// groups of 4 / 8 / 20 / 32 / 64 / all ran 1331 / 1267 / 1216 / 1206 / 1252 / 1445 us.
constexpr int GROUP_N = 32;

template <int FMT>
struct Pair {
    static constexpr int CH = tile_chunks(FMT);
    static constexpr int SF_BYTES = CH * CHUNK;               // scales of 128 rows per K tile
    static constexpr int OFF_B = 128 * 128;                   // this CTA's 128 x rows, then half the tile's w rows
    static constexpr int OFF_SFA = 2 * OFF_B;
    static constexpr int OFF_SFB = OFF_SFA + SF_BYTES;        // all 256 w rows: each CTA multiplies with every one
    static constexpr int STAGE = OFF_SFB + 2 * SF_BYTES;      // a multiple of 1024
    static constexpr int STAGES = 5;
    static constexpr int STORE = 32 * 128;                    // 32 rows x 64 columns of y, per epilogue warp
    static constexpr int OFF_STORE = STAGES * STAGE;
    static constexpr int OFF_BIAS = OFF_STORE + EPI_WARPS * STORE;   // the bias of those columns
    static constexpr int OFF_BAR = OFF_BIAS + EPI_WARPS * 128;
    static constexpr int SMEM = OFF_BAR + (2 * STAGES + 2) * 8 + 16 + 1024;
    static_assert(STAGE % 1024 == 0 && SMEM <= 232448, "shared memory");
    // Tensor memory: two 256-column accumulators sharing 128 columns, and two buffers of
    // scales (4 columns per 128 rows and chunk: 4 CH of x, 8 CH of w)
    static constexpr int ACC1 = 128;
    static constexpr int SF_COL0 = 384;
    static constexpr int SF_COLS = 12 * CH;
    static_assert(SF_COL0 + 2 * SF_COLS <= 512 && ACC1 + TILE <= SF_COL0, "tensor memory");
};

__device__ __forceinline__ void tile_at(const Params &p, int tile, int &m, int &n) {
    const int span = GROUP_N * p.num_m;
    const int g = tile / span, r = tile - g * span;
    const int gw = min(GROUP_N, p.num_n - g * GROUP_N);
    m = r / gw;
    n = g * GROUP_N + (r - m * gw);
}

template <int FMT>
__global__ void __launch_bounds__(TILE_THREADS, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap tw,
                const __grid_constant__ CUtensorMap tsx, const __grid_constant__ CUtensorMap tsw,
                const __grid_constant__ CUtensorMap ty, Params p) {
    using C = Pair<FMT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
    uint64_t *empty = full + C::STAGES;
    uint64_t *acc_full = empty + C::STAGES;     // the tile's products have landed
    uint64_t *acc_free = acc_full + 1;          // leader's: the columns both accumulators share have been read
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_free + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int first = (int)(blockIdx.x >> 1), step = (int)(gridDim.x >> 1);
    const int num_tiles = p.num_m * p.num_n;

    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(acc_full, 1);
        mbar_init(acc_free, 2 * EPI_WARPS);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    wait_for_previous();   // every warp: the bounded waits below must not count the previous kernel's time

    if (warp == 0) {
        if (elect_one()) {
            tma_prefetch_desc(&tx);
            tma_prefetch_desc(&tw);
            tma_prefetch_desc(&tsx);
            tma_prefetch_desc(&tsw);
        }
        uint32_t it = 0;
        bool ok = true;
        for (int tile = first; tile < num_tiles && ok; tile += step) {
            int m, n;
            tile_at(p, tile, m, n);
            for (int kt = 0; kt < p.ktiles; ++kt, ++it) {
                const uint32_t slot = it % C::STAGES;
                ok = __all_sync(0xffffffffu, mbar_wait(&empty[slot], ((it / C::STAGES) & 1) ^ 1, abort_flag));
                if (!ok) break;
                if (elect_one()) {
                    // both CTAs' bytes are counted on the leader's barrier
                    const uint32_t bar = mapa_shared(&full[slot], 0);
                    if (rank == 0) mbar_expect_tx(&full[slot], 2 * C::STAGE);
                    uint8_t *st = smem + slot * C::STAGE;
                    tma_load_2d_pair(st, &tx, bar, kt * 128, m * TILE + (int)rank * 128);
                    tma_load_2d_pair(st + C::OFF_B, &tw, bar, kt * 128, n * TILE + (int)rank * 128);
                    tma_load_2d_pair(st + C::OFF_SFA, &tsx, bar, kt * (C::SF_BYTES / 8), 2 * m + (int)rank);
                    tma_load_2d_pair(st + C::OFF_SFB, &tsw, bar, kt * (C::SF_BYTES / 8), 2 * n);
                }
                __syncwarp();
            }
        }
        // the leader's last commits arrive here: none may land after this CTA has gone
        for (uint32_t i = 0; i < C::STAGES && ok; ++i) {
            if (it < i + 1) break;
            const uint32_t u = it - 1 - i;
            ok = mbar_wait(&empty[u % C::STAGES], (u / C::STAGES) & 1, abort_flag);
        }
    } else if (warp == 1 && rank == 0) {
        // The whole warp runs this and one lane issues, from uniform registers: descriptors are
        // sums of one per operand, tensor memory addresses constants (all 512 columns are
        // this CTA's, so they start at 0), and one commit signals both CTAs.
        const uint32_t base = smem_u32(smem);
        const uint64_t desc_a = smem_desc_sw128(base, 16, 1024), desc_sf = smem_desc_rows16(base + C::OFF_SFA);
        constexpr uint32_t SF_STEP = C::SF_BYTES >> 4, CHUNK_STEP = CHUNK >> 4;
        uint32_t slot = 0, phase = 0;                  // of this K tile, then of the two before it
        uint32_t slot1 = 0, phase1 = 0, slot2 = 0, phase2 = 0;
        uint32_t it = 0, lt = 0;
        bool ok = tmem == 0;
        for (int tile = first; tile < num_tiles && ok; tile += step, ++lt) {
            // the accumulator two tiles back has been read wholly before the last one's shared columns
            if (lt > 0) ok = __all_sync(0xffffffffu, mbar_wait_cluster(acc_free, (lt - 1) & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const uint32_t d = (lt & 1) ? C::ACC1 : 0;
            for (int kt = 0; kt < p.ktiles; ++kt, ++it) {
                ok = mbar_wait(&full[slot], phase, abort_flag);
                // two scale buffers: the MMAs two K tiles back must have read this one
                if (ok && it >= 2) ok = mbar_wait(&empty[slot2], phase2, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint64_t at = (slot * C::STAGE) >> 4;
                const uint64_t da = desc_a + at, db = da + (C::OFF_B >> 4), ds = desc_sf + at;
                const uint32_t ta = C::SF_COL0 + (it & 1) * C::SF_COLS, tb = ta + 4 * C::CH;
                const int steps = p.ksteps - kt * (BK / KSTEP);
                const uint32_t more = kt > 0;
                if (elect_one()) {
#pragma unroll
                    for (int c = 0; c < C::CH; ++c) {
                        // w's two 128-row chunks lie side by side: 8 columns per K chunk
                        tmem_cp_scales<true>(ta + 4 * c, ds + c * CHUNK_STEP);
                        tmem_cp_scales<true>(tb + 8 * c, ds + SF_STEP + c * CHUNK_STEP);
                        tmem_cp_scales<true>(tb + 8 * c + 4, ds + 2 * SF_STEP + c * CHUNK_STEP);
                    }
#pragma unroll
                    for (int s = 0; s < BK / KSTEP; ++s) {
                        const int c = FMT == MX ? s >> 1 : s;
                        if (s < steps)
                            umma_fp4<FMT == MX, true>(d, da + 2 * s, db + 2 * s,
                                                      idesc_fp4(256, TILE, FMT == MX, FMT == MX ? (s & 1) * 2 : 0),
                                                      ta + 4 * c, tb + 8 * c, s > 0 ? 1u : more);
                    }
                    umma_commit_both(&empty[slot]);
                    if (kt == p.ktiles - 1) umma_commit_both(acc_full);
                }
                __syncwarp();
                slot2 = slot1, phase2 = phase1;
                slot1 = slot, phase1 = phase;
                if (++slot == C::STAGES) slot = 0, phase ^= 1;
            }
        }
        if (!ok) drain_in_flight();
    } else if (warp >= 4) {
        const int wq = warp & 3, half = (warp - 4) >> 2;
        uint8_t *buf = smem + C::OFF_STORE + (warp - 4) * C::STORE;
        const uint32_t bias = smem_u32(smem + C::OFF_BIAS + (warp - 4) * 128);
        uint32_t lt = 0;
        bool ok = true;
        for (int tile = first; tile < num_tiles; tile += step, ++lt) {
            int m, n;
            tile_at(p, tile, m, n);
            const int row0 = m * TILE + (int)rank * 128 + wq * 32;      // this warp's first row
            ok = __all_sync(0xffffffffu, mbar_wait(acc_full, lt & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            const uint32_t acc = tmem + ((lt & 1) ? C::ACC1 : 0) + ((uint32_t)(wq * 32) << 16);
            // 64 columns at a time, of the shared ones first (the end of accumulator 0, the start
            // of accumulator 1); once those are in registers the next tile may start
#pragma unroll 1
            for (int i = 0; i < 2; ++i) {
                const int c0 = (((lt & 1) ? 2 * i : 2 - 2 * i) + half) * 64, col = n * TILE + c0;
                uint32_t v[2][32];
                tmem_ld32(acc + c0, v[0]);
                tmem_ld32(acc + c0 + 32, v[1]);
                uint16_t b0 = 0, b1 = 0;
                if (p.bias) {
                    const uint16_t *b = reinterpret_cast<const uint16_t *>(p.bias) + col + 2 * lane;
                    if (col + 2 * lane < p.N) b0 = b[0];
                    if (col + 2 * lane + 1 < p.N) b1 = b[1];
                }
                tmem_ld_wait();
                if (i == 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(mapa_shared(acc_free, 0));
                }
                if (col >= p.N || row0 >= p.M) continue;                // uniform over the warp
                if (p.bias) {
                    st_shared_f32(bias + lane * 4, b0 | (uint32_t)b1 << 16);
                    __syncwarp();
                }
                uint32_t w[32];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t b[4] = {0, 0, 0, 0};
                        if (p.bias) ld_shared_words(bias + (32 * h + 8 * q) * 2, b);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[16 * h + 4 * q + e] = bf2u(
                                __floats2bfloat162_rn(fmaf(__uint_as_float(v[h][8 * q + 2 * e]), p.t, blo(b[e])),
                                                      fmaf(__uint_as_float(v[h][8 * q + 2 * e + 1]), p.t, bhi(b[e]))));
                    }
                if (p.wide) {
                    if (lane == 0) tma_store_wait_read();                // the last store has read the buffer
                    __syncwarp();
                }
                // 16-byte piece q of row r at q ^ (r & 7): the layout the TMA store reads
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    st_shared_words(smem_u32(buf) + lane * 128 + ((q ^ (lane & 7)) << 4), w[4 * q], w[4 * q + 1],
                                    w[4 * q + 2], w[4 * q + 3]);
                if (p.wide) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(&ty, buf, col, row0);               // clipped at y's last row and column
                        tma_store_commit();
                    }
                } else {
                    // Rows too odd for TMA: two columns per lane, a row at a time.  (4-byte words
                    // across neighbouring lanes where the row starts half way into one took 2 us
                    // longer at 333 x 4861 x 1795, which runs 11.0; 333 x 4864, through TMA, 9.3.)
                    __syncwarp();
                    const int rows = min(32, p.M - row0), left = p.N - col - 2 * lane;
                    const uint32_t at = smem_u32(buf) + (lane & 3) * 4;
                    uint16_t *dst = reinterpret_cast<uint16_t *>(p.y) + (int64_t)row0 * p.ldy + col + 2 * lane;
#pragma unroll 4
                    for (int r = 0; r < rows; ++r, dst += p.ldy) {
                        const uint32_t o = ld_shared_word(at + r * 128 + (((lane >> 2) ^ (r & 7)) << 4));
                        if (left > 0) dst[0] = (uint16_t)o;
                        if (left > 1) dst[1] = (uint16_t)(o >> 16);
                    }
                    __syncwarp();
                }
            }
            tc_fence_before();
        }
        if (p.wide && lane == 0) tma_store_wait_all();
        if (!ok) drain_in_flight();
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();   // neither CTA leaves while the pair's MMAs or arrivals may touch it
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// CTA pairs resident at once.  0: cannot be told.
template <int FMT>
int resident_pairs() {
    using C = Pair<FMT>;
    static std::atomic<int> pairs[64];               // per device, once known
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return 0;
    if (pairs[dev].load() == 0) {
        auto kernel = tile_kernel<FMT>;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) return 0;
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2;
        attr.val.clusterDim.y = 1;
        attr.val.clusterDim.z = 1;
        cfg.gridDim = dim3(2 * (num_sms() / 2));
        cfg.blockDim = dim3(TILE_THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) return 0;
        pairs[dev].store(n);
    }
    return pairs[dev].load();
}

template <int FMT>
int launch_tiles(const h3_tensor *xc, const h3_tensor *wc, Params &p, cudaStream_t stream) {
    using C = Pair<FMT>;
    CUtensorMap tx, tw, tsx, tsw;
    H3_CHECK(make_tmap_bytes(&tx, xc->data, xc->shape[1], xc->shape[0],
                             xc->shape[0] > 1 ? xc->strides[0] : xc->shape[1], 128, 128));
    H3_CHECK(make_tmap_bytes(&tw, wc->data, wc->shape[1], wc->shape[0],
                             wc->shape[0] > 1 ? wc->strides[0] : wc->shape[1], 128, 128));
    H3_CHECK(make_tmap_words(&tsx, p.sx, (uint64_t)p.chunks * CHUNK, (p.M + 127) / 128, C::SF_BYTES, 1));
    H3_CHECK(make_tmap_words(&tsw, p.sw, (uint64_t)p.chunks * CHUNK, (p.N + 127) / 128, C::SF_BYTES, 2));
    p.num_m = (p.M + TILE - 1) / TILE;
    p.num_n = (p.N + TILE - 1) / TILE;
    if ((int64_t)p.num_m * p.num_n > 0x3fffffff) return H3_ERR_UNSUPPORTED;
    // a store through TMA is cut off at y's last row exactly, but along a row at 16 bytes only: rows
    // of whole 16 bytes, or the columns beside y's would be written
    p.wide = aligned16(p.y) && p.ldy % 8 == 0 && p.N % 8 == 0;
    CUtensorMap ty = tx;                             // not used where rows are too odd for it
    if (p.wide) {
        const cuuint64_t dims[2] = {(cuuint64_t)p.N, (cuuint64_t)p.M};
        const cuuint64_t strides[1] = {(cuuint64_t)(p.M > 1 ? p.ldy : p.N) * 2};
        const cuuint32_t box[2] = {64, 32};
        H3_CHECK(make_tmap_bf16(&ty, p.y, 2, dims, strides, box));
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1] = overlapped_launch();
    cfg.blockDim = dim3(TILE_THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    cfg.attrs = attr;
    const int tiles = p.num_m * p.num_n, slots = resident_pairs<FMT>();
    if (slots < 1) return H3_ERR_LAUNCH;
    cfg.gridDim = dim3(2 * (tiles < slots ? tiles : slots));
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, tile_kernel<FMT>, tx, tw, tsx, tsw, ty, p) != cudaSuccess) {
        cudaGetLastError();
        return H3_ERR_LAUNCH;
    }
    return launch_status();
}

// 0 chooses per launch, 1 forces the swap form, 2 the tile form (h3_fp4_variant)
std::atomic<int> g_variant{0};

// Whether the swap form takes less time than the tile form, by an estimate (us): a wave of
// tiles 0.47 per K tile and 1 to hand over, of the swap form's 128 x 128 tiles 0.62 per K tile
// of a CTA's share (0.82 in several waves); the rest of a launch 5.5 and 8.  Both forms
// measured at M 129 to 1500 and six N x K from 1000 x 1000 to 27648 x 5120, nvfp4: 256 x 5120
// x 13824 swap 20.5, tiles 24.1; 512 x 5120 x 5120 swap 19.8, tiles 13.4; 777 x 5120 x 5120
// swap 20.6, tiles 20.5.  The constants are those of a slower state of the tile form, so the
// choice keeps to the swap form a little too long: at worst 1.17 times the tiles' time (384 x
// 5120 x 5120: 15.4 and 13.4; 777 x 4861 x 1795: 16.6 and 14.9), else within 1.07.
template <int FMT>
bool swap_form(const Params &p) {
    if ((p.N + 127) / 128 > 65535 || (p.M + 127) / 128 > 65535) return false;     // its grid's limits
    if (p.M <= 128) return true;
    const int64_t tiles = (int64_t)((p.M + TILE - 1) / TILE) * ((p.N + TILE - 1) / TILE);
    const int64_t small = (int64_t)((p.M + 127) / 128) * ((p.N + 127) / 128);
    const int pairs = resident_pairs<FMT>(), split = swap_split<FMT, 128>(small, p.ktiles), slots = 2 * num_sms();
    if (pairs < 1 || split < 1) return false;
    const double in_tiles = 5.5 + (double)((tiles + pairs - 1) / pairs) * (p.ktiles * 0.47 + 1.0);
    const double waves = (double)((small + slots - 1) / slots);
    const double in_swap = 8.0 + waves * ((p.ktiles + split - 1) / split) * (waves > 1 ? 0.82 : 0.62);
    return in_swap < in_tiles;
}

template <int FMT>
int multiply(const h3_tensor *xc, const h3_tensor *wc, Params &p, cudaStream_t stream) {
    const int v = g_variant.load();
    if (v == 2 || (v == 0 && !swap_form<FMT>(p))) return launch_tiles<FMT>(xc, wc, p, stream);
    if (p.M <= 16) return launch_swap<FMT, 16, false>(xc, wc, p, stream);
    if (p.M <= 32) return launch_swap<FMT, 32, false>(xc, wc, p, stream);
    if (p.M <= 64) return launch_swap<FMT, 64, false>(xc, wc, p, stream);
    return launch_swap<FMT, 128, false>(xc, wc, p, stream);
}

// x quantised inside the product (at most FUSED_ROWS rows)
template <int FMT>
int multiply_fused(const h3_tensor *wc, Params &p, cudaStream_t stream) {
    return launch_swap<FMT, FUSED_TILE, true>(nullptr, wc, p, stream);
}

// Checks of y, bias and the operands' widths; fills everything but the tile counts.
int check_product(const h3_tensor *y, const h3_tensor *xc, const h3_tensor *xs, const h3_tensor *wc,
                  const h3_tensor *ws, const h3_tensor *bias, int64_t rows, int64_t cols, int fmt, float tx, float tw,
                  Params *p) {
    if (!wc) return H3_ERR_NULL;
    H3_CHECK(check_bf16(y));
    if (fmt != MX && fmt != NV) return H3_ERR_UNSUPPORTED;
    if (cols < 1 || wc->ndim != 2) return H3_ERR_BAD_SHAPE;
    const int64_t outs = wc->shape[0];
    H3_CHECK(check_held(wc, ws, fmt, outs, cols));
    H3_CHECK(check_held(xc, xs, fmt, rows, cols));
    if (y->ndim != 2 || y->shape[0] != rows || y->shape[1] != outs) return H3_ERR_BAD_SHAPE;
    if ((outs > 1 && y->strides[1] != 1) || (rows > 1 && y->strides[0] < outs)) return H3_ERR_BAD_LAYOUT;
    if (bias) {
        H3_CHECK(check_bf16(bias));
        if (bias->ndim != 1 || bias->shape[0] != outs) return H3_ERR_BAD_SHAPE;
        if (outs > 1 && bias->strides[0] != 1) return H3_ERR_BAD_LAYOUT;
    }
    if (!held_scale_ok(fmt, tx) || !held_scale_ok(fmt, tw)) return H3_ERR_UNSUPPORTED;
    p->t = tx * tw;
    if (isinf(p->t)) return H3_ERR_UNSUPPORTED;      // 0 times it would be NaN
    if (rows > 0x3fffffffLL || outs > 0x3fffffffLL || cols > (1 << 24)) return H3_ERR_UNSUPPORTED;
    p->M = (int)rows;
    p->N = (int)outs;
    p->ktiles = (int)((cols + BK - 1) / BK);
    p->ksteps = (int)((cols + KSTEP - 1) / KSTEP);
    p->chunks = (int)scale_chunks(fmt, cols);
    p->sx = static_cast<const uint8_t *>(xs->data);
    p->sw = static_cast<const uint8_t *>(ws->data);
    p->y = static_cast<__nv_bfloat16 *>(y->data);
    p->ldy = rows > 1 ? y->strides[0] : 0;
    p->bias = bias && outs > 0 ? static_cast<const __nv_bfloat16 *>(bias->data) : nullptr;
    p->wide = aligned_to(y->data, 8) && p->ldy % 4 == 0;
    return H3_OK;
}

}  // namespace fp4
}  // namespace h3

using namespace h3;

extern "C" int h3_fp4_variant(int variant) {
    if (variant < 0 || variant > 2) return -1;
    return fp4::g_variant.exchange(variant);
}

extern "C" int h3_linear_fp4_quantized(const h3_tensor *y, const h3_tensor *x_codes, const h3_tensor *x_scales,
                                       const h3_tensor *w_codes, const h3_tensor *w_scales, const h3_tensor *bias,
                                       int64_t cols, int32_t format, float x_tensor_scale, float w_tensor_scale,
                                       void *stream) {
    if (!x_codes) return H3_ERR_NULL;
    fp4::Params p{};
    H3_CHECK(fp4::check_product(y, x_codes, x_scales, w_codes, w_scales, bias, x_codes->shape[0], cols, format,
                                x_tensor_scale, w_tensor_scale, &p));
    if (p.M == 0 || p.N == 0) return H3_OK;
    return format == fp4::MX ? fp4::multiply<fp4::MX>(x_codes, w_codes, p, (cudaStream_t)stream)
                             : fp4::multiply<fp4::NV>(x_codes, w_codes, p, (cudaStream_t)stream);
}

extern "C" int h3_linear_fp4(const h3_tensor *y, const h3_tensor *x, const h3_tensor *workspace,
                             const h3_tensor *w_codes, const h3_tensor *w_scales, const h3_tensor *bias, int32_t format,
                             float x_tensor_scale, float w_tensor_scale, void *stream) {
    H3_CHECK(check_bf16(x));
    if (x->ndim != 2 || x->shape[1] < 1) return H3_ERR_BAD_SHAPE;
    if (format != fp4::MX && format != fp4::NV) return H3_ERR_UNSUPPORTED;
    if (!fp4::tensor_scale_ok(format, x_tensor_scale)) return H3_ERR_UNSUPPORTED;
    const int64_t rows = x->shape[0], cols = x->shape[1];
    if (rows > 0x3fffffffLL || cols > (1 << 24)) return H3_ERR_UNSUPPORTED;
    if ((cols > 1 && x->strides[1] != 1) || (rows > 1 && x->strides[0] < 0)) return H3_ERR_BAD_LAYOUT;
    // x in 4 bits: its codes, then its scales
    const int64_t pitch = fp4::code_pitch(cols), groups = (rows + 127) / 128, chunks = fp4::scale_chunks(format, cols);
    const bool fused = !workspace;
    uint8_t *at = nullptr;
    if (fused) {
        if (rows > fp4::FUSED_ROWS) return H3_ERR_NULL;
    } else {
        H3_CHECK(check_desc(workspace, H3_U8));
        if (workspace->ndim != 1 || workspace->shape[0] < rows * pitch + groups * chunks * fp4::CHUNK)
            return H3_ERR_BAD_SHAPE;
        if (rows > 0 && (workspace->strides[0] != 1 || !aligned16(workspace->data))) return H3_ERR_BAD_LAYOUT;
        at = static_cast<uint8_t *>(workspace->data);
    }
    // (of a fused product only the shapes are looked at; its data pointers stand for themselves)
    uint8_t *held = fused ? reinterpret_cast<uint8_t *>(uintptr_t(16)) : at;
    const h3_tensor xc = {held, {rows, pitch}, {pitch, 1}, 2, H3_U8};
    const h3_tensor xs = {held + rows * pitch, {groups, chunks, fp4::CHUNK}, {chunks * fp4::CHUNK, fp4::CHUNK, 1}, 3, H3_U8};
    fp4::Params p{};
    H3_CHECK(fp4::check_product(y, &xc, &xs, w_codes, w_scales, bias, rows, cols, format, x_tensor_scale,
                                w_tensor_scale, &p));
    if (p.M == 0 || p.N == 0) return H3_OK;
    if (fused) {
        p.sx = nullptr;
        p.x = static_cast<const __nv_bfloat16 *>(x->data);
        p.ldx = rows > 1 ? x->strides[0] : 0;
        p.cols = (int)cols;
        p.x_vec = aligned16(x->data) && p.ldx % 8 == 0;
        p.x_scale = fp4::TensorScale::make(x_tensor_scale);
        return format == fp4::MX ? fp4::multiply_fused<fp4::MX>(w_codes, p, (cudaStream_t)stream)
                                 : fp4::multiply_fused<fp4::NV>(w_codes, p, (cudaStream_t)stream);
    }
    H3_CHECK(fp4::quantize(&xc, &xs, x, format, x_tensor_scale, (cudaStream_t)stream));
    p.dependent = 1;
    return format == fp4::MX ? fp4::multiply<fp4::MX>(&xc, w_codes, p, (cudaStream_t)stream)
                             : fp4::multiply<fp4::NV>(&xc, w_codes, p, (cudaStream_t)stream);
}

// device error word of this translation unit (bounded waits of the products)
extern "C" unsigned int h3_fp4_device_error_read_and_clear(void) {
    unsigned int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, h3::g_h3_device_error, sizeof(v));
    cudaMemcpyToSymbol(h3::g_h3_device_error, &zero, sizeof(zero));
    return v;
}
