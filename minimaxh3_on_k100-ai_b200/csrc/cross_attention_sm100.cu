// Cross attention of query tokens to an encoder's states (sm_100a), head dim 128:
//
//   o[b,i,h] = sum_{j < len_b} softmax_j(scale * q[b,i,h] . k[b,j,g]) v[b,j,g],  g = h / (H / Hkv)
//
// each sample with its own number of states len_b (read on the device; none: zeros), query
// heads in groups over fewer key/value heads, keys and values of one sample shared by the
// batch where they have batch size 1.  What lies behind len_b is never added, whatever it
// holds: scores there are replaced by -inf and the rows of V by zeros (0 * NaN is NaN).  A
// row whose scores are all -inf attends to nothing: zeros.
//
// tile form (more rows per key/value head than the rows form takes): the products and the
// softmax of the self attention kernel (attention_sm100.cu) -- 128-row Q tiles, two per
// CTA, S and O in tensor memory, P through a swizzled shared tile, separate issuers for
// Q K^T and P V -- made persistent: an encoder's states are few, a work item (two Q tiles
// of one head) has only a handful of key tiles, and loading Q, filling the pipe and
// storing O would take as long as its products.  Here the barriers' phases run on from
// item to item: Q_t of the next item loads once the last S_t has been computed, and its
// first S_t runs while the softmax warps still store O_t.  Two softmax statistics per row
// in fp32, P rounded to BF16 (relative to the running maximum, as the tensor core takes
// it), O accumulated in fp32 and rounded once.
//
// rows form (a token, or a few, per sample): bound by reading K and V, so the keys are
// split over the warps of a CTA and the CTAs of a cluster.  A producer warp streams key
// tiles by TMA through a ring; each computing warp takes 16 keys of a tile against all the
// rows (mma.sync m16n8k16: the rows fill an M of 16 or 32, a 128-row tcgen05 tile would be
// nearly empty and its softmax a single lane per row), with its own running maximum and
// sum.  Partial results join in shared memory, then over the cluster through distributed
// shared memory in rank order: one launch, no scratch, the same bits every time.
#include <math.h>
#include <stdint.h>

#include "attn_math.cuh"
#include "h3_abi_util.h"
#include "h3_common.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.h"

namespace h3 {
namespace cross {

using attn::ex2;
using attn::fadd2;
using attn::ffma2;
using attn::max3f;
using attn::pack_bf16x2;
using attn::pk2;
using attn::st_shared_v4;
using attn::swz;
using attn::up2;

constexpr int HD = 128;
constexpr int TILE_BYTES = 128 * 128 * 2;        // a 128 x 128 BF16 tile
constexpr int HALF = TILE_BYTES / 2;             // its 64-column (128B swizzle span) half
constexpr float RESCALE_THRESHOLD = 8.0f;        // log2 domain: O is rescaled when the maximum grows by more

struct Params {
    int Sq, Sk, H, group, B;     // group: query heads per key/value head
    int kv_shared;               // K and V have batch size 1
    float scale_log2;
    const int64_t *lens;         // [B] or null
    int items, per_head;         // tile form: work items, items per (sample, head)
    int ordered;                 // samples with more states first
    // rows form: row r of a (sample, key/value head) is query r / group, head r % group of the group
    const __nv_bfloat16 *q;
    __nv_bfloat16 *out;
    int64_t q_b, q_s, q_h, o_b, o_s, o_h;
    int rows;                    // rows per (sample, key/value head); all samples' where they are folded
    int fold;                    // rows run over the batch too (K and V shared, no lengths)
    int kv_heads, chunks;        // row chunks per (sample, key/value head)
};

__device__ __forceinline__ int states(const Params &p, int b) {
    if (!p.lens) return p.Sk;
    const int64_t n = p.lens[b];
    return n < 0 ? 0 : n > p.Sk ? p.Sk : (int)n;
}

// ---------------------------------------------------------------------------
// tile form
// ---------------------------------------------------------------------------
constexpr int BM = 128, BN = 128;
constexpr int TILE_THREADS = 384;
constexpr int MAX_ORDERED = 512;                 // samples that are sorted by length; more are taken as they come

template <int NQ>                                // Q tiles per work item: 1 or 2
struct Tile {
    // S_t(j+1) is computed as soon as softmax t has read S_t(j), a whole step ahead of its
    // use, so K_{j+1} may load after both S(j): one slot.  P_t(j+1) V_{j+1} comes right
    // when its P is ready, so V_{j+1} has to be there by then: two.
    static constexpr int KSLOTS = NQ == 2 ? 1 : 2;
    static constexpr int VSLOTS = 2;
    static constexpr int OFF_Q = 0;
    static constexpr int OFF_P = OFF_Q + NQ * TILE_BYTES;
    static constexpr int OFF_K = OFF_P + NQ * TILE_BYTES;
    static constexpr int OFF_V = OFF_K + KSLOTS * TILE_BYTES;
    static constexpr int OFF_BAR = OFF_V + VSLOTS * TILE_BYTES;
    static constexpr int NUM_BARS = 2 * KSLOTS + 3 * VSLOTS + 6 * NQ;
    static constexpr int OFF_ORDER = OFF_BAR + NUM_BARS * 8 + 16;
    static constexpr int SMEM = OFF_ORDER + MAX_ORDERED * 2 + 1024;
    static constexpr uint32_t TMEM = NQ * 256;
    static constexpr int O_COL = NQ * BN;
    static_assert(SMEM <= 232448, "shared memory");
};

template <int NQ>
__global__ void __launch_bounds__(TILE_THREADS, 1)
    tile_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to, Params p) {
    using C = Tile<NQ>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
    uint64_t *k_empty = k_full + C::KSLOTS;
    uint64_t *v_full = k_empty + C::KSLOTS;
    uint64_t *v_empty = v_full + C::VSLOTS;
    uint64_t *v_clean = v_empty + C::VSLOTS;  // rows of V behind the last state are zero
    uint64_t *q_full = v_clean + C::VSLOTS;
    uint64_t *q_free = q_full + NQ;           // [t]: the item's last S_t has been computed
    uint64_t *s_full = q_free + NQ;           // [t]: S_t(j) in tensor memory
    uint64_t *s_free = s_full + NQ;           // [t]: softmax t has read S_t(j)
    uint64_t *p_ready = s_free + NQ;          // [t]: P_t(j) in shared memory, O_t rescaled
    uint64_t *o_done = p_ready + NQ;          // [t]: P_t(j) V_j has landed in O_t
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(o_done + NQ);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    uint16_t *order = reinterpret_cast<uint16_t *>(smem + C::OFF_ORDER);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::KSLOTS; ++i) {
            mbar_init(&k_full[i], 1);
            mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < C::VSLOTS; ++i) {
            mbar_init(&v_full[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&v_clean[i], 1);
        }
        for (int t = 0; t < NQ; ++t) {
            mbar_init(&q_full[t], 1);
            mbar_init(&q_free[t], 1);
            mbar_init(&s_full[t], 1);
            mbar_init(&s_free[t], 128);
            mbar_init(&p_ready[t], 128);
            mbar_init(&o_done[t], 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM);
        tmem_relinquish();
    }
    wait_for_previous();
    if (p.ordered) {
        // samples by their number of key tiles, most first (their rank by counting)
        int *cost = reinterpret_cast<int *>(smem + C::OFF_Q);
        for (int i = threadIdx.x; i < p.B; i += TILE_THREADS) cost[i] = (states(p, i) + BN - 1) / BN;
        __syncthreads();
        for (int i = threadIdx.x; i < p.B; i += TILE_THREADS) {
            const int mine = cost[i];
            int r = 0;
            for (int j = 0; j < p.B; ++j) r += cost[j] > mine || (cost[j] == mine && j < i);
            order[r] = (uint16_t)i;
        }
        fence_proxy_async_smem();   // Q's tile is loaded over the costs
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Every role walks the same items; an item's number of key tiles comes from its
    // sample's length.  `n` counts key tiles over all items, `qi` items with any.
    auto item_at = [&](int i, int &b, int &h, int &q0, int &len) {
        // round k deals items k G .. k G + G - 1 to the G CTAs, every other round in reverse:
        // whoever got a long one gets a short one next
        const int k = i / (int)gridDim.x, c = i - k * (int)gridDim.x;
        const int item = p.ordered && (k & 1) ? min(p.items - k * (int)gridDim.x, (int)gridDim.x) - 1 - c + k * (int)gridDim.x : i;
        const int hb = item / p.per_head;
        b = hb / p.H;
        h = hb - b * p.H;
        q0 = (item - hb * p.per_head) * NQ * BM;
        if (p.ordered) b = order[b];
        len = states(p, b);
    };
    bool ok = true;

    if (warp == 0 || warp == 3) {
        // ------------------------------------------------------------ TMA: Q and K, or V
        const bool kq = warp == 0;
        if (elect_one()) {
            tma_prefetch_desc(kq ? &tk : &tv);
            if (kq) tma_prefetch_desc(&tq);
        }
        uint32_t n = 0, qi = 0;
        for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
            int b, h, q0, len;
            item_at(item, b, h, q0, len);
            const int nkv = (len + BN - 1) / BN, kb = p.kv_shared ? 0 : b, kh = h / p.group;
            for (int j = 0; j < nkv && ok; ++j, ++n) {
                if (kq) {
                    if (j == 0) {
                        for (int t = 0; t < NQ && ok; ++t) {
                            ok = __all_sync(0xffffffffu, mbar_wait(&q_free[t], (qi & 1) ^ 1, abort_flag));
                            if (ok && elect_one()) {
                                mbar_expect_tx(&q_full[t], TILE_BYTES);
                                for (int hf = 0; hf < 2; ++hf)
                                    tma_load_4d(smem + C::OFF_Q + t * TILE_BYTES + hf * HALF, &tq, &q_full[t], hf * 64,
                                                q0 + t * BM, h, b);
                            }
                            __syncwarp();
                        }
                        ++qi;
                    }
                    const uint32_t s = n % C::KSLOTS;
                    ok = ok && __all_sync(0xffffffffu, mbar_wait(&k_empty[s], ((n / C::KSLOTS) & 1) ^ 1, abort_flag));
                    if (ok && elect_one()) {
                        mbar_expect_tx(&k_full[s], TILE_BYTES);
                        for (int hf = 0; hf < 2; ++hf)
                            tma_load_4d(smem + C::OFF_K + s * TILE_BYTES + hf * HALF, &tk, &k_full[s], hf * 64, j * BN,
                                        kh, kb);
                    }
                    __syncwarp();
                } else {
                    const uint32_t s = n % C::VSLOTS;
                    uint8_t *dst = smem + C::OFF_V + s * TILE_BYTES;
                    ok = __all_sync(0xffffffffu, mbar_wait(&v_empty[s], ((n / C::VSLOTS) & 1) ^ 1, abort_flag));
                    if (ok && elect_one()) {
                        mbar_expect_tx(&v_full[s], TILE_BYTES);
                        for (int hf = 0; hf < 2; ++hf)
                            tma_load_4d(dst + hf * HALF, &tv, &v_full[s], hf * 64, j * BN, kh, kb);
                    }
                    __syncwarp();
                    const int valid = len - j * BN;
                    if (ok && valid < BN && len < p.Sk) {
                        // rows of another use of the buffer: zeros, so that P's zeros times them add nothing
                        ok = __all_sync(0xffffffffu, mbar_wait(&v_full[s], (n / C::VSLOTS) & 1, abort_flag));
                        for (int i = valid * 8 + lane; i < BN * 8 && ok; i += 32)
                            for (int hf = 0; hf < 2; ++hf) st_shared_v4(smem_u32(dst) + hf * HALF + i * 16, 0, 0, 0, 0);
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&v_clean[s]);
                    }
                }
            }
        }
        // the last commits arrive on these barriers: none may land after the CTA has gone
        if (kq) {
            for (int t = 0; t < NQ && qi > 0 && ok; ++t) ok = mbar_wait(&q_free[t], (qi - 1) & 1, abort_flag);
            for (uint32_t i = 1; i <= C::KSLOTS && i <= n && ok; ++i)
                ok = mbar_wait(&k_empty[(n - i) % C::KSLOTS], ((n - i) / C::KSLOTS) & 1, abort_flag);
        } else {
            for (uint32_t i = 1; i <= C::VSLOTS && i <= n && ok; ++i)
                ok = mbar_wait(&v_empty[(n - i) % C::VSLOTS], ((n - i) / C::VSLOTS) & 1, abort_flag);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ S_t(j) = Q_t K_j^T
        constexpr uint32_t ID_S = idesc_bf16_f32(BM, BN, false);
        const uint32_t q_base = smem_u32(smem + C::OFF_Q), k_base = smem_u32(smem + C::OFF_K);
        uint32_t n = 0, qi = 0;
        for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
            int b, h, q0, len;
            item_at(item, b, h, q0, len);
            const int nkv = (len + BN - 1) / BN;
            for (int j = 0; j < nkv && ok; ++j, ++n) {
                const uint32_t s = n % C::KSLOTS;
                ok = mbar_wait(&k_full[s], (n / C::KSLOTS) & 1, abort_flag);
                for (int t = 0; t < NQ; ++t) {
                    if (ok && j == 0) ok = mbar_wait(&q_full[t], qi & 1, abort_flag);
                    if (ok && n > 0) ok = mbar_wait(&s_free[t], (n - 1) & 1, abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t a = q_base + t * TILE_BYTES, kk0 = k_base + s * TILE_BYTES;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk) {
                            const uint32_t o = (kk >> 2) * HALF + (kk & 3) * 32;
                            umma_ss(tmem + t * BN, smem_desc_sw128(a + o, 16, 1024), smem_desc_sw128(kk0 + o, 16, 1024),
                                    ID_S, kk > 0 ? 1u : 0u);
                        }
                        umma_commit(&s_full[t]);
                        if (j == nkv - 1) umma_commit(&q_free[t]);
                        if (t == NQ - 1) umma_commit(&k_empty[s]);
                    }
                    __syncwarp();
                }
            }
            if (nkv > 0) ++qi;
        }
        if (!ok) drain_in_flight();
    } else if (warp == 2) {
        // ------------------------------------------------------------ O_t += P_t(j) V_j
        constexpr uint32_t ID_PV = idesc_bf16_f32(BM, HD, true);
        const uint32_t p_base = smem_u32(smem + C::OFF_P), v_base = smem_u32(smem + C::OFF_V);
        uint32_t n = 0, clean = 0;               // clean: per slot, the parity its next zeroing completes
        for (int item = blockIdx.x; item < p.items && ok; item += gridDim.x) {
            int b, h, q0, len;
            item_at(item, b, h, q0, len);
            const int nkv = (len + BN - 1) / BN;
            for (int j = 0; j < nkv && ok; ++j, ++n) {
                const uint32_t s = n % C::VSLOTS;
                ok = mbar_wait(&v_full[s], (n / C::VSLOTS) & 1, abort_flag);
                if (len - j * BN < BN && len < p.Sk) {
                    ok = ok && mbar_wait(&v_clean[s], (clean >> s) & 1, abort_flag);
                    clean ^= 1u << s;
                }
                for (int t = 0; t < NQ; ++t) {
                    ok = __all_sync(0xffffffffu, ok && mbar_wait(&p_ready[t], n & 1, abort_flag));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t a = p_base + t * TILE_BYTES, vv = v_base + s * TILE_BYTES;
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < 8; ++kk)
                            umma_ss(tmem + C::O_COL + t * HD,
                                    smem_desc_sw128(a + (kk >> 2) * HALF + (kk & 3) * 32, 16, 1024),
                                    smem_desc_sw128(vv + kk * 2048, HALF, 1024), ID_PV, (j > 0 || kk > 0) ? 1u : 0u);
                        umma_commit(&o_done[t]);
                        if (t == NQ - 1) umma_commit(&v_empty[s]);
                    }
                    __syncwarp();
                }
            }
        }
        if (!ok) drain_in_flight();
    } else if (((warp - 4) >> 2) < NQ) {
        // ------------------------------------------------------------ softmax, output
        // The group's warps find out one by one that a wait gave up, and one may still pass a wait
        // that another gave up on.  So `ok` decides only what a warp computes: each passes both
        // named barriers of every item to the end.
        const int t = (warp - 4) >> 2;
        const int row = (warp & 3) * 32 + lane;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + t * BN + lane_off;
        const uint32_t o_addr = tmem + C::O_COL + t * HD + lane_off;
        uint8_t *p_ptr = smem + C::OFF_P + t * TILE_BYTES;
        const uint32_t p_tile = smem_u32(p_ptr);
        const float c = p.scale_log2;
        uint32_t n = 0;
        for (int item = blockIdx.x; item < p.items; item += gridDim.x) {
            int b, h, q0, len;
            item_at(item, b, h, q0, len);
            const int nkv = (len + BN - 1) / BN;
            float m = -INFINITY, l0 = 0.f, l1 = 0.f;
            int j = 0;
            for (; j < nkv && ok; ++j, ++n) {
                ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], n & 1, abort_flag));
                if (!ok) break;
                tc_fence_after();
                uint32_t s[BN];
                tmem_ld32(s_addr + 0, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
                tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
                tmem_ld32(s_addr + 64, *reinterpret_cast<uint32_t(*)[32]>(&s[64]));
                tmem_ld32(s_addr + 96, *reinterpret_cast<uint32_t(*)[32]>(&s[96]));
                tmem_ld_wait();
                tc_fence_before();
                mbar_arrive(&s_free[t]);     // the next S_t may overwrite it
                const int valid = len - j * BN;
                if (valid < BN) {
#pragma unroll
                    for (int i = 0; i < BN; ++i)
                        if (i >= valid) s[i] = __float_as_uint(-INFINITY);
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < BN; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mx[k] = max3f(mx[k], __uint_as_float(s[i + 2 * k]), __uint_as_float(s[i + 2 * k + 1]));
                const float mnew = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
                float alpha = 1.f;
                bool rescale = false;
                if (j == 0) {
                    m = mnew;
                } else if (mnew > m + RESCALE_THRESHOLD) {
                    alpha = ex2(m - mnew);
                    m = mnew;
                    rescale = true;
                }
                const float neg_m = m == -INFINITY ? 0.f : -m;       // nothing but -inf so far: every P is 0
                const uint64_t c2 = pk2(c, c), nm2 = pk2(neg_m, neg_m);
                uint32_t w[BN / 2];
                // two groups of 32 key pairs with their own sums: shorter addition chains
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    uint64_t rs0 = pk2(0.f, 0.f), rs1 = pk2(0.f, 0.f);
#pragma unroll
                    for (int ii = 0; ii < 32; ++ii) {
                        const int i = g * 32 + ii;
                        float x0, x1;
                        up2(ffma2(pk2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, nm2), x0, x1);
                        const float p0 = ex2(x0), p1 = ex2(x1);
                        if (ii & 1) rs1 = fadd2(rs1, pk2(p0, p1));
                        else rs0 = fadd2(rs0, pk2(p0, p1));
                        w[i] = pack_bf16x2(p0, p1);
                    }
                    float r0, r1, r2, r3;
                    up2(rs0, r0, r1);
                    up2(rs1, r2, r3);
                    float &l = g == 0 ? l0 : l1;
                    l = l * alpha + ((r0 + r1) + (r2 + r3));
                }
                if (j == 0) {
                    // the previous item's output, staged in the P tile, must have been read
                    if (row == 0) tma_store_wait_read();
                    named_bar_sync(1 + t, 128);
                } else {
                    // P_t(j-1) V_{j-1} has read the P tile and landed in O_t
                    ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], (n - 1) & 1, abort_flag));
                    if (!ok) break;
                    if (__any_sync(0xffffffffu, rescale)) {          // tcgen05.ld/st take whole warps
                        tc_fence_after();
#pragma unroll 1
                        for (int cc = 0; cc < 4; ++cc) {
                            uint32_t o[32];
                            tmem_ld32(o_addr + cc * 32, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st32(o_addr + cc * 32, o);
                        }
                        tmem_st_wait();
                    }
                }
#pragma unroll
                for (int q = 0; q < 16; ++q)
                    st_shared_v4(p_tile + (q >> 3) * HALF + swz(row, q & 7), w[4 * q], w[4 * q + 1], w[4 * q + 2],
                                 w[4 * q + 3]);
                fence_proxy_async_smem();
                tc_fence_before();
                mbar_arrive(&p_ready[t]);
            }
            if (j == 0) {                        // no states, or given up before the barrier of the first tile
                if (row == 0) tma_store_wait_read();
                named_bar_sync(1 + t, 128);
            } else if (ok) {
                ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], (n - 1) & 1, abort_flag));
                tc_fence_after();
            }
            const float lsum = l0 + l1;
            // No state, or none with a finite score: zeros.  A maximum that fp32 cannot hold: NaN (the
            // fused product minus it is -inf for every finite score, which would read as no state).
            const float inv = m == INFINITY ? NAN : lsum == 0.f ? 0.f : 1.0f / lsum;
#pragma unroll 1
            for (int cc = 0; cc < 4 && ok; ++cc) {
                uint32_t o[32];
                if (nkv > 0) {
                    tmem_ld32(o_addr + cc * 32, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    st_shared_v4(p_tile + (cc >> 1) * HALF + swz(row, (cc & 1) * 4 + q),
                                 pack_bf16x2(__uint_as_float(o[8 * q + 0]) * inv, __uint_as_float(o[8 * q + 1]) * inv),
                                 pack_bf16x2(__uint_as_float(o[8 * q + 2]) * inv, __uint_as_float(o[8 * q + 3]) * inv),
                                 pack_bf16x2(__uint_as_float(o[8 * q + 4]) * inv, __uint_as_float(o[8 * q + 5]) * inv),
                                 pack_bf16x2(__uint_as_float(o[8 * q + 6]) * inv, __uint_as_float(o[8 * q + 7]) * inv));
            }
            tc_fence_before();
            fence_proxy_async_smem();
            named_bar_sync(1 + t, 128);
            // rows past Sq are clipped; where a warp gave up its rows are not there
            if (row == 0 && q0 + t * BM < p.Sq && !*abort_flag) {
                tma_store_4d(&to, p_ptr, 0, q0 + t * BM, h, b);
                tma_store_4d(&to, p_ptr + HALF, 64, q0 + t * BM, h, b);
                tma_store_commit();
            }
        }
        if (row == 0) tma_store_wait_all();
        if (!ok) drain_in_flight();
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM);
    }
}

// ---------------------------------------------------------------------------
// rows form
// ---------------------------------------------------------------------------
constexpr int KW = 16;                           // keys per warp and tile
constexpr int MAX_SPLIT = 16;                    // CTAs per cluster

template <int MT, int WARPS>                     // 16-row MMA tiles (rows per CTA / 16), warps that compute
struct Rows {
    static constexpr int ROWS = 16 * MT;
    static constexpr int THREADS = (WARPS + 1) * 32;
    static constexpr int KEYS = WARPS * KW;      // keys per tile
    static constexpr int KV_BYTES = KEYS * HD * 2;   // a K or V tile
    static constexpr int KV_HALF = KV_BYTES / 2;
    static constexpr int STAGES = 3;
    static constexpr int RING = STAGES * 2 * KV_BYTES;
    // in the ring's place at the end: O of each warp, then their sum (a float4 of padding
    // per row keeps the four lanes of a quad on different banks)
    static constexpr int PITCH = HD + 4;
    static constexpr int OFF_SUM = WARPS * ROWS * PITCH * 4;
    static constexpr int OFF_BAR = RING > OFF_SUM + ROWS * PITCH * 4 ? RING : OFF_SUM + ROWS * PITCH * 4;
    static constexpr int OFF_ML = OFF_BAR + 2 * STAGES * 8 + 16;         // [warp, joint][row] maximum and sum
    static constexpr int SMEM = OFF_ML + (WARPS + 1) * ROWS * 8 + 1024;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr, uint32_t rank) {
    float v;
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
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

// grid: x = cluster rank (share of the keys), y = (sample, key/value head, row chunk)
template <int MT, int WARPS>
__global__ void __launch_bounds__(Rows<MT, WARPS>::THREADS)
    rows_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, Params p) {
    using C = Rows<MT, WARPS>;
    constexpr int ROW_WARPS = WARPS, ROW_THREADS = C::THREADS, KEYS = C::KEYS, KV_BYTES = C::KV_BYTES, KV_HALF = C::KV_HALF;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
    uint64_t *empty = full + C::STAGES;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(empty + C::STAGES);
    float *ml = reinterpret_cast<float *>(smem + C::OFF_ML);      // maxima, then sums, each [warps + 1][ROWS]
    float *o_part = reinterpret_cast<float *>(smem);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = (int)gridDim.x, rank = (int)blockIdx.x;
    int y = (int)blockIdx.y;
    const int chunk = y % p.chunks;
    y /= p.chunks;
    const int kh = y % p.kv_heads, b = y / p.kv_heads;            // b = 0 where the batch is folded
    const int row0 = chunk * C::ROWS, rows = min(C::ROWS, p.rows - row0);
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], ROW_WARPS);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    wait_for_previous();
    const int len = states(p, b);
    const int tiles = (len + KEYS - 1) / KEYS;
    const int t0 = (int)((int64_t)tiles * rank / split), t1 = (int)((int64_t)tiles * (rank + 1) / split);

    // query and output offset of row r of this CTA
    auto row_at = [&](int r, int64_t sb, int64_t ss, int64_t sh) -> int64_t {
        int g = row0 + r, bb = b;
        if (p.fold) {
            bb = g / (p.Sq * p.group);
            g -= bb * p.Sq * p.group;
        }
        const int s = g / p.group;
        return bb * sb + s * ss + (int64_t)(kh * p.group + (g - s * p.group)) * sh;
    };

    __syncthreads();

    if (warp == ROW_WARPS) {
        const int kb = p.kv_shared ? 0 : b;
        bool ok = true;
        for (int i = 0; i < t1 - t0; ++i) {
            const int s = i % C::STAGES;
            if (i >= C::STAGES)
                ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], (i / C::STAGES - 1) & 1, abort_flag));
            if (!ok) break;
            if (elect_one()) {
                uint8_t *st = smem + s * 2 * KV_BYTES;
                mbar_expect_tx(&full[s], 2 * KV_BYTES);
                for (int hf = 0; hf < 2; ++hf)
                    tma_load_4d(st + hf * KV_HALF, &tk, &full[s], hf * 64, (t0 + i) * KEYS, kh, kb);
                for (int hf = 0; hf < 2; ++hf)
                    tma_load_4d(st + KV_BYTES + hf * KV_HALF, &tv, &full[s], hf * 64, (t0 + i) * KEYS, kh, kb);
            }
            __syncwarp();
        }
        if (!ok) drain_in_flight();
    } else {
        // A fragments of the rows: lane holds rows lane/4 and lane/4 + 8, columns 2 (lane%4) + {0, 1, 8, 9} + 16 k
        uint32_t qf[MT][8][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
                const int r = mt * 16 + (lane >> 2) + hi * 8;
                const __nv_bfloat16 *src = p.q + row_at(min(r, rows - 1), p.q_b, p.q_s, p.q_h) + (lane & 3) * 2;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    qf[mt][k][hi] = r < rows ? *reinterpret_cast<const uint32_t *>(src + 16 * k) : 0u;
                    qf[mt][k][hi + 2] = r < rows ? *reinterpret_cast<const uint32_t *>(src + 16 * k + 8) : 0u;
                }
            }
        float o[MT][16][4] = {};
        float m[MT][2], l[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) m[mt][0] = m[mt][1] = -INFINITY, l[mt][0] = l[mt][1] = 0.f;
        bool ok = true;
        for (int i = 0; i < t1 - t0; ++i) {
            const int s = i % C::STAGES;
            ok = __all_sync(0xffffffffu, mbar_wait(&full[s], (i / C::STAGES) & 1, abort_flag));
            if (!ok) break;
            const int key0 = (t0 + i) * KEYS + warp * KW;         // this warp's KW keys
            if (key0 < len) {
                const uint32_t kt = smem_u32(smem + s * 2 * KV_BYTES), vt = kt + KV_BYTES;
                // lanes 0-7, 8-15, 16-23, 24-31 address the four 8 x 8 matrices: keys 0-7 and
                // 8-15 (K: bit 4 of the lane, V: bit 3), columns 0-7 and 8-15 (the other bit)
                const int kr = warp * KW + (lane & 7) + (lane & 16 ? 8 : 0), kc = lane & 8 ? 1 : 0;
                const int vr = warp * KW + (lane & 7) + (lane & 8 ? 8 : 0), vc = lane & 16 ? 1 : 0;
                // fragments are fetched ahead of the products that use them: all of a row tile's,
                // or (MT = 2, where registers are short) four at a time
                constexpr int AHEAD = MT == 1 ? 8 : 4;
                float sc[MT][2][4] = {};
                uint32_t bf[AHEAD][4];
#pragma unroll
                for (int k0 = 0; k0 < 8; k0 += AHEAD) {
#pragma unroll
                    for (int k = 0; k < AHEAD; ++k)
                        ldsm4(kt + ((k0 + k) >> 2) * KV_HALF + swz(kr, ((k0 + k) & 3) * 2 + kc), bf[k]);
#pragma unroll
                    for (int k = 0; k < AHEAD; ++k)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma16816(sc[mt][0], qf[mt][k0 + k], bf[k][0], bf[k][1]);
                            mma16816(sc[mt][1], qf[mt][k0 + k], bf[k][2], bf[k][3]);
                        }
                }
                // the first of V's fragments, to arrive behind the softmax
#pragma unroll
                for (int d = 0; d < AHEAD; ++d) ldsm4_trans(vt + (d >> 2) * KV_HALF + swz(vr, (d & 3) * 2 + vc), bf[d]);
                const int valid = len - key0;                     // of these KW keys
                uint32_t pf[MT][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int key = nt * 8 + (lane & 3) * 2 + (e & 1);
                            sc[mt][nt][e] = key < valid ? sc[mt][nt][e] * p.scale_log2 : -INFINITY;
                        }
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        float mx = max3f(fmaxf(sc[mt][0][2 * hi], sc[mt][0][2 * hi + 1]), sc[mt][1][2 * hi],
                                         sc[mt][1][2 * hi + 1]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        if (mx > m[mt][hi]) {                     // the same in the row's four lanes
                            const float alpha = ex2(m[mt][hi] - mx);
                            m[mt][hi] = mx;
                            l[mt][hi] *= alpha;
#pragma unroll
                            for (int d = 0; d < 16; ++d) o[mt][d][2 * hi] *= alpha, o[mt][d][2 * hi + 1] *= alpha;
                        }
                        const float base = m[mt][hi] == -INFINITY ? 0.f : m[mt][hi];
                        float pr[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) pr[e] = ex2(sc[mt][e >> 1][2 * hi + (e & 1)] - base);
                        l[mt][hi] += (pr[0] + pr[1]) + (pr[2] + pr[3]);
                        pf[mt][hi] = pack_bf16x2(pr[0], pr[1]);
                        pf[mt][hi + 2] = pack_bf16x2(pr[2], pr[3]);
                    }
                }
#pragma unroll
                for (int d0 = 0; d0 < 8; d0 += AHEAD) {
#pragma unroll
                    for (int d = 0; d < AHEAD && d0 > 0; ++d)
                        ldsm4_trans(vt + ((d0 + d) >> 2) * KV_HALF + swz(vr, ((d0 + d) & 3) * 2 + vc), bf[d]);
                    if (valid < KW) {                             // zeros for the rows behind the last state
#pragma unroll
                        for (int d = 0; d < AHEAD; ++d)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int key = (lane & 3) * 2 + (e & 1) * 8;
                                if (key >= valid) bf[d][e] = 0;
                                else if (key + 1 >= valid) bf[d][e] &= 0xffffu;
                            }
                    }
#pragma unroll
                    for (int d = 0; d < AHEAD; ++d)
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma16816(o[mt][2 * (d0 + d)], pf[mt], bf[d][0], bf[d][1]);
                            mma16816(o[mt][2 * (d0 + d) + 1], pf[mt], bf[d][2], bf[d][3]);
                        }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        if (!ok) drain_in_flight();
        // every warp has read its last tile: the ring becomes the partial results
        named_bar_sync(1, ROW_WARPS * 32);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hi = 0; hi < 2; ++hi) {
                const int r = mt * 16 + (lane >> 2) + hi * 8;
                float sum = l[mt][hi];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                if ((lane & 3) == 0) {
                    ml[warp * C::ROWS + r] = m[mt][hi];
                    ml[(ROW_WARPS + 1 + warp) * C::ROWS + r] = sum;
                }
                if (r < rows) {
#pragma unroll
                    for (int d = 0; d < 16; ++d)
                        *reinterpret_cast<float2 *>(o_part + (warp * C::ROWS + r) * C::PITCH + d * 8 + (lane & 3) * 2) =
                            make_float2(o[mt][d][2 * hi], o[mt][d][2 * hi + 1]);
                }
            }
        named_bar_sync(1, ROW_WARPS * 32);
        // the warps' results as one
        float *sum_o = o_part + ROW_WARPS * C::ROWS * C::PITCH;
        for (int i = threadIdx.x; i < rows * (HD / 4); i += ROW_WARPS * 32) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < ROW_WARPS; ++w) top = fmaxf(top, ml[w * C::ROWS + r]);
            const float base = top == -INFINITY ? 0.f : top;
            float lt = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < ROW_WARPS; ++w) {
                const float f = ex2(ml[w * C::ROWS + r] - base);
                const float4 v = *reinterpret_cast<const float4 *>(o_part + (w * C::ROWS + r) * C::PITCH + d);
                lt += ml[(ROW_WARPS + 1 + w) * C::ROWS + r] * f;
                acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
            }
            *reinterpret_cast<float4 *>(sum_o + r * C::PITCH + d) = acc;
            if (d == 0) {
                ml[ROW_WARPS * C::ROWS + r] = top;
                ml[(2 * ROW_WARPS + 1) * C::ROWS + r] = lt;
            }
        }
    }
    __syncwarp();
    if (split > 1) cluster_sync();
    else __syncthreads();
    // the cluster's results as one, in rank order; each CTA stores its share of the rows' columns
    {
        const uint32_t m_at = smem_u32(ml + ROW_WARPS * C::ROWS), l_at = smem_u32(ml + (2 * ROW_WARPS + 1) * C::ROWS);
        const uint32_t o_at = smem_u32(o_part + ROW_WARPS * C::ROWS * C::PITCH);
        for (int i = rank * ROW_THREADS + threadIdx.x; i < rows * (HD / 4); i += split * ROW_THREADS) {
            const int r = i / (HD / 4), d = (i % (HD / 4)) * 4;
            float mr[MAX_SPLIT], top = -INFINITY;
#pragma unroll
            for (int c = 0; c < MAX_SPLIT; ++c)
                if (c < split) mr[c] = ld_cluster_f32(m_at + r * 4, c);
#pragma unroll
            for (int c = 0; c < MAX_SPLIT; ++c)
                if (c < split) top = fmaxf(top, mr[c]);
            const float base = top == -INFINITY ? 0.f : top;
            float lt = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            // eight ranks' pieces are requested before the first is needed
#pragma unroll
            for (int c0 = 0; c0 < MAX_SPLIT; c0 += 8) {
                float lr[8];
                float4 v[8];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (c0 + c < split) {
                        lr[c] = ld_cluster_f32(l_at + r * 4, c0 + c);
                        v[c] = ld_cluster_f4(o_at + (r * C::PITCH + d) * 4, c0 + c);
                    }
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (c0 + c < split) {
                        const float f = ex2(mr[c0 + c] - base);
                        lt += lr[c] * f;
                        acc.x += v[c].x * f, acc.y += v[c].y * f, acc.z += v[c].z * f, acc.w += v[c].w * f;
                    }
            }
            const float inv = lt == 0.f ? 0.f : 1.0f / lt;        // no state, or none with a finite score
            const float f[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
            *reinterpret_cast<uint2 *>(p.out + row_at(r, p.o_b, p.o_s, p.o_h) + d) = pack4(f);
        }
    }
    if (split > 1) cluster_sync();   // no CTA leaves while another reads its shared memory
}

}  // namespace cross
}  // namespace h3

using namespace h3;

namespace {

// [B, S, H, 128] BF16 view; zero_batch: a batch stride of 0 (one sample for all) is allowed
int check_operand(const h3_tensor *t, bool zero_batch) {
    H3_CHECK(check_bf16(t));
    if (t->ndim != 4 || t->shape[3] != cross::HD) return H3_ERR_BAD_SHAPE;
    if (numel(t) == 0) return H3_OK;
    if (t->strides[3] != 1 || !aligned16(t->data)) return H3_ERR_BAD_LAYOUT;
    for (int i = 0; i < 3; ++i)
        if (t->shape[i] > 1 && (t->strides[i] % 8 != 0 || t->strides[i] < 0 ||
                                (t->strides[i] == 0 && !(i == 0 && zero_batch))))
            return H3_ERR_BAD_LAYOUT;
    if (t->shape[1] > 0x3fffffffLL || t->shape[2] > 65535 || t->shape[0] > 65535) return H3_ERR_UNSUPPORTED;
    return H3_OK;
}

// tensor map (D, S, H, B) with boxes of 64 columns x `rows` positions
int heads_tmap(CUtensorMap *map, const h3_tensor *t, int64_t batch, unsigned rows) {
    const cuuint64_t dims[4] = {(cuuint64_t)t->shape[3], (cuuint64_t)t->shape[1], (cuuint64_t)t->shape[2],
                                (cuuint64_t)batch};
    // a dimension of size 1 may carry any stride; give TMA a legal one
    const int64_t ss = t->shape[1] == 1 ? 128 : t->strides[1];
    const int64_t sh = t->shape[2] == 1 ? 128 : t->strides[2];
    const int64_t sb = batch == 1 ? 128 : t->strides[0];
    const cuuint64_t strides[3] = {(cuuint64_t)ss * 2, (cuuint64_t)sh * 2, (cuuint64_t)sb * 2};
    const cuuint32_t box[4] = {64, rows, 1, 1};
    return make_tmap_bf16(map, t->data, 4, dims, strides, box);
}

// Form of the cross attention (h3_cross_attention_variant): 0 chooses per launch, 1 forces
// the rows form, 2 the tile form.
std::atomic<int> g_variant{0};

template <int NQ>
int launch_tiles(const h3_tensor *out, const h3_tensor *q, const h3_tensor *k, const h3_tensor *v, cross::Params &p,
                 cudaStream_t stream) {
    using C = cross::Tile<NQ>;
    CUtensorMap tq, tk, tv, to;
    H3_CHECK(heads_tmap(&tq, q, p.B, cross::BM));
    H3_CHECK(heads_tmap(&to, out, p.B, cross::BM));
    if (p.Sk > 0) {
        H3_CHECK(heads_tmap(&tk, k, p.kv_shared ? 1 : p.B, cross::BN));
        H3_CHECK(heads_tmap(&tv, v, p.kv_shared ? 1 : p.B, cross::BN));
    } else {
        tk = tv = tq;   // never loaded from
    }
    static std::atomic<bool> ready[64];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return H3_ERR_UNSUPPORTED;
    if (!ready[dev].load()) {
        if (cudaFuncSetAttribute(cross::tile_kernel<NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) !=
            cudaSuccess)
            return H3_ERR_LAUNCH;
        ready[dev].store(true);
    }
    p.per_head = (p.Sq + NQ * cross::BM - 1) / (NQ * cross::BM);
    const int64_t items = (int64_t)p.per_head * p.H * p.B;
    if (items > 0x3fffffff) return H3_ERR_UNSUPPORTED;
    p.items = (int)items;
    const int grid = p.items < num_sms() ? p.items : num_sms();
    // with a length per sample items differ in cost: dealt in descending order they level out
    p.ordered = p.lens && p.B > 1 && p.B <= cross::MAX_ORDERED && p.items > grid;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr = overlapped_launch();
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(cross::TILE_THREADS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, cross::tile_kernel<NQ>, tq, tk, tv, to, p) != cudaSuccess) {
        cudaGetLastError();
        return H3_ERR_LAUNCH;
    }
    return launch_status();
}

template <int MT, int WARPS>
void rows_config(cudaLaunchConfig_t *cfg, cudaLaunchAttribute *attr) {
    using C = cross::Rows<MT, WARPS>;
    attr->id = cudaLaunchAttributeClusterDimension;
    attr->val.clusterDim.x = 1;
    attr->val.clusterDim.y = 1;
    attr->val.clusterDim.z = 1;
    cfg->blockDim = dim3(C::THREADS);
    cfg->dynamicSmemBytes = C::SMEM;
    cfg->attrs = attr;
    cfg->numAttrs = 1;
}

// In how many shares the keys of `groups` (sample, key/value head, row chunk) groups are
// taken: as many as run in one wave and have a key tile each.  0: the device cannot say.
template <int MT, int WARPS>
int rows_split(int64_t groups, int Sk) {
    using C = cross::Rows<MT, WARPS>;
    auto kernel = cross::rows_kernel<MT, WARPS>;
    // per device: clusters of 1..16 CTAs resident at once (a cluster stays within one group
    // of SMs, so large ones leave SMs empty: 148 SMs hold 15 clusters of 8 one-CTA SMs)
    static std::atomic<int> resident[64][cross::MAX_SPLIT + 1];
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return 0;
    if (resident[dev][1].load() == 0) {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr;
        rows_config<MT, WARPS>(&cfg, &attr);
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess ||
            cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return 0;
        for (int c = cross::MAX_SPLIT; c >= 1; --c) {
            attr.val.clusterDim.x = c;
            cfg.gridDim = dim3(c, 1024, 1);
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();
                n = 0;
            }
            resident[dev][c].store(n);
        }
        if (resident[dev][1].load() < 1) return 0;
    }
    const int tiles = (Sk + C::KEYS - 1) / C::KEYS;
    int split = tiles < 1 ? 1 : tiles < cross::MAX_SPLIT ? tiles : cross::MAX_SPLIT;
    while (split > 1 && resident[dev][split].load() < groups) --split;
    return split;
}

template <int MT, int WARPS>
int launch_rows(const h3_tensor *k, const h3_tensor *v, cross::Params &p, cudaStream_t stream) {
    using C = cross::Rows<MT, WARPS>;
    CUtensorMap tk{}, tv{};
    if (p.Sk > 0) {
        H3_CHECK(heads_tmap(&tk, k, p.kv_shared ? 1 : p.B, C::KEYS));
        H3_CHECK(heads_tmap(&tv, v, p.kv_shared ? 1 : p.B, C::KEYS));
    }
    p.chunks = (p.rows + C::ROWS - 1) / C::ROWS;
    const int64_t groups = (int64_t)(p.fold ? 1 : p.B) * p.kv_heads * p.chunks;
    if (groups > 65535) return H3_ERR_UNSUPPORTED;
    const int split = rows_split<MT, WARPS>(groups, p.Sk);
    if (split < 1) return H3_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    rows_config<MT, WARPS>(&cfg, attr);
    attr[0].val.clusterDim.x = split;
    attr[1] = overlapped_launch();
    cfg.numAttrs = 2;
    cfg.gridDim = dim3(split, (unsigned)groups, 1);
    cfg.stream = stream;
    if (cudaLaunchKernelEx(&cfg, cross::rows_kernel<MT, WARPS>, tk, tv, p) != cudaSuccess) {
        cudaGetLastError();
        return H3_ERR_LAUNCH;
    }
    return launch_status();
}

// Whether the rows form takes less time than the tile form, from the times of one step of
// either measured on B200 (us): a key tile of the rows form 1.05 (16 rows, 128 keys, one
// CTA per SM), 1.45 (16 rows, 64 keys, two) or 1.1 (32 rows, 64 keys); 128 keys of one Q tile
// 1.47, of two 2.07, and 1.5 to store an item; the rest of a launch 5 to 9.5.  Checked at
// 16..512 queries, 512..18432 states, 2..640 groups: e.g. 32 queries, 40 heads, 512 states
// 12.9 us in rows and 10.8 in tiles, 2304 states 23.1 and 31.5; 512 queries of 2 heads over
// 18432 states 79 and 207.
bool rows_form(const cross::Params &p, int64_t rows, int64_t groups) {
    const int sms = num_sms();
    const int64_t tiles = (p.Sq + cross::BM - 1) / cross::BM, heads = (int64_t)p.H * p.B;
    const double nkv = (p.Sk + 127) / 128;
    const bool two = tiles > 1 && tiles * heads > sms;
    const int64_t items = two ? (tiles + 1) / 2 * heads : tiles * heads;
    const double waves = (double)((items + sms - 1) / sms);
    const double in_tiles = 5.0 + waves * (nkv * (two ? 2.07 : 1.47) + 1.5);
    double in_rows;
    if (rows <= 16) {
        in_rows = groups <= sms ? 6.0 + (nkv / (rows_split<1, 8>(groups, p.Sk) + 1e-9) + 0.5) * 1.05
                                : 6.0 + (double)((groups + 2 * sms - 1) / (2 * sms)) * 2 * nkv * 1.45;
    } else {
        const double per = 2 * nkv / (rows_split<2, 4>(groups, p.Sk) + 1e-9) + 0.5;
        in_rows = 9.5 + (double)((groups + sms - 1) / sms) * per * 1.1;
    }
    return in_rows < in_tiles;
}

}  // namespace

extern "C" int h3_cross_attention_variant(int variant) {
    if (variant < 0 || variant > 2) return -1;
    return g_variant.exchange(variant);
}

extern "C" int h3_cross_attention(const h3_tensor *out, const h3_tensor *q, const h3_tensor *k, const h3_tensor *v,
                                  const h3_tensor *lengths, float scale, void *stream) {
    H3_CHECK(check_operand(out, false));
    H3_CHECK(check_operand(q, false));
    H3_CHECK(check_operand(k, true));
    H3_CHECK(check_operand(v, true));
    H3_CHECK(check_same_shape(out, q));
    H3_CHECK(check_same_shape(k, v));
    const int64_t B = q->shape[0], H = q->shape[2], Hkv = k->shape[2];
    if (k->shape[0] != B && k->shape[0] != 1) return H3_ERR_BAD_SHAPE;
    if (H > 0 && (Hkv < 1 || H % Hkv != 0)) return H3_ERR_BAD_SHAPE;
    if (lengths) {
        H3_CHECK(check_desc(lengths, H3_I64));
        if (lengths->ndim != 1 || lengths->shape[0] != B) return H3_ERR_BAD_SHAPE;
        if (B > 1 && lengths->strides[0] != 1) return H3_ERR_BAD_LAYOUT;
    }
    if (!(scale > 0.f) || !(scale <= H3_CROSS_SCALE_MAX)) return H3_ERR_UNSUPPORTED;
    if (numel(q) == 0) return H3_OK;
    cross::Params p{};
    p.B = (int)B;
    p.Sq = (int)q->shape[1];
    p.Sk = (int)k->shape[1];
    p.H = (int)H;
    p.kv_heads = (int)Hkv;
    p.group = (int)(H / Hkv);
    // K and V of one sample for all: batch size 1, or a broadcast batch (both of them)
    const bool k1 = k->shape[0] == 1 || k->strides[0] == 0, v1 = v->shape[0] == 1 || v->strides[0] == 0;
    p.kv_shared = B > 1 && p.Sk > 0 && k1;
    if (B > 1 && p.Sk > 0 && k1 != v1) return H3_ERR_BAD_LAYOUT;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.lens = lengths ? static_cast<const int64_t *>(lengths->data) : nullptr;
    p.q = static_cast<const __nv_bfloat16 *>(q->data);
    p.out = static_cast<__nv_bfloat16 *>(out->data);
    p.q_b = q->strides[0], p.q_s = q->strides[1], p.q_h = q->strides[2];
    p.o_b = out->strides[0], p.o_s = out->strides[1], p.o_h = out->strides[2];
    // samples that share K, V and their length are rows of one product
    p.fold = p.kv_shared && !p.lens;
    const int64_t rows = (int64_t)p.Sq * p.group * (p.fold ? B : 1);
    const int variant = g_variant.load();
    const int64_t groups = (p.fold ? 1 : B) * Hkv * (rows <= 16 ? 1 : (rows + 31) / 32);
    const bool fits = groups <= 65535 && rows <= 0x3fffffff;
    if (fits && (variant == 1 || (variant == 0 && rows_form(p, rows, groups)))) {
        p.rows = (int)rows;
        if (rows > 16) return launch_rows<2, 4>(k, v, p, (cudaStream_t)stream);
        // Eight warps fill an SM on their own, four leave room for a second CTA.  Measured at one
        // query, 18432 states, 8 key/value heads (clusters of 10): 18.5 us with eight, 21.5 with four;
        // at 160 (sample, head) groups of 512 states, more than there are SMs: 15.6 and 11.3 us.
        return groups <= num_sms() ? launch_rows<1, 8>(k, v, p, (cudaStream_t)stream)
                                   : launch_rows<1, 4>(k, v, p, (cudaStream_t)stream);
    }
    // one Q tile per item where that leaves no SM more than its share, two otherwise
    const int64_t tiles = (int64_t)(p.Sq + cross::BM - 1) / cross::BM;
    if (tiles == 1 || tiles * H * B <= num_sms()) return launch_tiles<1>(out, q, k, v, p, (cudaStream_t)stream);
    return launch_tiles<2>(out, q, k, v, p, (cudaStream_t)stream);
}

// device error word of this translation unit (bounded waits of the cross attention)
extern "C" unsigned int h3_cross_device_error_read_and_clear(void) {
    unsigned int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, h3::g_h3_device_error, sizeof(v));
    cudaMemcpyToSymbol(h3::g_h3_device_error, &zero, sizeof(zero));
    return v;
}
