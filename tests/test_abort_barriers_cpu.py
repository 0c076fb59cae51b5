"""After a wait that gave up, all warps of a softmax group pass the same named barriers.

A named barrier waits for its 128 threads without a limit, and the four warps of a group
learn one by one that a bounded wait gave up: one may still pass a wait that another has
given up on.  The group's code is taken from the kernel's source and run on the host, a
warp at a time, with every wait's outcome chosen: from the first wait that gives up on,
each later one may give up too or may still pass.  All warps have to reach the same number
of barriers, and a tile that a warp has not finished must not be stored.
"""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = next(Path(__file__).resolve().parent.parent.glob("minimaxh3*/csrc"))

HARNESS = r"""
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <algorithm>
using std::min;
#define __device__
#define __forceinline__ inline

// ---- what the group's code uses, for lane 0 of a warp
static int g_waits, g_fail_at, g_after, g_barriers, g_stores, g_bad_stores, g_unfinished;
static int g_abort;                       // the CTA's flag
static bool mbar_wait(uint64_t *, uint32_t, volatile int *abort) {
    const int at = g_waits++;
    if (at < g_fail_at) return true;
    if (at > g_fail_at && g_after) return true;     // passes although another has given up
    *abort = 1;
    g_unfinished = 1;
    return false;
}
static void named_bar_sync(int, int) { ++g_barriers; }
static bool __all_sync(unsigned, bool v) { return v; }
static bool __any_sync(unsigned, bool v) { return v; }
static void __syncwarp() {}
static void tc_fence_after() {}
static void tc_fence_before() {}
static void tmem_ld_wait() {}
static void tmem_st_wait() {}
static void fence_proxy_async_smem() {}
static void mbar_arrive(uint64_t *) {}
static void drain_in_flight() {}
static void tma_store_wait_read() {}
static void tma_store_wait_all() {}
static void tma_store_commit() {}
template <typename... A> static void tma_store_4d(A...) { ++g_stores; g_bad_stores += g_unfinished; }
static void tmem_ld32(uint32_t, uint32_t (&r)[32]) { std::memset(r, 0, sizeof r); }
static void tmem_st32(uint32_t, const uint32_t (&)[32]) {}
static void st_shared_v4(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) {}
struct uint4 { uint32_t x, y, z, w; };
static uint4 ld_shared_v4(uint32_t) { return {}; }
template <typename T> static void st_global_v4(T *, const uint4 &) { ++g_stores; g_bad_stores += g_unfinished; }
static uint32_t smem_u32(const void *) { return 0; }
static uint32_t swz(int, int) { return 0; }
static uint32_t pack_bf16x2(float, float) { return 0; }
static float ex2(float) { return 1.f; }
static float max3f(float a, float b, float c) { return std::max(a, std::max(b, c)); }
static uint64_t pk2(float, float) { return 0; }
static void up2(uint64_t, float &a, float &b) { a = b = 0.f; }
static uint64_t ffma2(uint64_t, uint64_t, uint64_t) { return 0; }
static uint64_t fadd2(uint64_t, uint64_t) { return 0; }
static void exp2_poly2(float, float, float &a, float &b) { a = b = 0.f; }
static float bf16_round_up(float x) { return x; }
static float __uint_as_float(uint32_t) { return 0.f; }
static uint32_t __float_as_uint(float) { return 0; }
static struct { int x; } blockIdx, gridDim = {1};
typedef uint16_t __nv_bfloat16;

constexpr int BM = 128, BN = 128, HD = 128, TILE_BYTES = 32768, HALF = 16384;
constexpr float RESCALE_THRESHOLD = 8.f;
static const int LENS[] = {%(lens)s};
constexpr int ITEMS = sizeof LENS / sizeof LENS[0];

%(setup)s

static void group(const int warp, const int lane) {
    volatile int *abort_flag = &g_abort;
    uint64_t bars[8] = {};
    uint64_t *s_full = bars, *s_free = bars + 2, *p_ready = bars + 4, *o_done = bars + 6;
    uint32_t tmem = 0;
    uint8_t smem[1] = {};
    bool ok = true;
    {
%(code)s
    }
}

int main() {
    int wrong = 0;
    for (int mode = 0; mode < %(modes)s; ++mode) {
        set_mode(mode);
        // a run in which no wait gives up
        g_waits = g_barriers = g_stores = g_abort = g_unfinished = 0, g_fail_at = 1 << 30;
        group(4, 0);
        const int waits = g_waits, barriers = g_barriers, stores = g_stores;
        if (!waits || !barriers || !stores) return std::puts("nothing was run"), 2;
        for (int at = 0; at < waits; ++at)
            for (int after = 0; after < 2; ++after) {
                g_abort = g_unfinished = g_bad_stores = 0;
                // warp 3 of the group gives up at its wait `at`; warp 0, which stores, passes all
                g_waits = g_barriers = g_stores = 0, g_fail_at = at, g_after = after;
                group(7, 0);
                const int mine = g_barriers;
                g_waits = g_barriers = g_stores = 0, g_fail_at = 1 << 30;
                group(4, 0);
                const int others = g_barriers;
                if (mine != others || others != barriers || g_bad_stores) {
                    std::printf("mode %%d, wait %%d of %%d: %%d barriers, the others %%d (%%d), %%d stores of unfinished tiles\n", mode,
                                at, waits, mine, others, barriers, g_bad_stores);
                    ++wrong;
                }
            }
    }
    return wrong != 0;
}
"""


def _branch(text: str, start: str) -> str:
    """From ``start`` to the closing brace of the block it stands in."""
    at = text.index(start)
    depth, i = 0, at
    while depth >= 0:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
    return text[at:i - 1]


def _run(tmp_path, code, lens, setup, modes=1):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no host compiler")
    src = tmp_path / "group.cpp"
    src.write_text(HARNESS % dict(lens=", ".join(map(str, lens)), code=code, setup=setup, modes=modes))
    exe = tmp_path / "group"
    built = subprocess.run([gxx, "-std=c++17", "-O1", "-w", str(src), "-o", str(exe)], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr[:4000]
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0, ran.stdout[-2000:]


CROSS = r"""
constexpr int NQ = 2;
struct C { static constexpr int OFF_P = 0, O_COL = 256; };
struct Params { int items, Sq; float scale_log2; };
static Params p = {ITEMS, 1 << 20, 1.f};
static int to;
static void set_mode(int) {}
static void item_at(int i, int &b, int &h, int &q0, int &len) { b = h = q0 = 0, len = LENS[i]; }
"""


def test_cross_attention_tile_form(tmp_path):
    """Items of several key tiles, of one, of none, first, last and in between."""
    text = (CSRC / "cross_attention_sm100.cu").read_text()
    code = _branch(text, "const int t = (warp - 4) >> 2;")
    for lens in ((300, 0, 128, 0, 0, 129, 1), (0, 500), (77, 0), (1000,)):
        _run(tmp_path, code, lens, CROSS)


ATTENTION = r"""
#define H3_ATTN_MAX_ACC 4
#define H3_ATTN_MAX_BF16 0
#define H3_ATTN_EARLY_P %d
constexpr int O_COL = 256, TILE = TILE_BYTES, SUM_GROUPS = 2, GROUP_PAIRS = 32, POLY_PAIRS = 0;
struct Params { int Sq, Sk, ndst, rows_per_dst; float scale_log2; int64_t d_row, d_head; __nv_bfloat16 *dst[1]; };
static Params p = {1 << 20, 0, 0, 1 << 20, 1.f};
static int to, nkv;
static const int q0 = 0, h = 0, b = 0;
static uint8_t sQ[1 << 17], sP[1 << 17];
// number of key tiles, and whether the rows go to one tensor or to their owners
static void set_mode(int m) { p.ndst = m %% 2, nkv = m / 2 + 1, p.Sk = nkv * BN; }
"""


@pytest.mark.parametrize("early_p", [0, 1])
def test_self_attention(tmp_path, early_p):
    text = (CSRC / "attention_sm100.cu").read_text()
    code = _branch(text, "const int t = (warp - 4) >> 2;")
    _run(tmp_path, code, (0,), ATTENTION % early_p, modes=8)
