"""Microscaled 4-bit quantisation and projections against the 64-bit oracle.

Quantisation is exact arithmetic followed by one rounding that the formats define, so
codes and scales must equal the oracle's.  A projection of given 4-bit operands differs
from the exact sum by its fp32 accumulation and one BF16 rounding:

* BF16: at most half a step, 2^-8 of the value;
* accumulation: the tensor core adds the 64 products of an instruction to the running
  sum with at least 23 fractional bits of the largest term kept, i.e. an error below
  2 * 2^-23 of the sum of magnitudes so far; K/64 instructions, plus up to 8 partial sums
  joined and the bias added in fp32: (K/64 + 9) * 2^-22 of sum |x w| + |b| covers it.
"""
import pytest
import torch

from oracle import fp4_oracle as Q

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMATS = ("mxfp4", "nvfp4")


@pytest.fixture(scope="module")
def h3():
    import h3b200
    h3b200.load()
    assert h3b200._lib.host(), "the host extension is not built"
    return h3b200


@pytest.fixture
def ctypes_only(h3, monkeypatch):
    monkeypatch.setattr(h3._lib, "_host", False)


def _parts(h3, q):
    c, s = h3.unpack_fp4(q)
    return Q.nibbles(c.cpu(), q.cols), s.cpu().long()


def _check_quantized(h3, x, fmt, t=1.0):
    q = h3.quantize_fp4(x, fmt, t)
    code, byte = _parts(h3, q)
    want_code, want_byte = Q.quantize(x.reshape(-1, x.shape[-1]).cpu(), fmt, t)
    assert torch.equal(byte, want_byte.long())
    # -0 and +0 are the same value
    code, want_code = (torch.where(c == 8, 0, c) for c in (code, want_code))
    assert torch.equal(code, want_code)
    back = h3.dequantize_fp4(q).cpu().double()
    assert torch.equal(torch.nan_to_num(back, nan=7e77), torch.nan_to_num(Q.values(code, byte, fmt, t), nan=7e77))
    # columns past the last one: zero codes in every byte of the pitch
    tail = q.codes[:, (q.cols + 1) // 2:]
    assert int(tail.long().sum()) == 0
    return q


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 5120), (2, 15), (5, 16), (7, 17), (3, 31), (4, 32), (9, 33),
                                       (130, 64), (33, 100), (257, 1795), (128, 1792), (1000, 130), (300, 4096 + 8)])
def test_quantize(h3, fmt, rows, cols):
    g = torch.Generator(device=DEV).manual_seed(rows * 7 + cols)
    x = (torch.randn(rows, cols, generator=g, device=DEV) *
         torch.exp(torch.randn(cols, generator=g, device=DEV))).bfloat16()
    _check_quantized(h3, x, fmt)
    if fmt == "nvfp4":
        _check_quantized(h3, x, fmt, 2.0 ** -8)
        _check_quantized(h3, x, fmt, 4.0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_every_ratio(h3, fmt):
    """Every BF16 significand against every block maximum's significand, across the whole
    exponent range: all ties, subnormals and saturations occur."""
    sig = torch.arange(128, 256, device=DEV).float()
    size = Q.BLOCK[fmt]
    x = torch.zeros(128, 128 * 5, size, device=DEV)
    for i, e in enumerate((0, -1, -2, -3, -4)):
        block = x[:, 128 * i:128 * (i + 1)]
        block[..., 0] = sig[:, None]
        block[..., 1:] = (sig * 2.0 ** e)[None, :, None] * (1 - 2 * (torch.arange(size - 1, device=DEV) % 2))
    x = x.flatten(1)
    for scale in (2.0 ** -140, 2.0 ** -133, 2.0 ** -120, 2.0 ** -17, 2.0 ** -14, 2.0 ** -7, 1.0, 2.0 ** 4, 2.0 ** 100):
        _check_quantized(h3, (x * scale).bfloat16(), fmt)
    if fmt == "nvfp4":
        _check_quantized(h3, (x * 2.0 ** -60).bfloat16(), fmt, 2.0 ** -60)
        _check_quantized(h3, (x * 2.0 ** 60).bfloat16(), fmt, 2.0 ** 60)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_special_values(h3, fmt):
    x = torch.randn(6, 96, device=DEV).bfloat16()
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 40] = float("-inf")
    x[3, 95] = float("nan")
    x[4] = torch.finfo(torch.bfloat16).max
    x[5] = torch.finfo(torch.bfloat16).smallest_normal / 64
    q = _check_quantized(h3, x, fmt)
    back = h3.dequantize_fp4(q)
    size = Q.BLOCK[fmt]
    for r, c in ((1, 5), (2, 40), (3, 95)):
        assert bool(back[r, c // size * size:(c // size + 1) * size].isnan().all())
    assert int(back.isnan().sum()) == 3 * size


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_views_and_targets(h3, fmt):
    big = torch.randn(40, 3, 700, device=DEV).bfloat16()
    for x in (big[:, 1, 8:520], big[:, 1, 3:200], big[:, :, 16:80], big[0, 0:1, 1:2], big[:, 0, :].expand(40, 700)):
        _check_quantized(h3, x, fmt)
    # a broadcast row (stride 0)
    _check_quantized(h3, big[3, 0].expand(5, 700), fmt)
    # into views of larger buffers: what is around them stays
    q = h3.quantize_fp4(big[:, 0, :320], fmt)
    wide = torch.full((42, 192), 7, dtype=torch.uint8, device=DEV)
    held = h3.Fp4Tensor(wide[1:41, 16:176], torch.full_like(q.scales, 9), 40, 320, fmt)
    h3.quantize_fp4_(held, big[:, 0, :320])
    assert torch.equal(held.codes, q.codes)
    assert int((wide == 7).sum()) >= 42 * 192 - 40 * 160
    assert bool((wide[0] == 7).all() and (wide[41] == 7).all() and (wide[:, :16] == 7).all())
    out = torch.full((42, 400), 3.0, device=DEV).bfloat16()
    h3.dequantize_fp4_(out[1:41, 8:328], q)
    assert torch.equal(out[1:41, 8:328], h3.dequantize_fp4(q))
    assert bool((out[0] == 3).all() and (out[41] == 3).all() and (out[:, :8] == 3).all() and (out[:, 328:] == 3).all())
    odd = torch.full((42, 401), 3.0, device=DEV).bfloat16()
    h3.dequantize_fp4_(odd[1:41, 5:325], q)
    assert torch.equal(odd[1:41, 5:325], h3.dequantize_fp4(q)) and bool((odd[:, 325:] == 3).all())


def test_quantize_empty(h3):
    q = h3.quantize_fp4(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV))
    assert q.shape == (0, 64) and h3.dequantize_fp4(q).shape == (0, 64)


# ---------------------------------------------------------------------------
# projections
# ---------------------------------------------------------------------------
def _weight(h3, n, k, fmt, seed, t=None):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(n, k, generator=g, device=DEV) * 0.02).bfloat16()
    return h3.quantize_fp4(w, fmt, (2.0 ** -8 if t is None else t) if fmt == "nvfp4" else 1.0)


def _values(h3, q):
    return Q.values(*_parts(h3, q), q.format, q.tensor_scale).to(DEV)


def _check_product(y, xv, wv, bias=None):
    ref, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    bound = ref.abs() * 2.0 ** -8 + (xv.shape[1] / 64 + 9) * 2.0 ** -22 * mag
    err = (y.double() - ref).abs()
    worst = float((err / bound.clamp_min(1e-300)).max()) if err.numel() else 0.0
    assert bool((err <= bound).all()), f"error {worst:.3g} times its bound"


@pytest.fixture(params=[1, 2], ids=["swap", "tiles"])
def form(h3, request):
    old = h3.load().h3_fp4_variant(request.param)
    yield request.param
    h3.load().h3_fp4_variant(old)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 128, 256), (1, 1, 1), (1, 5120, 5120), (2, 3, 15), (15, 127, 32), (16, 128, 33),
                                   (17, 129, 64), (31, 200, 100), (32, 512, 255), (33, 256, 256), (63, 300, 257),
                                   (64, 128, 512), (65, 640, 1795), (127, 128, 320), (128, 256, 5120), (129, 130, 96),
                                   (255, 257, 1000), (256, 256, 256), (300, 1000, 768), (513, 777, 1300),
                                   (1111, 520, 2048)])
def test_linear(h3, form, fmt, M, N, K):
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    bias = torch.randn(N, generator=g, device=DEV).bfloat16()
    w = _weight(h3, N, K, fmt, 1)
    xq = h3.quantize_fp4(x, fmt)
    xv, wv = _values(h3, xq), _values(h3, w)
    y = h3.linear_fp4(x, w, bias)
    _check_product(y, xv, wv, bias)
    _check_product(h3.linear_fp4(x, w), xv, wv)
    yq = h3.linear_fp4(xq, w, bias)                        # the same rows quantised beforehand
    _check_product(yq, xv, wv, bias)
    if form == 1 or M > 8:                                 # up to 8 rows x is quantised inside form 1
        assert torch.equal(yq, y)
    assert torch.equal(h3.linear_fp4(x, w, bias), y)       # the same bits every time
    assert h3.load().h3_device_error() == 0


def test_linear_rows_do_not_mix(h3, form):
    """A NaN or an infinity in one row of x, or in one weight row, reaches that row or
    column of the result and no other."""
    for fmt in FORMATS:
        for M in (5, 300):
            x = torch.randn(M, 700, device=DEV).bfloat16()
            w = torch.randn(300, 700, device=DEV).bfloat16()
            good = h3.linear_fp4(x, h3.quantize_fp4(w, fmt))
            x[3, 650] = float("nan")
            w[140, 5] = float("inf")
            y = h3.linear_fp4(x, h3.quantize_fp4(w, fmt))
            bad = torch.zeros_like(y, dtype=torch.bool)
            bad[3], bad[:, 140] = True, True
            assert torch.equal(y.isnan(), bad)
            assert torch.equal(y[~bad], good[~bad])


def test_linear_layouts(h3, form):
    """Batched and strided x, strided out with its surroundings untouched, odd row pitch."""
    for fmt in FORMATS:
        w = _weight(h3, 333, 640, fmt, 2)
        big = torch.randn(3, 50, 700, device=DEV).bfloat16()
        x = big[:, :, 8:648]
        y = h3.linear_fp4(x, w)
        assert y.shape == (3, 50, 333)
        assert torch.equal(y.view(150, 333), h3.linear_fp4(x.reshape(150, 640), w))
        for width, c0 in ((500, 8), (501, 3)):
            for rows in (7, 150):
                out = torch.full((rows + 2, width), 5.0, device=DEV).bfloat16()
                h3.linear_fp4_(out[1:rows + 1, c0:c0 + 333], x.reshape(150, 640)[:rows], w)
                assert torch.equal(out[1:rows + 1, c0:c0 + 333], h3.linear_fp4(x.reshape(150, 640)[:rows], w))
                out[1:rows + 1, c0:c0 + 333] = 5.0
                assert bool((out == 5).all())


def test_linear_tensor_scales(h3):
    x = (torch.randn(70, 512, device=DEV) * 1e4).bfloat16()
    t = h3.fp4_tensor_scale(float(x.float().abs().max()))
    w = _weight(h3, 200, 512, "nvfp4", 3, t=2.0 ** -9)
    xq = h3.quantize_fp4(x, "nvfp4", t)
    y = h3.linear_fp4(x, w, x_tensor_scale=t)
    _check_product(y, _values(h3, xq), _values(h3, w))
    # the quantisation itself keeps what 4 bits can: half a step of 1/6 of the block's largest, at most
    assert float((h3.dequantize_fp4(xq).float() - x.float()).norm() / x.float().norm()) < 0.125


def test_linear_many_tiles(h3, form):
    """More tiles than the GPU holds at once: both accumulators and every ring slot are reused."""
    for fmt in FORMATS:
        x = torch.randn(4000, 1100, device=DEV).bfloat16()
        w = _weight(h3, 5000, 1100, fmt, 6)
        _check_product(h3.linear_fp4(x, w), _values(h3, h3.quantize_fp4(x, fmt)), _values(h3, w))
    assert h3.load().h3_device_error() == 0


def test_variant_refuses_unknown_forms(h3):
    assert h3.load().h3_fp4_variant(3) == -1 and h3.load().h3_fp4_variant(-1) == -1
    assert h3.load().h3_fp4_variant(0) == 0


def test_linear_empty(h3):
    w = _weight(h3, 64, 64, "mxfp4", 4)
    assert h3.linear_fp4(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), w).shape == (0, 64)


def test_linear_refusals(h3):
    w = _weight(h3, 64, 64, "nvfp4", 4)
    x = torch.randn(8, 64, device=DEV).bfloat16()
    with pytest.raises(ValueError, match="columns"):
        h3.linear_fp4(x[:, :32], w)
    with pytest.raises(ValueError, match="mxfp4"):
        h3.linear_fp4(h3.quantize_fp4(x, "mxfp4"), w)
    with pytest.raises(ValueError):
        h3.linear_fp4(x.float(), w)
    with pytest.raises(ValueError):
        h3.linear_fp4(x, w, bias=torch.zeros(63, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="tensor scale"):
        h3.linear_fp4(x, w, x_tensor_scale=3.0)
    with pytest.raises(ValueError, match="copy"):
        h3.linear_fp4_(torch.empty(64, 4, 2, dtype=torch.bfloat16, device=DEV).permute(2, 1, 0), x.view(2, 4, 64), w)


def test_graph_and_streams(h3, form):
    """Captured and replayed with new inputs, and run on two streams at once."""
    w = _weight(h3, 512, 1024, "nvfp4", 5)
    xs = [torch.randn(m, 1024, device=DEV).bfloat16() for m in (4, 200)]
    want = [h3.linear_fp4(x, w) for x in xs]
    for x, ref in zip(xs, want):
        inp = torch.zeros_like(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            h3.linear_fp4(inp, w)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = h3.linear_fp4(inp, w)
        for _ in range(3):
            inp.copy_(x)
            graph.replay()
            assert torch.equal(y, ref)
            inp.zero_()
            graph.replay()
            assert int(y.count_nonzero()) == 0
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    outs = [[] for _ in xs]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(h3.linear_fp4(xs[i], w))
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        assert all(torch.equal(y, ref) for y in got)
    assert h3.load().h3_device_error() == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_both_ways_of_calling_agree(h3, monkeypatch, fmt):
    """The extension's calls and the ctypes ones: the same bits, shapes and errors."""
    x = torch.randn(3, 41, 700, device=DEV).bfloat16()
    w = _weight(h3, 100, 700, fmt, 7)
    bias = torch.randn(100, device=DEV).bfloat16()
    inputs = (x, x[0], x[0, :5], x[:, :, 5:], x[0, :, 5:], x[0, 1:2], x[:0], x.transpose(0, 1))

    def all_of(t):
        q = h3.quantize_fp4(t, fmt)
        p = h3.quantize_fp4(torch.nn.functional.pad(t, (0, 700 - t.shape[-1])), fmt)
        y = h3.linear_fp4(torch.nn.functional.pad(t, (0, 700 - t.shape[-1])), w, bias)
        return [*h3.unpack_fp4(q), h3.dequantize_fp4(q), h3.linear_fp4(p, w, bias), y, y.new_tensor(y.shape)]

    n = h3._lib.CALLS["n"]
    fast = [all_of(t) for t in inputs]
    made = h3._lib.CALLS["n"] - n
    monkeypatch.setattr(h3._lib, "_host", False)
    n = h3._lib.CALLS["n"]
    slow = [all_of(t) for t in inputs]
    assert h3._lib.CALLS["n"] - n == made
    for a, b in zip(fast, slow):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_refusals_without_the_extension(h3, ctypes_only):
    test_linear_refusals(h3)


def test_other_device_is_refused(h3):
    """Tensors of a device that is not the current one (here: the CPU) never reach a launch."""
    w = _weight(h3, 64, 64, "nvfp4", 4)
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for f in (lambda: h3.linear_fp4(x, w), lambda: h3.quantize_fp4(x),
              lambda: h3.linear_fp4(x.to(DEV), w, bias=torch.zeros(64, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("M", [1, 4, 12, 40, 300, 1500])
def test_calls_back_to_back(h3, M):
    """Kernels overlap the end of the one before them in the stream; what that one writes --
    the weights, the rows, the bias, all into the same buffers every time -- must be seen,
    and what it still reads must not be overwritten."""
    for fmt in FORMATS:
        ws = [(torch.randn(640, 1100, device=DEV) * 0.02).bfloat16() for _ in range(6)]
        xs = [torch.randn(M, 1100, device=DEV).bfloat16() for _ in range(6)]
        bs = [torch.randn(640, device=DEV).bfloat16() for _ in range(6)]
        want = []
        for w, x, b in zip(ws, xs, bs):
            torch.cuda.synchronize()
            q = h3.quantize_fp4(w, fmt)
            torch.cuda.synchronize()
            want.append(h3.linear_fp4(x, q, b))
            torch.cuda.synchronize()
        weight, x, bias = h3.fp4_empty(640, 1100, fmt), torch.zeros_like(xs[0]), torch.zeros_like(bs[0])
        xq, y = h3.fp4_empty(M, 1100, fmt), torch.zeros_like(want[0])
        got = []
        for i in range(60):
            bias.copy_(bs[i % 6])
            x.copy_(xs[i % 6])
            h3.quantize_fp4_(weight, ws[i % 6])
            h3.linear_fp4_(y, x, weight, bias)
            got.append(y.clone())
            if M > 8:
                h3.quantize_fp4_(xq, x)
                h3.linear_fp4_(y, xq, weight, bias)
                got.append(y.clone())
        per = 2 if M > 8 else 1
        assert all(torch.equal(o, want[i // per % 6]) for i, o in enumerate(got))
    assert h3.load().h3_device_error() == 0


def test_offsets_past_32_bits(h3):
    """Matrices of more than 2^31 elements: the last rows come out as on their own."""
    x = torch.zeros(420000, 5120, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, 5120, device=DEV).bfloat16()
    q = h3.quantize_fp4(x, "nvfp4")
    tail = h3.dequantize_fp4(q)[-3:].clone()
    assert torch.equal(tail, h3.dequantize_fp4(h3.quantize_fp4(x[-3:].clone(), "nvfp4")))
    del q, x
    w = _weight(h3, 27648, 64, "mxfp4", 8)
    x = torch.randn(80000, 64, device=DEV).bfloat16()
    y = h3.linear_fp4(x, w)                          # 2.2e9 results, in tiles
    h3.load().h3_fp4_variant(2)
    try:
        assert torch.equal(y[-300:], h3.linear_fp4(x[-300:].clone(), w))
    finally:
        h3.load().h3_fp4_variant(0)
    assert h3.load().h3_device_error() == 0
