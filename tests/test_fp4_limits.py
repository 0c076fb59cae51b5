"""The ends of the 4-bit projections' ranges: tensor scales, rows, outputs and columns."""
import ctypes

import pytest
import torch

DEV = "cuda"
H3_ERR_UNSUPPORTED = 5


@pytest.fixture(scope="module")
def h3():
    import h3b200
    return h3b200


def _bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_scales_that_overflow_together_are_refused_by_the_entry_points(h3):
    """2^64 times 2^64 is infinite in fp32, and a sum of 0 times that NaN.  (A weight without
    rows: what is accepted has nothing to do.)"""
    lib, d = h3.load(), h3._lib.desc
    x, w, y = _bf16(4, 48), h3.fp4_empty(0, 48, "nvfp4", device="cpu"), _bf16(4, 0)
    xq, work = h3.fp4_empty(4, 48, "nvfp4", device="cpu"), torch.zeros(1024, dtype=torch.uint8)

    def status(tx, tw, quantized, workspace=work):
        ref = lambda t: None if t is None else ctypes.byref(d(t))  # noqa: E731
        if quantized:
            return lib.h3_linear_fp4_quantized(*[ref(t) for t in (y, xq.codes, xq.scales, w.codes, w.scales, None)], 48,
                                               1, tx, tw, None)
        return lib.h3_linear_fp4(*[ref(t) for t in (y, x, workspace, w.codes, w.scales, None)], 1, tx, tw, None)

    for args in ((True,), (False,), (False, None)):
        assert status(2.0 ** 64, 2.0 ** 64, *args) == H3_ERR_UNSUPPORTED
        assert status(2.0 ** 64, 2.0 ** 63, *args) == 0 and status(2.0 ** 63, 2.0 ** 64, *args) == 0
        assert status(2.0 ** -64, 2.0 ** -64, *args) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 8, 40, 200, 1000])
def test_largest_and_smallest_scales(h3, M):
    """Products at the ends of the range: rows of zeros give the bias, and a single product
    (code 6 times code 6 at the block scale that keeps it in fp32) is rounded once."""
    bias = torch.randn(300, device=DEV).bfloat16()
    for tx, tw, block in ((2.0 ** 64, 2.0 ** 63, 2.0 ** -9), (2.0 ** 63, 2.0 ** 64, 2.0 ** -9),
                          (2.0 ** -64, 2.0 ** -64, 448.0)):
        x, weight = torch.zeros(M, 64, device=DEV), torch.zeros(300, 64, device=DEV)
        x[:, 5], weight[:, 5] = 6 * block * tx, 6 * block * tw
        w = h3.quantize_fp4(weight.bfloat16(), "nvfp4", tw)
        zeros = torch.zeros(M, 64, device=DEV).bfloat16()
        for rows, value in ((zeros, None), (x.bfloat16(), (6 * block) ** 2 * tx * tw)):
            want = bias.expand(M, -1) if value is None else torch.full((M, 300), value, device=DEV).bfloat16()
            add = bias if value is None else None
            assert torch.equal(h3.linear_fp4(rows, w, add, x_tensor_scale=tx), want)
            assert torch.equal(h3.linear_fp4(h3.quantize_fp4(rows, "nvfp4", tx), w, add), want)
    assert h3.load().h3_device_error() == 0


@pytest.mark.gpu
def test_scales_that_overflow_together_are_refused(h3):
    w = h3.fp4_empty(64, 64, "nvfp4", 2.0 ** 64)
    for M in (4, 40):
        x = torch.zeros(M, 64, dtype=torch.bfloat16, device=DEV)
        with pytest.raises(ValueError, match="multiply"):
            h3.linear_fp4(x, w, x_tensor_scale=2.0 ** 64)
        with pytest.raises(ValueError, match="multiply"):
            h3.linear_fp4(h3.quantize_fp4(x, "nvfp4", 2.0 ** 64), w)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M", [65535 * 128 + 1, 65535 * 128 + 777])
def test_more_rows_than_the_swap_form_has_blocks_for(h3, fmt, M):
    """Rows of x past 65535 blocks of 128: any count is taken.  A row's result is the one it
    has among fewer rows (in the tile form, which adds in the same order whatever the size)."""
    N, K = 24, 32
    w = h3.quantize_fp4((torch.randn(N, K, device=DEV) * 0.02).bfloat16(), fmt)
    bias = torch.randn(N, device=DEV).bfloat16()
    x = torch.randn(M, K, device=DEV).bfloat16()
    y = h3.linear_fp4(x, w, bias)
    old = h3.load().h3_fp4_variant(2)
    try:
        for at in (0, M // 2, M - 500):
            assert torch.equal(y[at:at + 500], h3.linear_fp4(x[at:at + 500], w, bias))
    finally:
        h3.load().h3_fp4_variant(old)
    assert h3.load().h3_device_error() == 0


@pytest.mark.gpu
def test_few_rows_by_more_outputs_than_the_fused_form_takes(h3, monkeypatch):
    """A weight of more than 65535 blocks of 128 rows, and so few rows of x that they would be
    quantised inside the product: any count of outputs is taken, through either way of
    calling.  An output is the one of its weight row among fewer (one instruction covers K)."""
    N, K = 65535 * 128 + 1, 16
    w = h3.quantize_fp4((torch.randn(N, K, device=DEV) * 0.02).bfloat16(), "nvfp4")
    codes, scales = h3.unpack_fp4(w)
    tail = h3.pack_fp4(codes[-600:], scales[-600:], "nvfp4", cols=K)
    bias = torch.randn(N, device=DEV).bfloat16()
    for M in (1, 8):
        x = torch.randn(M, K, device=DEV).bfloat16()
        old = h3.load().h3_fp4_variant(2)
        want = h3.linear_fp4(h3.quantize_fp4(x), tail, bias[-600:])
        h3.load().h3_fp4_variant(old)
        for fast in (True, False):
            with monkeypatch.context() as m:
                if not fast:
                    m.setattr(h3._lib, "_host", False)
                y = h3.linear_fp4(x, w, bias)
            assert y.shape == (M, N) and torch.equal(y[:, -600:], want)
    assert h3.linear_fp4(x[:0], w, bias).shape == (0, N)
    assert h3.load().h3_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_the_longest_sums(h3, fmt):
    """K = 2^24 columns, the most there may be, in both forms and quantised inside; one more is
    refused.  (K/64 instructions with 2^-22 each, 9 more for the join; one rounding to BF16.)"""
    K = 1 << 24
    x, w = (torch.randn(n, K, device=DEV).bfloat16() for n in (2, 3))
    xq, wq = h3.quantize_fp4(x, fmt), h3.quantize_fp4(w, fmt)
    xv, wv = (h3.dequantize_fp4(q).double() for q in (xq, wq))
    ref, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    bound = ref.abs() * 2.0 ** -8 + (K / 64 + 9) * 2.0 ** -22 * mag
    for form in (0, 1, 2):
        old = h3.load().h3_fp4_variant(form)
        for y in (h3.linear_fp4(x, wq), h3.linear_fp4(xq, wq)):
            assert bool(((y.double() - ref).abs() <= bound).all())
        h3.load().h3_fp4_variant(old)
    with pytest.raises(RuntimeError, match="unsupported"):
        h3.quantize_fp4(torch.zeros(1, K + 1, dtype=torch.bfloat16, device=DEV), fmt)
    assert h3.load().h3_device_error() == 0
