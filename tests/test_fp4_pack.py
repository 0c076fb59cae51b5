"""pack_fp4 of what checkpoints hold: scale bytes and tensor scales of any value.

With t not a power of two, a read-back is code * (s t), formed with two fp32 roundings
(2^-24 each) and rounded to BF16 (2^-8).  A product multiplies its fp32 sum by
fp32(t_x t_w) and adds the bias in one rounding: 2^-24 of the sum more than the bound of
the products with powers of two, (K/64 + 9) 2^-22 of sum |x w| + |b| and 2^-8 of the result,
which the 9 steps of 2^-22 hold with room (they stand for 8 partial sums and the bias).
"""
import copy
import ctypes
import math

import pytest
import torch

from oracle import fp4_oracle as Q

DEV = "cuda"
SCALES = (1 / 3, 0.0123, 2.0 ** -64 * 1.25, 2.0 ** 63 * 1.999, 4.7683716e-07)


@pytest.fixture(scope="module")
def h3():
    import h3b200
    return h3b200


def test_signed_scales_are_refused(h3):
    """e4m3's sign bit means nothing to the products, and would make read-backs negative."""
    codes = torch.full((3, 24), 0x22, dtype=torch.uint8)
    scales = torch.full((3, 3), 0x38, dtype=torch.uint8)
    for byte in (128, 0xb8, 255):
        bad = scales.clone()
        bad[2, 1] = byte
        with pytest.raises(ValueError, match="sign"):
            h3.pack_fp4(codes, bad, "nvfp4")
        with pytest.raises(ValueError, match="sign"):
            h3.pack_fp4(codes, bad.view(torch.float8_e4m3fn), "nvfp4")
    for byte in (0, 126, 127):                            # zero, 448 and NaN
        scales[2, 1] = byte
        assert torch.equal(h3.unpack_fp4(h3.pack_fp4(codes, scales, "nvfp4"))[1], scales)
    # the exponents of mxfp4 take the whole byte
    every = torch.arange(256, dtype=torch.uint8).view(-1, 1)
    assert torch.equal(h3.unpack_fp4(h3.pack_fp4(torch.zeros(256, 16, dtype=torch.uint8), every, "mxfp4"))[1], every)


def test_scales_that_checkpoints_carry_are_kept(h3):
    """Any fp32 number in [2^-64, 2^64], as fp32."""
    codes, scales = torch.zeros(3, 24, dtype=torch.uint8), torch.zeros(3, 3, dtype=torch.uint8)
    for t in SCALES:
        q = h3.pack_fp4(codes, scales, "nvfp4", tensor_scale=t)
        want = ctypes.c_float(t).value
        assert q.tensor_scale == want and copy.deepcopy(q).tensor_scale == want
        assert h3.pack_fp4(codes, scales, "nvfp4", tensor_scale=torch.tensor(t)).tensor_scale == want
        assert h3.Fp4Tensor(q.codes, q.scales, 3, 48, "nvfp4", t).tensor_scale == want
    for bad in (0.0, -1.0, 2.0 ** -65, 2.0 ** 64 * 1.0001, math.nan, math.inf):
        with pytest.raises(ValueError, match="tensor scale"):
            h3.pack_fp4(codes, scales, "nvfp4", tensor_scale=bad)
    with pytest.raises(ValueError, match="tensor scale"):
        h3.pack_fp4(codes, scales[:, :2], "mxfp4", tensor_scale=2.0)


def test_quantising_still_takes_powers_of_two_only(h3):
    lib, d = h3.load(), lambda t: ctypes.byref(h3._lib.desc(t))
    x, y = torch.zeros(4, 48, dtype=torch.bfloat16), torch.zeros(4, 0, dtype=torch.bfloat16)
    q, w = h3.fp4_empty(4, 48, "nvfp4", device="cpu"), h3.fp4_empty(0, 48, "nvfp4", device="cpu")
    work = torch.zeros(1024, dtype=torch.uint8)
    assert lib.h3_quantize_fp4(d(q.codes), d(q.scales), d(x), 1, 0.3, None) == 5
    for ws in (None, d(work)):
        assert lib.h3_linear_fp4(d(y), d(x), ws, d(w.codes), d(w.scales), None, 1, 0.3, 1.0, None) == 5
        assert lib.h3_linear_fp4(d(y), d(x), ws, d(w.codes), d(w.scales), None, 1, 0.5, 0.3, None) == 0
    # what is held may have any, on both sides
    assert lib.h3_linear_fp4_quantized(d(y), d(q.codes), d(q.scales), d(w.codes), d(w.scales), None, 48, 1, 0.3, 0.7,
                                       None) == 0
    for bad in (0.0, -1.0, 2.0 ** 65, math.nan):
        assert lib.h3_linear_fp4_quantized(d(y), d(q.codes), d(q.scales), d(w.codes), d(w.scales), None, 48, 1, 1.0,
                                           bad, None) == 5
    # mxfp4 has none
    m, e = h3.fp4_empty(0, 48, "mxfp4", device="cpu"), h3.fp4_empty(0, 48, "mxfp4", device="cpu")
    empty = torch.zeros(0, 48, dtype=torch.bfloat16)
    assert lib.h3_dequantize_fp4(d(empty), d(m.codes), d(m.scales), 0, 2.0, None) == 5
    assert lib.h3_dequantize_fp4(d(empty), d(e.codes), d(e.scales), 0, 1.0, None) == 0
    with pytest.raises(ValueError, match="power of two"):
        h3.fp4_empty(4, 48, "nvfp4", 0.3, device="cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("t", SCALES)
def test_read_back_and_products_with_any_scale(h3, t):
    g = torch.Generator(device=DEV).manual_seed(3)
    codes = torch.randint(0, 256, (300, 100), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.randint(1, 127, (300, 13), generator=g, device=DEV, dtype=torch.uint8)
    w = h3.pack_fp4(codes, scales, "nvfp4", tensor_scale=t)
    unit = h3.pack_fp4(codes, scales, "nvfp4")
    exact = Q.values(Q.nibbles(codes.cpu(), 200), scales.cpu().long(), "nvfp4", w.tensor_scale).to(DEV)
    for back in (h3.dequantize_fp4(w), h3.dequantize_fp4_(torch.empty(300, 200, dtype=torch.bfloat16, device=DEV), w)):
        assert bool(((back.double() - exact).abs() <= exact.abs() * (2.0 ** -8 + 2.0 ** -22)).all())
    for M in (1, 8, 30, 200, 1000):
        x = torch.randn(M, 200, generator=g, device=DEV).bfloat16()
        bias = torch.randn(300, generator=g, device=DEV).bfloat16()
        xq = h3.quantize_fp4(x)
        c, b = h3.unpack_fp4(xq)
        xv = Q.values(Q.nibbles(c.cpu(), 200), b.cpu().long(), "nvfp4").to(DEV)
        for add in (bias, None):
            ref, mag = xv @ exact.t(), xv.abs() @ exact.abs().t()
            if add is not None:
                ref, mag = ref + add.double(), mag + add.double().abs()
            bound = ref.abs() * 2.0 ** -8 + (200 / 64 + 9) * 2.0 ** -22 * mag
            for y in (h3.linear_fp4(x, w, add), h3.linear_fp4(xq, w, add)):
                assert bool(((y.double() - ref).abs() <= bound).all())
        # the rows' scale may be any too where they come in 4 bits
        if 2.0 ** -60 < t < 2.0 ** 60:
            rows = h3.pack_fp4(c, b, "nvfp4", tensor_scale=1 / 7)
            ref = xv @ exact.t() * rows.tensor_scale
            bound = ref.abs() * 2.0 ** -8 + (200 / 64 + 9) * 2.0 ** -22 * (xv.abs() @ exact.abs().t()) * rows.tensor_scale
            assert bool(((h3.linear_fp4(rows, w).double() - ref).abs() <= bound).all())
    if math.frexp(w.tensor_scale)[0] != 0.5:              # (the last one is 2^-21 in fp32)
        with pytest.raises(ValueError, match="power of two"):
            h3.quantize_fp4_(w, torch.zeros(300, 200, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="power of two"):
        h3.linear_fp4(x, unit, x_tensor_scale=t)
    assert h3.load().h3_device_error() == 0
