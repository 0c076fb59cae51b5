"""Host side of the microscaled 4-bit matrices: layout round trip, refusals, and the
64-bit oracle against values worked out by hand."""
import pytest
import torch

from oracle import fp4_oracle as Q

FORMATS = ("mxfp4", "nvfp4")


@pytest.fixture(scope="module")
def h3():
    import h3b200
    return h3b200


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 15), (130, 33), (128, 64), (257, 1795)])
def test_pack_round_trip(h3, fmt, rows, cols):
    g = torch.Generator().manual_seed(rows + cols)
    code = torch.randint(0, 16, (rows, cols), generator=g)
    byte = torch.randint(0, 127, (rows, -(-cols // Q.BLOCK[fmt])), generator=g).to(torch.uint8)
    q = h3.pack_fp4(Q.bytes_of(code), byte, fmt, cols=cols)
    assert q.shape == (rows, cols)
    assert tuple(q.codes.shape) == (rows, -(-cols // 32) * 16)
    c, s = h3.unpack_fp4(q)
    assert torch.equal(Q.nibbles(c, cols), code) and torch.equal(s, byte)
    # columns past the last one are zero codes, and so is an odd width's last high nibble
    assert int(q.codes[:, (cols + 1) // 2:].sum()) == 0


def test_pack_places_scales(h3):
    """Row 128a + 32j + i, block 4c + b: chunk [a][c], byte 16i + 4j + b."""
    rows, cols = 200, 16 * 9
    byte = torch.arange(rows * 9).remainder(126).view(rows, 9).to(torch.uint8)
    q = h3.pack_fp4(torch.zeros(rows, cols // 2, dtype=torch.uint8), byte, "nvfp4")
    for r, b in ((0, 0), (1, 0), (31, 3), (32, 4), (127, 8), (128, 0), (199, 7)):
        assert int(q.scales[r // 128, b // 4, 16 * (r % 32) + 4 * (r % 128 // 32) + b % 4]) == int(byte[r, b])


def test_refusals(h3):
    u8 = dict(dtype=torch.uint8)
    with pytest.raises(ValueError, match="format"):
        h3.fp4_empty(4, 32, "int4", device="cpu")
    with pytest.raises(ValueError, match="column"):
        h3.fp4_empty(4, 0, device="cpu")
    for bad in (0.0, -1.0, 3.0, 2.0 ** -65, 2.0 ** 65, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="tensor scale"):
            h3.fp4_empty(4, 32, "nvfp4", bad, device="cpu")
    with pytest.raises(ValueError, match="tensor scale"):
        h3.fp4_empty(4, 32, "mxfp4", 2.0, device="cpu")
    with pytest.raises(ValueError, match="scales a row"):
        h3.pack_fp4(torch.zeros(4, 16, **u8), torch.zeros(4, 2, **u8), "mxfp4")
    with pytest.raises(ValueError, match="same rows"):
        h3.pack_fp4(torch.zeros(4, 16, **u8), torch.zeros(5, 1, **u8), "mxfp4")
    with pytest.raises(ValueError, match="bytes"):
        h3.pack_fp4(torch.zeros(4, 16), torch.zeros(4, 1, **u8), "mxfp4")
    # no CPU fallback
    x = torch.zeros(4, 32, dtype=torch.bfloat16)
    q = h3.fp4_empty(4, 32, device="cpu")
    for f in (lambda: h3.quantize_fp4(x), lambda: h3.dequantize_fp4(q), lambda: h3.linear_fp4(x, q),
              lambda: h3.linear_fp4(q, q)):
        with pytest.raises(ValueError, match="CUDA"):
            f()


def test_entry_points_refuse_bad_arguments(h3):
    """The C entry points check shapes, types, layouts and scales before any launch."""
    import ctypes
    lib = h3.load()
    d = h3._lib.desc
    null = ctypes.c_void_p(0)

    def quantize(q, x, fmt=1, t=1.0):
        return lib.h3_quantize_fp4(*[ctypes.byref(d(a)) for a in (q.codes, q.scales, x)], fmt, t, null)

    x = torch.zeros(4, 48, dtype=torch.bfloat16)
    q = h3.fp4_empty(4, 48, "nvfp4", device="cpu")
    assert quantize(q, x.float()) == 3                                   # x is not BF16
    assert quantize(q, torch.zeros(4, 96, dtype=torch.bfloat16)) == 2    # widths differ
    assert quantize(q, torch.zeros(5, 48, dtype=torch.bfloat16)) == 2    # rows differ
    assert quantize(q, torch.zeros(48, 4, dtype=torch.bfloat16).t()) == 4   # inner stride
    assert quantize(q, x, fmt=0, t=2.0) in (2, 5)                        # mxfp4 has other shapes and no scale
    assert quantize(q, x, fmt=2) == 5
    assert quantize(q, x, t=3.0) == 5
    assert lib.h3_quantize_fp4(None, ctypes.byref(d(q.scales)), ctypes.byref(d(x)), 1, 1.0, null) == 1
    bias = torch.zeros(4, dtype=torch.bfloat16)
    y = torch.zeros(4, 4, dtype=torch.bfloat16)

    def linear(y, x, w, bias, fmt=1, tx=1.0, work=torch.zeros(4 * 32 + 512, dtype=torch.uint8)):
        b = None if bias is None else ctypes.byref(d(bias))
        args = [None if a is None else ctypes.byref(d(a)) for a in (y, x, work, w.codes, w.scales)]
        return lib.h3_linear_fp4(*args, b, fmt, tx, 1.0, null)

    assert linear(y.float(), x, q, None) == 3
    assert linear(torch.zeros(4, 5, dtype=torch.bfloat16), x, q, None) == 2
    assert linear(y, x, h3.fp4_empty(4, 96, "nvfp4", device="cpu"), None) == 2
    assert linear(y, x, q, torch.zeros(5, dtype=torch.bfloat16)) == 2
    assert linear(y, x, q, bias.float()) == 3
    assert linear(y.t(), x, q, bias) == 4
    assert linear(y, x, q, bias, tx=0.3) == 5
    assert linear(y, x, q, bias, work=torch.zeros(4 * 32 + 511, dtype=torch.uint8)) == 2    # a byte short
    assert linear(y, x, q, bias, work=torch.zeros(1000, dtype=torch.bfloat16)) == 3
    assert linear(torch.zeros(9, 4, dtype=torch.bfloat16), torch.zeros(9, 48, dtype=torch.bfloat16), q, bias,
                  work=None) == 1                                        # only up to 8 rows go without
    assert linear(y.t(), x, q, bias, work=None) == 4
    empty = h3.fp4_empty(0, 48, "nvfp4", device="cpu")
    assert linear(torch.zeros(4, 0, dtype=torch.bfloat16), x, empty, None) == 0   # nothing to do


def test_tensor_scale_is_the_smallest_that_fits(h3):
    for amax in (1e-6, 0.0625, 1.0, 2688.0, 2688.1, 1e9):
        t = h3.fp4_tensor_scale(amax)
        assert amax <= 2688.0 * t and amax > 2688.0 * t / 2
    assert h3.fp4_tensor_scale(0.0) == 1.0
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            h3.fp4_tensor_scale(bad)


def test_oracle_known_values():
    x = torch.tensor([[0.0, 0.25, -0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -5.1, 0.26, 2.6, 0.5, 1.0]])
    code, byte = Q.quantize(x, "nvfp4")           # amax 7 / 6 = 1.1667 -> e4m3 1.125
    assert byte.tolist() == [[0x39]]
    code, byte = Q.quantize(torch.nn.functional.pad(x, (0, 16)), "mxfp4")     # floor(log2 7) - 2 = 0
    assert byte.tolist() == [[127]]
    # ties at .25 .75 1.25 1.75 2.5 3.5 5 go to the even codes 0 2 2 4 4 6 6; 7 saturates
    assert code[0, :16].tolist() == [0, 0, 0, 2, 2, 4, 4, 6, 6, 7, 7, 15, 1, 5, 1, 2]
