"""Copies of 4-bit matrices: what the entry points are given of a copy is its own memory."""
import copy
import io
import pickle
import struct

import pytest
import torch

from oracle import fp4_oracle as Q


@pytest.fixture(scope="module")
def h3():
    import h3b200
    return h3b200


def _saved(q):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


WAYS = {"deepcopy": copy.deepcopy, "pickle": lambda q: pickle.loads(pickle.dumps(q)), "save": _saved,
        "copy of copy": lambda q: copy.deepcopy(_saved(q))}


def _packed(h3, fmt, rows=130, cols=33, device="cpu"):
    g = torch.Generator().manual_seed(rows + cols)
    code = torch.randint(0, 16, (rows, cols), generator=g)
    byte = torch.randint(1, 100, (rows, -(-cols // Q.BLOCK[fmt])), generator=g).to(torch.uint8)
    return h3.pack_fp4(Q.bytes_of(code).to(device), byte.to(device), fmt, cols=cols,
                       tensor_scale=0.25 if fmt == "nvfp4" else 1.0)


def _two_tensors(h3, q):
    """The same matrix held as a view of wider rows and a tensor of scales."""
    wide = torch.zeros(q.rows + 2, q.codes.shape[1] + 48, dtype=torch.uint8, device=q.device)
    view = wide[1:-1, 16:-32]
    view.copy_(q.codes)
    return h3.Fp4Tensor(view, q.scales.clone(), q.rows, q.cols, q.format, q.tensor_scale)


def _addresses(q):
    return tuple(struct.unpack_from("P", d)[0] for d in (q.d_codes, q.d_scales))


def _check(h3, q, c):
    assert (c.rows, c.cols, c.format, c.tensor_scale, c.device) == (q.rows, q.cols, q.format, q.tensor_scale, q.device)
    assert torch.equal(c.codes, q.codes) and torch.equal(c.scales, q.scales)
    assert _addresses(c) == (c.codes.data_ptr(), c.scales.data_ptr())
    # the descriptors in full: what the constructor makes of the copy's tensors
    again = h3.Fp4Tensor(c.codes, c.scales, c.rows, c.cols, c.format, c.tensor_scale)
    assert (again.d_codes, again.d_scales) == (c.d_codes, c.d_scales)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("way", WAYS)
def test_a_copy_describes_its_own_memory(h3, fmt, way):
    for q in (_packed(h3, fmt), _two_tensors(h3, _packed(h3, fmt)), h3.fp4_empty(0, 40, fmt, device="cpu")):
        c = WAYS[way](q)
        _check(h3, q, c)
        if q.rows:
            assert not set(_addresses(c)) & set(_addresses(q))
            before = q.codes.clone()
            c.codes.zero_()
            assert torch.equal(q.codes, before)


def test_a_shallow_copy_shares_the_memory(h3):
    for q in (_packed(h3, "nvfp4"), _two_tensors(h3, _packed(h3, "nvfp4"))):
        c = copy.copy(q)
        _check(h3, q, c)
        assert _addresses(c) == _addresses(q)


def test_copies_within_a_container(h3):
    """A matrix that occurs twice is copied once, and weights beside it keep their own."""
    q = _packed(h3, "nvfp4")
    a, b, other = copy.deepcopy([q, q, _packed(h3, "mxfp4")])
    assert a is b and a is not q
    _check(h3, q, a)
    assert other.format == "mxfp4"


def test_bytes_that_do_not_fit_are_refused(h3):
    """What a damaged file rebuilds to."""
    q = _packed(h3, "nvfp4")
    rebuild, args = q.__reduce__()
    for bad in ((args[0][:-1], *args[1:]), (args[0].view(2, -1), *args[1:]), (args[0].int(), *args[1:]),
                (args[0], args[1] + 1, *args[2:]), (*args[:3], "int4", 1.0), (*args[:4], 2.0 ** 65)):
        with pytest.raises(ValueError):
            rebuild(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("way", WAYS)
def test_a_copy_outlives_the_original(h3, fmt, way):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(5, 200, generator=g, device="cuda").bfloat16()
    for make in (lambda: _packed(h3, fmt, 300, 200, "cuda"), lambda: _two_tensors(h3, _packed(h3, fmt, 300, 200, "cuda"))):
        q = make()
        want, values = h3.linear_fp4(x, q), h3.dequantize_fp4(q)
        c = WAYS[way](q)
        q.codes.fill_(0x77)
        q.scales.fill_(1)
        assert torch.equal(h3.linear_fp4(x, c), want) and torch.equal(h3.dequantize_fp4(c), values)
        # quantising into the copy leaves the original's bytes
        h3.quantize_fp4_(c, values)
        assert bool((q.codes == 0x77).all())


def test_what_it_was_made_of_may_be_pointed_elsewhere(h3):
    """A Parameter that moves with its module gets other memory under the same object; the
    matrix keeps the memory that its descriptors name, and the device of it."""
    made = _packed(h3, "nvfp4")
    codes, scales = (torch.nn.Parameter(t.clone(), requires_grad=False) for t in (made.codes, made.scales))
    q = h3.Fp4Tensor(codes, scales, made.rows, made.cols, "nvfp4", made.tensor_scale)
    assert _addresses(q) == (codes.data_ptr(), scales.data_ptr())
    codes[0, 0] = 0x55                                    # contents are shared
    assert int(q.codes[0, 0]) == 0x55
    want = q.codes.clone()
    for t in (codes, scales, q.codes, q.scales):
        t.data = torch.zeros_like(t)
    assert _addresses(q)[0] == q._buffer.data_ptr() and torch.equal(q._buffer, want)
    assert _addresses(q)[1] == q._held_scales.data_ptr()
    c = copy.deepcopy(q)
    assert torch.equal(c.codes, want) and torch.equal(c.scales, made.scales)
    module = torch.nn.Module()
    module.codes, module.scales = (torch.nn.Parameter(t.clone(), requires_grad=False) for t in (made.codes, made.scales))
    q = h3.Fp4Tensor(module.codes, module.scales, made.rows, made.cols, "nvfp4", made.tensor_scale)
    module.to("meta")
    assert module.codes.device.type == "meta" and q.device.type == "cpu" and torch.equal(q.codes, made.codes)
