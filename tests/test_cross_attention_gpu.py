"""Cross attention against softmax attention in 64 bits.

What rounds: P to BF16 (half a step, 2^-8 of each weight, relative to the running
maximum), the result to BF16 (2^-8 of it), the scores and sums in fp32 and ex2.approx
(2^-22 relative; scores here stay below 2^6 in the exponent, so 2^-16 of a weight from
rounding them).  With weights w (summing to 1):

    |err| <= 2^-8 |ref| + (2^-8 + 2^-15) sum_j w_j |v_j|

is a bound on every element, without statistics.  A row with one state has weight 1
exactly and returns v.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def h3():
    import h3b200
    h3b200.load()
    assert h3b200._lib.host(), "the host extension is not built"
    return h3b200


@pytest.fixture
def ctypes_only(h3, monkeypatch):
    monkeypatch.setattr(h3._lib, "_host", False)


@pytest.fixture(params=[1, 2], ids=["rows", "tiles"])
def form(h3, request):
    old = h3.load().h3_cross_attention_variant(request.param)
    yield request.param
    h3.load().h3_cross_attention_variant(old)


def _reference(q, k, v, lengths=None, scale=None):
    """(softmax attention, sum of |weight * v|) in fp64."""
    B, Sq, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    ref = torch.zeros(B, Sq, H, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(ref)
    for b in range(B):
        kb, vb = (t[b if t.shape[0] > 1 else 0].double() for t in (k, v))
        n = kb.shape[0] if lengths is None else max(0, min(kb.shape[0], int(lengths[b])))
        if n == 0:
            continue
        for h in range(H):
            g = h // (H // kb.shape[1])
            w = torch.softmax(q[b, :, h].double() @ kb[:n, g].t() * scale, -1)
            ref[b, :, h], mag[b, :, h] = w @ vb[:n, g], w @ vb[:n, g].abs()
    return ref, mag


def _check(h3, out, q, k, v, lengths=None, scale=None):
    ref, mag = _reference(q, k, v, lengths, scale)
    bound = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -15) * mag
    err = (out.double() - ref).abs()
    assert bool((err <= bound).all()), f"error {float((err / bound.clamp_min(1e-30)).max()):.3g} times its bound"
    assert h3.load().h3_device_error() == 0


def _inputs(B, Sq, Sk, H, Hkv, seed=0, kv_batch=None):
    g = torch.Generator(device=DEV).manual_seed(seed + B + 3 * Sq + 7 * Sk + H)
    q = torch.randn(B, Sq, H, 128, generator=g, device=DEV).bfloat16()
    kv = torch.randn(kv_batch or B, Sk, 2, Hkv, 128, generator=g, device=DEV).bfloat16()
    return q, kv[:, :, 0], kv[:, :, 1]


@pytest.mark.parametrize("B,Sq,Sk,H,Hkv", [
    (1, 1, 1, 1, 1), (1, 1, 512, 40, 40), (2, 1, 63, 4, 2), (3, 1, 64, 8, 1), (1, 1, 65, 5, 5), (1, 2, 1000, 16, 2),
    (4, 3, 129, 10, 5), (1, 16, 77, 3, 3), (2, 5, 300, 14, 2), (1, 17, 128, 2, 1), (1, 33, 40, 2, 2),
    (1, 128, 128, 2, 2), (2, 129, 127, 3, 1), (1, 256, 255, 4, 4), (2, 300, 513, 6, 2), (1, 1000, 130, 2, 2),
    (1, 1, 5000, 8, 8), (1, 257, 1, 2, 1)])
def test_shapes(h3, form, B, Sq, Sk, H, Hkv):
    q, k, v = _inputs(B, Sq, Sk, H, Hkv)
    out = h3.cross_attention(q, k, v)
    _check(h3, out, q, k, v)
    assert torch.equal(h3.cross_attention(q, k, v), out)      # the same bits every time


@pytest.mark.parametrize("Sq,H,Hkv,Sk", [(1, 8, 8, 300), (3, 8, 2, 300), (200, 4, 2, 300), (400, 2, 2, 1100),
                                         (140, 1, 1, 129)])
def test_lengths(h3, form, Sq, H, Hkv, Sk):
    """Every length around the tiles' borders, none and all; what lies behind is NaN and
    infinite; an item without states between others, first and last."""
    lengths = [0, Sk, 1, 0, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, Sk - 1, 2, 0]
    lengths = torch.tensor([min(n, Sk) for n in lengths], device=DEV)
    q, k, v = _inputs(len(lengths), Sq, Sk, H, Hkv, seed=1)
    k, v = k.clone(), v.clone()
    clean_k, clean_v = k.clone(), v.clone()
    for b, n in enumerate(lengths.tolist()):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
        if n < Sk:
            v[b, n:][::2] = float("nan")
    out = h3.cross_attention(q, k, v, lengths)
    assert not bool(out.isnan().any())
    _check(h3, out, q, clean_k, clean_v, lengths)
    assert int(out[lengths == 0].count_nonzero()) == 0
    one = torch.nonzero(lengths == 1).flatten()
    group = H // Hkv
    assert torch.equal(out[one], v[one, :1].repeat_interleave(group, 2).expand(-1, Sq, -1, -1))


def test_lengths_are_clamped(h3, form):
    q, k, v = _inputs(3, 40, 100, 2, 2, seed=2)
    out = h3.cross_attention(q, k, v, torch.tensor([-5, 1 << 40, 100], device=DEV))
    _check(h3, out, q, k, v, torch.tensor([0, 100, 100]))


def test_shared_states(h3, form):
    """One sample's keys and values for the whole batch: batch size 1, or a broadcast batch,
    with and without lengths."""
    for Sq, H, Hkv in ((1, 8, 8), (2, 4, 2), (150, 2, 2)):
        q, k, v = _inputs(5, Sq, 200, H, Hkv, seed=3, kv_batch=1)
        out = h3.cross_attention(q, k, v)
        _check(h3, out, q, k, v)
        wide_k, wide_v = (t.expand(5, -1, -1, -1) for t in (k, v))
        assert torch.equal(h3.cross_attention(q, wide_k, wide_v), out)
        lengths = torch.tensor([200, 0, 7, 128, 65], device=DEV)
        k2, v2 = k.clone(), v.clone()
        v2[0, 100] = float("inf")       # a state of the longer samples that the shorter ones do not have
        ragged = h3.cross_attention(q, k2, v2, lengths)
        short = [1, 2, 4]
        _check(h3, ragged[short], q[short], k, v, lengths[short])
        assert bool(torch.isinf(ragged[[0, 3]]).logical_or(ragged[[0, 3]].isnan()).any())


def test_no_states_at_all(h3, form):
    q, k, v = _inputs(2, 130, 4, 4, 2, seed=4)
    out = torch.full_like(q, 7.0)
    h3.cross_attention_(out, q, k[:, :0], v[:, :0])
    assert int(out.count_nonzero()) == 0
    assert h3.cross_attention(q[:, :0], k, v).shape == (2, 0, 4, 128)
    assert h3.cross_attention(q[:0], k[:0], v[:0]).shape == (0, 130, 4, 128)


def test_infinite_scores(h3, form):
    """Keys whose score is -inf add nothing; rows with no other key get zeros; NaN keys make
    their rows NaN and no others."""
    q = torch.ones(1, 4, 1, 128, device=DEV).bfloat16()
    q[0, 3] = -1
    k = torch.randn(1, 150, 1, 128, device=DEV).bfloat16()
    v = torch.randn(1, 150, 1, 128, device=DEV).bfloat16()
    k[0, :70, 0, 5] = float("-inf")
    out = h3.cross_attention(q[:, :3], k, v)
    _check(h3, out, q[:, :3], k[:, 70:], v[:, 70:])
    k[0, :, 0, 5] = float("-inf")
    assert int(h3.cross_attention(q[:, :3], k, v).count_nonzero()) == 0
    assert bool(h3.cross_attention(q, k, v)[0, 3].isnan().all())      # +inf - inf
    k = torch.randn(2, 150, 1, 128, device=DEV).bfloat16()
    k[0, 140, 0, 5] = float("nan")
    out = h3.cross_attention(q.expand(2, -1, -1, -1).contiguous(), k, v.expand(2, -1, -1, -1).contiguous())
    assert bool(out[0].isnan().all()) and not bool(out[1].isnan().any())


def test_growing_scores(h3, form):
    """The running maximum rises all along the keys: results are rescaled again and again."""
    g = torch.Generator(device=DEV).manual_seed(5)
    q = torch.rand(1, 20, 2, 128, generator=g, device=DEV).bfloat16()
    ramp = torch.linspace(0, 4, 1500, device=DEV).view(1, -1, 1, 1)
    k = (torch.rand(1, 1500, 2, 128, generator=g, device=DEV) * ramp).bfloat16()
    v = torch.randn(1, 1500, 2, 128, generator=g, device=DEV).bfloat16()
    _check(h3, h3.cross_attention(q, k, v), q, k, v)
    # fp32 rounding of scores up to 2^7 in the exponent: the bound's 2^-15 becomes 2^-13
    for scale in (1e-3, 0.3):
        ref, mag = _reference(q, k, v, None, scale)
        err = (h3.cross_attention(q, k, v, scale=scale).double() - ref).abs()
        assert bool((err <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -13) * mag).all())


def test_layouts(h3, form):
    """Heads-major storage, slices, an out view with its surroundings untouched."""
    for Sq in (1, 3, 140):
        q, k, v = _inputs(2, Sq, 90, 4, 2, seed=6)
        want = h3.cross_attention(q, k, v)
        qt, kt, vt = (t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v))
        assert torch.equal(h3.cross_attention(qt, kt, vt), want)
        big = torch.full((4, Sq + 2, 6, 136), 3.0, device=DEV).bfloat16()
        view = big[1:3, 1:Sq + 1, 1:5, :128]
        h3.cross_attention_(view, q, k, v)
        assert torch.equal(view, want)
        view.fill_(3.0)
        assert bool((big == 3).all())


def test_query_rows_are_independent(h3):
    """A query's result does not depend on the other queries of its tile."""
    q, k, v = _inputs(1, 700, 300, 2, 2, seed=7)
    full = h3.cross_attention(q, k, v)
    assert torch.equal(h3.cross_attention(q[:, 300:500], k, v), full[:, 300:500])


def test_agrees_with_mha(h3):
    """Equal heads, no lengths: the self attention entry point's arithmetic, bit for bit."""
    h3.load().h3_cross_attention_variant(2)
    try:
        for Sq, Sk, H in ((512, 512, 3), (100, 300, 2), (400, 129, 1)):
            q, k, v = _inputs(1, Sq, Sk, H, H, seed=8)
            assert torch.equal(h3.cross_attention(q, k, v), h3.mha(q, k, v))
    finally:
        h3.load().h3_cross_attention_variant(0)


def test_many_items(h3):
    """More work items than SMs, of unequal lengths: the barriers' phases run on."""
    g = torch.Generator(device=DEV).manual_seed(9)
    lengths = torch.randint(0, 400, (60,), generator=g, device=DEV)
    lengths[::7] = 0
    for Sq in (100, 700):
        q, k, v = _inputs(60, Sq, 400, 4, 2, seed=10)
        _check(h3, h3.cross_attention(q, k, v, lengths), q, k, v, lengths)


def test_refusals(h3):
    q, k, v = _inputs(2, 8, 50, 4, 2, seed=11)
    for bad in (lambda: h3.cross_attention(q, k[:, :, :1].expand(-1, -1, 3, -1), v[:, :, :1].expand(-1, -1, 3, -1)),
                lambda: h3.cross_attention(q.float(), k, v),
                lambda: h3.cross_attention(q[..., :64], k[..., :64], v[..., :64]),
                lambda: h3.cross_attention(q, k, v[:, :40]),
                lambda: h3.cross_attention(q, k, v, torch.tensor([1, 2, 3], device=DEV)),
                lambda: h3.cross_attention(q, k, v, torch.tensor([1, 2], device=DEV, dtype=torch.int32)),
                lambda: h3.cross_attention(q, k, v, torch.tensor([1, 2])),
                lambda: h3.cross_attention(q, k, v, scale=0.0),
                lambda: h3.cross_attention(q, k, v, scale=float("nan")),
                lambda: h3.cross_attention(q, k.expand(2, 50, 2, 128)[:1].expand(3, -1, -1, -1), v),
                lambda: h3.cross_attention(q[:1].expand(2, -1, -1, -1), k, v)):
        with pytest.raises(ValueError):
            bad()


def test_graph_and_streams(h3, form):
    cases = [_inputs(2, 1, 600, 8, 4, seed=12), _inputs(2, 300, 200, 4, 4, seed=13)]
    lengths = torch.tensor([150, 77], device=DEV)
    want = [h3.cross_attention(*c, lengths) for c in cases]
    for c, ref in zip(cases, want):
        q = torch.zeros_like(c[0])
        n = torch.zeros_like(lengths)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = h3.cross_attention(q, c[1], c[2], n)
        graph.replay()
        assert int(out.count_nonzero()) == 0
        q.copy_(c[0])
        n.copy_(lengths)
        graph.replay()
        assert torch.equal(out, ref)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[] for _ in cases]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(h3.cross_attention(*cases[i], lengths))
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        assert all(torch.equal(o, ref) for o in got)


def test_both_ways_of_calling_agree(h3, monkeypatch):
    q, k, v = _inputs(3, 20, 90, 4, 2, seed=14)
    lengths = torch.tensor([90, 0, 17], device=DEV)
    calls = (lambda: h3.cross_attention(q, k, v), lambda: h3.cross_attention(q, k, v, lengths),
             lambda: h3.cross_attention(q[:, ::2], k, v, lengths, scale=0.2),
             lambda: h3.cross_attention(q.transpose(1, 2)[:, :2].transpose(1, 2), k, v),
             lambda: h3.cross_attention(q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1)))
    fast = [f() for f in calls]
    monkeypatch.setattr(h3._lib, "_host", False)
    for f, a in zip(calls, fast):
        assert torch.equal(f(), a)


def test_refusals_without_the_extension(h3, ctypes_only):
    test_refusals(h3)


def test_calls_back_to_back(h3, form):
    """Each call overlaps the end of the kernel before it, which writes its inputs."""
    for Sq in (1, 20, 300):
        sets = [_inputs(3, Sq, 200, 4, 2, seed=20 + i) for i in range(4)]
        lens = [torch.tensor(n, device=DEV) for n in ([200, 3, 0], [1, 200, 64], [0, 0, 129], [77, 128, 200])]
        want = []
        for (q, k, v), n in zip(sets, lens):
            torch.cuda.synchronize()
            want.append(h3.cross_attention(q, k, v, n))
        torch.cuda.synchronize()
        q, n, out = torch.zeros_like(sets[0][0]), torch.zeros_like(lens[0]), torch.zeros_like(want[0])
        k, v = torch.zeros_like(sets[0][1]), torch.zeros_like(sets[0][2])
        got = []
        for i in range(40):
            for dst, src in ((k, sets[i % 4][1]), (v, sets[i % 4][2]), (n, lens[i % 4]), (q, sets[i % 4][0])):
                dst.copy_(src)
            got.append(h3.cross_attention_(out, q, k, v, n).clone())
        assert all(torch.equal(o, want[i % 4]) for i, o in enumerate(got))


def test_offsets_past_32_bits(h3):
    """More than 2^31 elements of keys and values; the last states and heads count."""
    q = torch.randn(1, 1, 128, 128, device=DEV).bfloat16()
    kv = torch.zeros(1, 70000, 2, 128, 128, dtype=torch.bfloat16, device=DEV)
    kv[:, -50:] = torch.randn(1, 50, 2, 128, 128, device=DEV).bfloat16()
    kv[:, :, 0, 126:] = torch.randn(1, 70000, 2, 128, device=DEV).bfloat16()
    k, v = kv[:, :, 0], kv[:, :, 1]
    out = h3.cross_attention(q, k, v)
    _check(h3, out[:, :, 126:], q[:, :, 126:], k[:, :, 126:], v[:, :, 126:])
    q2 = torch.randn(1, 200, 128, 128, device=DEV).bfloat16()
    out = h3.cross_attention(q2, k, v)
    _check(h3, out[:, :, 126:], q2[:, :, 126:], k[:, :, 126:], v[:, :, 126:])
