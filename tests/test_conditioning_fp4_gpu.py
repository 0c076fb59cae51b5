"""The conditioning sub-layer of a block run in 4 bits, from the public entry points:

    n  = RMSNorm + AdaLN (x)                      h3_rms_modulate
    q  = n Wq^T, [k | v] = states Wkv^T           quantize_fp4 / linear_fp4
    q, k = per-head RMSNorm                       h3_rms_norm
    a  = cross attention over each sample's states   cross_attention
    y  = x + gate * (a Wo^T + b)                  linear_fp4, h3_gated_residual

Every 4-bit product and the attention are checked against 64-bit arithmetic on the inputs
they were given (the stages' own error bounds: half a BF16 step of the result and of P,
and the fp32 accumulation), so no tolerance has to cover how a flipped code travels on.
The whole chain, captured and replayed with other inputs, gives the eager bits.
"""
import pytest
import torch

from oracle import fp4_oracle as Q

pytestmark = pytest.mark.gpu
DEV = "cuda"
HEADS, KV_HEADS, WIDTH, STATE_WIDTH = 4, 2, 512, 320


@pytest.fixture(scope="module")
def h3():
    import h3b200
    h3b200.load()
    return h3b200


def _randn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).bfloat16()


def _weights(h3, fmt, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = 2.0 ** -8 if fmt == "nvfp4" else 1.0
    make = lambda n, k: h3.quantize_fp4(_randn(g, n, k, std=0.03), fmt, t)  # noqa: E731
    return dict(q=make(HEADS * 128, WIDTH), kv=make(2 * KV_HEADS * 128, STATE_WIDTH), o=make(WIDTH, HEADS * 128),
                bias=_randn(g, WIDTH, std=0.1), norm=1 + _randn(g, WIDTH, std=0.1), head=1 + _randn(g, 128, std=0.1),
                scale=_randn(g, WIDTH, std=0.1), shift=_randn(g, WIDTH, std=0.1), gate=_randn(g, WIDTH, std=0.5))


def _layer(h3, w, x, states, lengths):
    """x [B, S, WIDTH], states [B, L, STATE_WIDTH] -> (y, the stages' inputs and results)."""
    B, S, _ = x.shape
    n = h3.h3_rms_modulate(x, w["norm"], w["scale"], w["shift"], 1e-6)
    q = h3.linear_fp4(n, w["q"])
    kv = h3.linear_fp4(states, w["kv"])
    heads = h3.h3_rms_norm(q.view(-1, 128), w["head"], 1e-6).view(B, S, HEADS, 128)
    kv4 = kv.view(B, -1, 2, KV_HEADS, 128)
    keys = h3.h3_rms_norm(kv4[:, :, 0].reshape(-1, 128), w["head"], 1e-6).view(B, -1, KV_HEADS, 128)
    a = h3.cross_attention(heads, keys, kv4[:, :, 1], lengths)
    o = h3.linear_fp4(a.view(B, S, -1), w["o"], w["bias"])
    y = h3.h3_gated_residual(x.view(-1, WIDTH), w["gate"], o.view(-1, WIDTH)).view_as(x)
    return y, dict(n=n, q=q, kv=kv, heads=heads, keys=keys, values=kv4[:, :, 1], a=a, o=o)


def _values(h3, q):
    c, s = h3.unpack_fp4(q)
    return Q.values(Q.nibbles(c.cpu(), q.cols), s.cpu().long(), q.format, q.tensor_scale).to(DEV)


def _check_product(h3, x, w, y, bias=None):
    x2 = x.reshape(-1, x.shape[-1])
    code, byte = Q.quantize(x2.cpu(), w.format)
    xv, wv = Q.values(code, byte, w.format).to(DEV), _values(h3, w)
    ref, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    if bias is not None:
        ref, mag = ref + bias.double(), mag + bias.double().abs()
    bound = ref.abs() * 2.0 ** -8 + (xv.shape[1] / 64 + 9) * 2.0 ** -22 * mag
    assert bool(((y.reshape(ref.shape).double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("B,S,L", [(1, 1, 77), (3, 1, 200), (2, 5, 33), (3, 150, 300), (1, 700, 512)])
def test_layer(h3, fmt, B, S, L):
    g = torch.Generator(device=DEV).manual_seed(B + S + L)
    w = _weights(h3, fmt, 1)
    x, states = _randn(g, B, S, WIDTH), _randn(g, B, L, STATE_WIDTH)
    lengths = torch.tensor([L, 0, L // 2][:B], device=DEV)
    states[-1, int(lengths[-1]):] = float("nan")          # padding of the encoder's batch
    y, s = _layer(h3, w, x, states, lengths)
    assert not bool(y.isnan().any())
    _check_product(h3, s["n"], w["q"], s["q"])
    good = torch.arange(L, device=DEV) < lengths[:, None]
    _check_product(h3, states[good], w["kv"], s["kv"][good])
    _check_product(h3, s["a"].view(B, S, -1), w["o"], s["o"], w["bias"])
    for b in range(B):
        m = int(lengths[b])
        if m == 0:
            assert int(s["a"][b].count_nonzero()) == 0
            continue
        for h in range(HEADS):
            k, v = (s[t][b, :m, h // (HEADS // KV_HEADS)].double() for t in ("keys", "values"))
            p = torch.softmax(s["heads"][b, :, h].double() @ k.t() * 128 ** -0.5, -1)
            ref, mag = p @ v, p @ v.abs()
            assert bool(((s["a"][b, :, h].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -15) * mag).all())
    assert h3.load().h3_device_error() == 0


def test_layer_captured(h3):
    g = torch.Generator(device=DEV).manual_seed(9)
    w = _weights(h3, "nvfp4", 2)
    sets = [(_randn(g, 2, S, WIDTH), _randn(g, 2, 90, STATE_WIDTH), torch.tensor(n, device=DEV))
            for S, n in ((4, [90, 13]), (4, [0, 64]))]
    want = [_layer(h3, w, *s)[0] for s in sets]
    x, states, lengths = (torch.zeros_like(t) for t in sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _layer(h3, w, x, states, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _layer(h3, w, x, states, lengths)[0]
    for i in (0, 1, 0, 0, 1):
        for dst, src in zip((x, states, lengths), sets[i]):
            dst.copy_(src)
        graph.replay()
        assert torch.equal(y, want[i])
