"""Calls from a host thread that has done nothing on the GPU before.

Such a thread has no CUDA context bound to it until its first launch, and the descriptors
of the kernels' TMA copies are made before that.  Each operator is the first thing a new
thread does, eagerly and into a capture that the main thread began; the result is the main
thread's, bit for bit.  Beside that: threads that share a stream, and streams that join.
"""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def h3():
    import h3b200
    h3b200.load()
    return h3b200


def _operators(h3):
    g = torch.Generator(device=DEV).manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    w = h3.quantize_fp4(rand(300, 256), "nvfp4")
    few, many = rand(4, 256), rand(500, 256)
    fq, mq = h3.quantize_fp4(few), h3.quantize_fp4(many)
    q1, q, kv = rand(2, 1, 4, 128), rand(2, 300, 4, 128), rand(2, 200, 2, 4, 128)
    k, v = kv[:, :, 0], kv[:, :, 1]
    lengths = torch.tensor([200, 60], device=DEV)
    dense = rand(512, 256)
    return {
        "linear_fp4 few rows": lambda: h3.linear_fp4(few, w),
        "linear_fp4 many rows": lambda: h3.linear_fp4(many, w),
        "linear_fp4 quantised few": lambda: h3.linear_fp4(fq, w),
        "linear_fp4 quantised many": lambda: h3.linear_fp4(mq, w),
        "quantize_fp4": lambda: h3.dequantize_fp4(h3.quantize_fp4(many)),
        "dequantize_fp4": lambda: h3.dequantize_fp4(mq),
        "cross_attention one query": lambda: h3.cross_attention(q1, k, v, lengths),
        "cross_attention": lambda: h3.cross_attention(q, k, v, lengths),
        "mha": lambda: h3.mha(q, k, v),
        "linear": lambda: h3.linear(many, dense),
    }


NAMES = ["linear_fp4 few rows", "linear_fp4 many rows", "linear_fp4 quantised few", "linear_fp4 quantised many",
         "quantize_fp4", "dequantize_fp4", "cross_attention one query", "cross_attention", "mha", "linear"]


def _in_a_new_thread(f):
    out = []

    def run():
        try:
            out.append(f())
        except BaseException as e:      # noqa: BLE001
            out.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(out[0], BaseException):
        raise out[0]
    return out[0]


@pytest.mark.parametrize("fast", [True, False], ids=["extension", "ctypes"])
@pytest.mark.parametrize("name", NAMES)
def test_first_call_of_a_thread(h3, monkeypatch, name, fast):
    if not fast:
        monkeypatch.setattr(h3._lib, "_host", False)
    f = _operators(h3)[name]
    want = f()
    torch.cuda.synchronize()
    got = _in_a_new_thread(f)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert h3.load().h3_device_error() == 0


@pytest.mark.parametrize("name", NAMES)
def test_first_call_of_a_thread_into_a_capture(h3, name):
    """The thread takes part in a capture that another thread began on the stream."""
    f = _operators(h3)[name]
    want = f()
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()

    def on_stream():
        with torch.cuda.stream(stream):
            return f()

    with torch.cuda.graph(graph, stream=stream, capture_error_mode="global"):
        got = _in_a_new_thread(on_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert h3.load().h3_device_error() == 0


def test_threads_on_one_stream(h3):
    """Calls of several threads interleave on one stream, a product's quantisation and the
    product itself among them; each keeps its own rows."""
    ws = [h3.quantize_fp4((torch.randn(700, 1100, device=DEV) * 0.1).bfloat16(), f) for f in ("nvfp4", "mxfp4") * 2]
    xs = [torch.randn(m, 1100, device=DEV).bfloat16() for m in (3, 40, 300, 1000)]
    want = [h3.linear_fp4(x, w) for x, w in zip(xs, ws)]
    back = [h3.dequantize_fp4(h3.quantize_fp4(x)) for x in xs]
    torch.cuda.synchronize()
    wrong, errors = [0] * len(xs), []

    def run(i):
        try:
            for _ in range(100):
                y, d = h3.linear_fp4(xs[i], ws[i]), h3.dequantize_fp4(h3.quantize_fp4(xs[i]))
                wrong[i] += not (torch.equal(y, want[i]) and torch.equal(d, back[i]))
        except Exception as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and wrong == [0] * len(xs)
    assert h3.load().h3_device_error() == 0


@pytest.mark.parametrize("M", [3, 100, 700])
def test_weights_written_on_another_branch_of_a_capture(h3, M):
    """The product reads its weights ahead of the quantisation's end; here they are written on a
    stream that joins just before."""
    x = torch.randn(M, 1100, device=DEV).bfloat16()
    w = (torch.randn(640, 1100, device=DEV) * 0.1).bfloat16()
    want = h3.linear_fp4(x, h3.quantize_fp4(w))
    wq, inp, side, graph = h3.fp4_empty(640, 1100), torch.zeros_like(x), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    wq.codes.zero_(), wq.scales.zero_()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            h3.quantize_fp4_(wq, w)
        rows = inp * 1.0
        held = h3.quantize_fp4(rows)
        here.wait_stream(side)
        y, z = h3.linear_fp4(rows, wq), h3.linear_fp4(held, wq)
    inp.copy_(x)
    for _ in range(3):
        wq.codes.zero_()
        graph.replay()
        assert torch.equal(y, want)
        assert torch.equal(z, h3.linear_fp4(h3.quantize_fp4(x), wq))
    # the same without a capture
    for _ in range(20):
        wq.codes.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            h3.quantize_fp4_(wq, w)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(h3.linear_fp4(x, wq), want)
    assert h3.load().h3_device_error() == 0
