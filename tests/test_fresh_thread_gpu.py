"""Calls from a host thread that has done nothing on the GPU before.

Such a thread has no CUDA context bound to it until its first launch, and the descriptors
of the kernels' TMA copies are made before that.  Each operator is the first thing a new
thread does, eagerly and into a graph that the thread captures; the result is the main
thread's, bit for bit.
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
