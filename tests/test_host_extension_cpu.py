"""The host extension is taken only where it fits: another torch's or Python's file is not
looked at, and one that does not load leaves the calls to the ctypes path."""
import importlib
import warnings

import pytest
import torch


@pytest.fixture
def lib(monkeypatch):
    import h3b200
    monkeypatch.setattr(h3b200._lib, "_host", None)
    return h3b200._lib


def test_built_for_this_torch(lib):
    assert lib.HOST_PATH.exists() and lib.host() and lib.host() is lib.host()


def test_another_torch_or_python_is_another_file(lib, monkeypatch):
    build = importlib.import_module("h3b200.build")
    here = build.host_path()
    assert here == lib.HOST_PATH
    monkeypatch.setattr(torch, "__version__", "2.99.0+cu999")
    torchs = build.host_path()
    monkeypatch.undo()
    monkeypatch.setattr(build.sys, "implementation", type("I", (), {"cache_tag": "cpython-399"}))
    assert len({here, torchs, build.host_path()}) == 3 and not torchs.exists()


def test_a_missing_file_is_no_extension(lib, monkeypatch, tmp_path):
    monkeypatch.setattr(lib, "HOST_PATH", tmp_path / "none.so")
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert lib.host() is False


def test_a_file_that_does_not_load_warns_and_leaves_ctypes(lib, monkeypatch, tmp_path):
    import h3b200
    bad = tmp_path / "_h3host.so"
    bad.write_bytes(b"\x7fELF of something else")
    monkeypatch.setattr(lib, "HOST_PATH", bad)
    with pytest.warns(RuntimeWarning, match="ctypes"):
        assert lib.host() is False
    x = torch.zeros(4, 32, dtype=torch.bfloat16)
    q = h3b200.fp4_empty(4, 32, device="cpu")
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        # the calls get as far as the ctypes path's checks
        for f in (lambda: h3b200.quantize_fp4(x), lambda: h3b200.linear_fp4(x, q), lambda: h3b200.dequantize_fp4(q),
                  lambda: h3b200.cross_attention(*[torch.zeros(1, 2, 2, 128, dtype=torch.bfloat16)] * 3)):
            with pytest.raises(ValueError, match="CUDA"):
                f()
