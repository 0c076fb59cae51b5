"""Argument checks of the cross attention's entry point: every refusal comes before a launch."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def h3():
    import h3b200
    return h3b200


def _bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_entry_point_refuses_bad_arguments(h3):
    lib = h3.load()

    def call(q, k, v, lengths=None, scale=0.1, out=None):
        ts = (torch.empty_like(q) if out is None else out, q, k, v, lengths)
        args = [None if t is None else ctypes.byref(h3._lib.desc(t)) for t in ts]
        return lib.h3_cross_attention(*args, scale, ctypes.c_void_p(0))

    q, k = _bf16(2, 4, 4, 128), _bf16(2, 9, 2, 128)
    assert call(q.float(), k, k) == 3
    assert call(_bf16(2, 4, 4, 64), _bf16(2, 9, 2, 64), _bf16(2, 9, 2, 64)) == 2      # head size
    assert call(q, k, _bf16(2, 8, 2, 128)) == 2                                       # K and V differ
    assert call(q, _bf16(3, 9, 2, 128), _bf16(3, 9, 2, 128)) == 2                     # batch
    assert call(q, _bf16(2, 9, 3, 128), _bf16(2, 9, 3, 128)) == 2                     # heads do not divide
    assert call(q, k, k, torch.zeros(3, dtype=torch.int64)) == 2
    assert call(q, k, k, torch.zeros(2, dtype=torch.bfloat16)) == 3
    assert call(q, k, k, torch.zeros(4, dtype=torch.int64)[::2]) == 4
    assert call(q, _bf16(2, 9, 2, 132)[..., :128], k) == 4                            # rows not 16-byte aligned
    assert call(q, _bf16(2, 9, 2, 256)[..., ::2], k) == 4                             # inner stride
    assert call(_bf16(1, 4, 4, 128).expand(2, -1, -1, -1), k, k, out=q) == 4          # q may not broadcast
    assert call(q, _bf16(1, 9, 2, 128).expand(2, -1, -1, -1), k) == 4                 # K shared, V not
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(q, k, k, scale=scale) == 5
    assert call(_bf16(0, 4, 4, 128), _bf16(0, 9, 2, 128), _bf16(0, 9, 2, 128)) == 0   # nothing to do
    assert call(_bf16(2, 0, 4, 128), k, k) == 0
    assert lib.h3_cross_attention_variant(3) == -1 and lib.h3_cross_attention_variant(0) == 0


def test_refuses_cpu_tensors(h3):
    q = _bf16(1, 2, 2, 128)
    with pytest.raises(ValueError, match="CUDA"):
        h3.cross_attention(q, q, q)
