"""The ends of the cross attention's ranges: scales and scores that fp32 cannot hold, the
result in the queries' place, many samples."""
import ctypes

import pytest
import torch

DEV = "cuda"
H3_ERR_UNSUPPORTED = 5


@pytest.fixture(scope="module")
def h3():
    import h3b200
    return h3b200


@pytest.fixture(params=[1, 2], ids=["rows", "tiles"])
def form(h3, request):
    old = h3.load().h3_cross_attention_variant(request.param)
    yield request.param
    h3.load().h3_cross_attention_variant(old)


def test_scales_past_fp32_are_refused_by_the_entry_point(h3):
    """scale * log2(e) has to be an fp32 number.  (No queries: what is accepted has nothing to do.)"""
    q, k = torch.zeros(1, 0, 2, 128, dtype=torch.bfloat16), torch.zeros(1, 3, 2, 128, dtype=torch.bfloat16)
    ref = [ctypes.byref(h3._lib.desc(t)) for t in (q, q, k, k)]

    def status(scale):
        return h3.load().h3_cross_attention(*ref, None, scale, None)

    assert status(2.36e38) == status(3.0e38) == status(3.4e38) == H3_ERR_UNSUPPORTED
    assert status(2.3e38) == status(1e-40) == 0


@pytest.mark.gpu
def test_the_largest_scale(h3, form):
    """A score of zero times the largest scale is zero: the mean of the states."""
    for Sq in (1, 40, 200):
        q = torch.zeros(1, Sq, 2, 128, device=DEV).bfloat16()
        kv = torch.randn(1, 64, 2, 2, 128, device=DEV).bfloat16()
        out = h3.cross_attention(q, kv[:, :, 0], kv[:, :, 1], scale=2.3e38)
        # every weight is 1 before the division: 64 fp32 additions, a division by 64, one rounding
        mean, size = kv[:, :, 1].double().mean(1), kv[:, :, 1].double().abs().mean(1)
        assert bool(((out.double() - mean[:, None]).abs() <= 2.0 ** -8 * mean.abs() + 64 * 2.0 ** -23 * size).all())
        for scale in (2.36e38, 3e38):
            with pytest.raises(ValueError, match="scale"):
                h3.cross_attention(q, kv[:, :, 0], kv[:, :, 1], scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,Sk", [(1, 9), (4, 300), (30, 1000), (200, 40), (300, 700)])
def test_scores_past_fp32_show_as_nan(h3, form, Sq, Sk):
    """A scaled score above fp32's largest number makes its row NaN (infinity minus infinity),
    wherever it lies among the keys; rows of the same tile whose scores fit are not touched."""
    q = torch.rand(1, Sq, 2, 128, device=DEV).bfloat16()
    kv = torch.rand(1, Sk, 2, 2, 128, device=DEV).bfloat16()
    k, v = kv[:, :, 0], kv[:, :, 1]
    want = h3.cross_attention(q, k, v, scale=1e-3)
    big = q.clone()
    big[:, ::3] = 1e16                          # scores of about 6e17: times 1e25 they overflow
    small = (q.float() * 1e-28).bfloat16()      # and of these the scaled scores are below 1
    mixed = torch.where(torch.arange(Sq, device=DEV).view(1, -1, 1, 1) % 3 == 0, big, small)
    out = h3.cross_attention(mixed, k, v, scale=1e25)
    assert bool(out[:, ::3].isnan().all())
    rest = torch.ones(Sq, dtype=torch.bool, device=DEV)
    rest[::3] = False
    assert torch.equal(out[:, rest], h3.cross_attention(small, k, v, scale=1e25)[:, rest])
    assert not bool(out[:, rest].isnan().any())
    # one key at the end does it too
    k = k.clone()
    k[:, -1] = 1e30
    out = h3.cross_attention(q, k, v, scale=1e9)
    assert bool(out.isnan().all())
    assert not bool(want.isnan().any()) and h3.load().h3_device_error() == 0


@pytest.mark.gpu
def test_into_the_queries(h3, form):
    """The result may take the queries' place."""
    for B, Sq, Sk, H, Hkv in ((2, 1, 300, 8, 2), (3, 40, 500, 4, 4), (1, 5, 5000, 8, 8), (2, 300, 200, 4, 2),
                              (1, 3001, 300, 4, 4)):
        q = torch.randn(B, Sq, H, 128, device=DEV).bfloat16()
        kv = torch.randn(B, Sk, 2, Hkv, 128, device=DEV).bfloat16()
        want = h3.cross_attention(q, kv[:, :, 0], kv[:, :, 1])
        for _ in range(3):
            z = q.clone()
            assert h3.cross_attention_(z, z, kv[:, :, 0], kv[:, :, 1]) is z
            assert torch.equal(z, want)
    assert h3.load().h3_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("B", [511, 512, 513, 2000])
@pytest.mark.parametrize("Sq", [1, 150])
def test_sample_counts_around_what_is_sorted(h3, form, B, Sq):
    """Up to 512 samples are dealt by their length, more as they come.  (P rounds to BF16 and the
    result does, 2^-8 each; 2^-15 for the scores and sums in fp32.)"""
    q = torch.randn(B, Sq, 2, 128, device=DEV).bfloat16()
    kv = torch.randn(B, 200, 2, 1, 128, device=DEV).bfloat16()
    k, v = kv[:, :, 0], kv[:, :, 1]
    lengths = torch.randint(0, 201, (B,), device=DEV)
    out = h3.cross_attention(q, k, v, lengths)
    s = torch.einsum("bqhd,bkd->bhqk", q.double(), k[:, :, 0].double()) * 128 ** -0.5
    s.masked_fill_((torch.arange(200, device=DEV) >= lengths[:, None])[:, None, None], float("-inf"))
    w = torch.softmax(s, -1).nan_to_num(0.0)                       # a sample without states: zeros
    ref, mag = (torch.einsum("bhqk,bkd->bqhd", w, t) for t in (v[:, :, 0].double(), v[:, :, 0].double().abs()))
    assert bool(((out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -15) * mag).all())
    assert h3.load().h3_device_error() == 0
