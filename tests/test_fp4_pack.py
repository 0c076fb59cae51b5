"""pack_fp4 of what checkpoints hold: scale bytes."""
import pytest
import torch


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
