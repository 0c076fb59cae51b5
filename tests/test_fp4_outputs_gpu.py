"""What lies beside a projection's output stays as it was.

Outputs are views of wider, longer buffers: every remainder of the width by 8 columns (16
bytes, the unit of the widest stores) at pitches that are and are not a multiple of it, at
aligned and unaligned starts, and single rows.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def h3():
    import h3b200
    h3b200.load()
    return h3b200


@pytest.fixture(params=[0, 1, 2], ids=["chosen", "swap", "tiles"])
def form(h3, request):
    old = h3.load().h3_fp4_variant(request.param)
    yield request.param
    h3.load().h3_fp4_variant(old)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M", [1, 2, 8, 9, 40, 171, 300])
def test_columns_and_rows_around_the_output(h3, form, fmt, M):
    x = torch.randn(M, 100, device=DEV).bfloat16()
    xq = h3.quantize_fp4(x, fmt)
    for N in (1, 7, 63, 65, 248, 249, 250, 251, 252, 253, 254, 255, 256, 257, 281, 321, 333):
        w = h3.quantize_fp4((torch.randn(N, 100, device=DEV) * 0.1).bfloat16(), fmt)
        bias = torch.randn(N, device=DEV).bfloat16()
        want = h3.linear_fp4(x, w, bias)              # its own tensor
        want_q = h3.linear_fp4(xq, w, bias)
        for pitch in {-(-N // 8) * 8, -(-N // 8) * 8 + 8, -(-N // 8) * 8 + 4, N, N + 1, N + 3}:
            for start in (pitch, pitch + 4, pitch + 3):
                buf = torch.full((start + (M + 1) * pitch + 64,), 5.0, device=DEV).bfloat16()
                out = buf[start:start + M * pitch].view(M, pitch)[:, :N]
                for rows, ref in ((x, want), (xq, want_q)):
                    h3.linear_fp4_(out, rows, w, bias)
                    assert torch.equal(out, ref), (N, pitch, start)
                    out.fill_(5.0)
                    assert bool((buf == 5).all()), (N, pitch, start)
    assert h3.load().h3_device_error() == 0


def test_projections_side_by_side(h3, form):
    """q, k and v of odd widths into slices of one buffer, in any order."""
    x = torch.randn(200, 320, device=DEV).bfloat16()
    widths = (251, 125, 129)
    ws = [h3.quantize_fp4((torch.randn(n, 320, device=DEV) * 0.1).bfloat16()) for n in widths]
    want = torch.cat([h3.linear_fp4(x, w) for w in ws], 1)
    for order in ((0, 1, 2), (2, 1, 0), (1, 2, 0)):
        # slices that begin on 16 bytes, and ones that follow each other closely
        for starts in ((0, 256, 384), (0, 251, 376)):
            buf = torch.full((200, 520), 5.0, device=DEV).bfloat16()
            for i in order:
                h3.linear_fp4_(buf[:, starts[i]:starts[i] + widths[i]], x, ws[i])
            assert torch.equal(torch.cat([buf[:, s:s + n] for s, n in zip(starts, widths)], 1), want)
            for s, n in zip(starts, widths):
                buf[:, s:s + n] = 5.0
            assert bool((buf == 5).all())
