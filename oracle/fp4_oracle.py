"""The microscaled 4-bit formats and their projection in 64 bits, on the CPU.

Test infrastructure: written from the formats' definitions (blocks of 32 with a
power-of-two scale, blocks of 16 with an e4m3 scale and a power of two for the matrix;
e2m1 values, ties to the even code), independent of the library's kernels.
"""
from __future__ import annotations

import torch

BLOCK = {"mxfp4": 32, "nvfp4": 16}
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _nearest(values: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """Index of the nearest of the ascending ``values``, ties to the even index; exact
    for x and values whose midpoint differences are exact in fp64."""
    hi = torch.bucketize(x, values).clamp(1, len(values) - 1)
    lo = hi - 1
    below, above = x - values[lo], values[hi] - x
    return torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def e4m3_values() -> torch.Tensor:
    """The non-negative finite e4m3 numbers, by their byte (0..126)."""
    b = torch.arange(127)
    e, m = b // 8, (b % 8).double()
    return torch.where(e == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * torch.ldexp(torch.ones(127, dtype=torch.float64), e - 7))


def quantize(x: torch.Tensor, fmt: str, t: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes 0..15 [rows, cols], scale bytes [rows, blocks]) of x (any float dtype, CPU)."""
    rows, cols = x.shape
    size = BLOCK[fmt]
    blocks = -(-cols // size)
    g = torch.zeros(rows, blocks * size, dtype=torch.float64)
    g[:, :cols] = x.double()
    g = g.view(rows, blocks, size)
    bad = ~torch.isfinite(g).all(-1)
    g = torch.where(bad[..., None], torch.zeros((), dtype=torch.float64), g)
    amax = g.abs().amax(-1)
    if fmt == "mxfp4":
        e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, torch.full_like(amax, -127).int()).clamp(-127, 127)
        byte = e + 127
        ratio = torch.ldexp(g, -e[..., None])
        byte[bad] = 255
    else:
        # amax / (6 t) against e4m3's values, both sides times 6: exact in 64 bits
        byte = _nearest(6 * e4m3_values(), amax / t)
        scale = e4m3_values()[byte]
        # x / (scale t) against the codes' values, both sides times the scale
        ratio = None
        byte[bad] = 127
    if ratio is not None:
        code = _nearest(E2M1, ratio.abs())
    else:
        code = torch.zeros(g.shape, dtype=torch.long)
        for i in range(1, 8):        # past the border between values i-1 and i (a tie: to the even one)
            border = (E2M1[i - 1] + E2M1[i]) / 2 * scale[..., None]
            a = g.abs() / t
            code += ((a > border) | ((a == border) & (i % 2 == 0))).long()
        code = torch.where(scale[..., None] > 0, code, 0)
    code = code + 8 * ((g < 0) & (code > 0)).long()
    return code.view(rows, -1)[:, :cols], byte


def values(code: torch.Tensor, byte: torch.Tensor, fmt: str, t: float = 1.0) -> torch.Tensor:
    """fp64 values of codes 0..15 and scale bytes."""
    v = E2M1[(code % 8).long()]
    v = torch.where(code >= 8, -v, v)
    if fmt == "mxfp4":
        s = torch.ldexp(torch.ones(byte.shape, dtype=torch.float64), byte.int() - 127)
        s = torch.where(byte == 255, torch.nan, s)
    else:
        s = torch.cat([e4m3_values(), torch.full((129,), torch.nan, dtype=torch.float64)])[byte.long()] * t
    return v * s.repeat_interleave(BLOCK[fmt], 1)[:, : code.shape[1]]


def nibbles(codes: torch.Tensor, cols: int) -> torch.Tensor:
    """Row-major code bytes [rows, ceil(cols/2)] -> codes [rows, cols]."""
    return torch.stack((codes & 15, codes >> 4), -1).flatten(1)[:, :cols].long()


def bytes_of(code: torch.Tensor) -> torch.Tensor:
    """Codes [rows, cols] -> row-major code bytes [rows, ceil(cols/2)]."""
    c = torch.nn.functional.pad(code, (0, code.shape[1] % 2)).to(torch.uint8)
    return c[:, 0::2] | (c[:, 1::2] << 4)
