"""Microscaled 4-bit matrices and projections on the sm_100a C-ABI library.

A block of consecutive columns of a row shares one scale; a value is an e2m1 code
(0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) times that scale:

* ``"mxfp4"``: blocks of 32, the scale a power of two;
* ``"nvfp4"``: blocks of 16, the scale an e4m3 number times ``tensor_scale``, one number
  for the whole matrix: a power of two for what is quantised here (``fp4_tensor_scale``
  gives one that fits), any fp32 number for what a checkpoint brings.

Weights are held as ``Fp4Tensor`` (made once, by ``quantize_fp4`` from BF16 or by
``pack_fp4`` from a checkpoint's codes and scales); ``linear_fp4`` quantises its
activations on the way in.  Inference only: nothing here takes part in autograd.
No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import math

import torch

from ._lib import CALLS, call, host, packed, packed_bytes, require_cuda, stream_of

__all__ = ["Fp4Tensor", "FP4_BLOCK", "fp4_empty", "fp4_tensor_scale", "quantize_fp4", "quantize_fp4_", "dequantize_fp4",
           "dequantize_fp4_", "pack_fp4", "unpack_fp4", "linear_fp4", "linear_fp4_"]

FP4_BLOCK = {"mxfp4": 32, "nvfp4": 16}
_FORMAT = {"mxfp4": 0, "nvfp4": 1}
FUSED_ROWS = 8       # up to so many rows the product quantises x itself, without a workspace,
FUSED_OUTS = 65535 * 128    # for up to so many rows of the weight (its grid's limit)


def _check_format(fmt: str) -> int:
    try:
        return _FORMAT[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"unknown 4-bit format {fmt!r}: 'mxfp4' or 'nvfp4'") from None


def _check_held_scale(fmt: str, scale: float) -> float:
    """The scale of a matrix, as fp32."""
    scale = float(scale)
    if scale == 1.0:
        return scale
    scale = ctypes.c_float(scale).value
    if fmt == "mxfp4":
        raise ValueError("mxfp4 has no tensor scale")
    if not 2.0 ** -64 <= scale <= 2.0 ** 64:
        raise ValueError(f"the tensor scale must lie in [2^-64, 2^64], got {scale}")
    return scale


def _check_tensor_scale(fmt: str, scale: float) -> float:
    """The scale of what is quantised here."""
    scale = float(scale)
    if scale == 1.0:
        return scale
    held = _check_held_scale(fmt, scale)
    if held != scale or math.frexp(held)[0] != 0.5:
        raise ValueError(f"the tensor scale must be a power of two to quantise with it, got {scale}")
    return held


class Fp4Tensor:
    """A matrix of ``rows`` x ``cols`` 4-bit values: ``codes`` uint8
    [rows, ceil(cols/32)*16] (two codes a byte) and ``scales`` uint8
    [ceil(rows/128), ceil(blocks/4), 512], as the products read them.  Immutable but for
    its contents: the descriptors the entry points take are made once.  They hold addresses,
    so a copy (``copy``, ``pickle``, ``torch.save``) takes the tensors and makes its own
    (``torch.load`` builds this class with ``weights_only=False``)."""

    __slots__ = ("rows", "cols", "format", "tensor_scale", "d_codes", "d_scales", "_buffer", "_held_scales", "_codes",
                 "_scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, cols: int, format: str,
                 tensor_scale: float = 1.0):
        _check_format(format)
        self.rows, self.cols, self.format = rows, cols, format
        self.tensor_scale = _check_held_scale(format, tensor_scale)
        if codes.device != scales.device:
            raise ValueError("codes and scales must be on the same device")
        # tensors of its own over the same memory: what is given may be pointed elsewhere (a
        # Parameter that moves with its module), and these keep the memory described here alive
        self._buffer, self._held_scales = codes.detach(), scales.detach()
        self._codes = self._scales = None
        self.d_codes, self.d_scales = packed(self._buffer), packed(self._held_scales)

    @classmethod
    def _uninitialised(cls, like: torch.Tensor, rows: int, cols: int, format: str, tensor_scale: float) -> Fp4Tensor:
        """On ``like``'s device, codes and scales in one allocation."""
        pitch, groups, chunks = _layout(rows, cols, format)
        return cls._within(like.new_empty(rows * pitch + groups * chunks * 512, dtype=torch.uint8), rows, cols, format,
                           tensor_scale)

    @classmethod
    def _within(cls, buffer: torch.Tensor, rows: int, cols: int, format: str, tensor_scale: float) -> Fp4Tensor:
        """Of a buffer that holds the codes, then the scales."""
        _check_format(format)
        scale = _check_held_scale(format, tensor_scale)
        pitch, groups, chunks = _layout(rows, cols, format)
        if buffer.dtype != torch.uint8 or buffer.shape != (rows * pitch + groups * chunks * 512,) or buffer.stride(0) != 1:
            raise ValueError(f"not the bytes of a {format} matrix [{rows}, {cols}]")
        at = buffer.data_ptr()
        return cls._of(buffer, packed_bytes(at, (rows, pitch), (pitch, 1)),
                       packed_bytes(at + rows * pitch, (groups, chunks, 512), (chunks * 512, 512, 1)), rows, cols,
                       format, scale)

    @classmethod
    def _of(cls, buffer, d_codes, d_scales, rows, cols, format, tensor_scale) -> Fp4Tensor:
        """Of a buffer laid out as ``_within`` takes it, with its descriptors."""
        self = cls.__new__(cls)
        self._buffer, self.d_codes, self.d_scales, self.rows, self.cols = buffer, d_codes, d_scales, rows, cols
        self.format, self.tensor_scale = format, tensor_scale
        self._held_scales = self._codes = self._scales = None
        return self

    def __reduce__(self):
        rest = (self.rows, self.cols, self.format, self.tensor_scale)
        if self._held_scales is not None:    # given as two tensors
            return Fp4Tensor, (self._buffer, self._held_scales, *rest)
        return Fp4Tensor._within, (self._buffer, *rest)

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            pitch, _, _ = _layout(self.rows, self.cols, self.format)
            self._codes = (self._buffer[: self.rows * pitch].view(self.rows, pitch) if self._held_scales is None
                           else self._buffer.detach())
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            pitch, groups, chunks = _layout(self.rows, self.cols, self.format)
            self._scales = (self._buffer[self.rows * pitch:].view(groups, chunks, 512) if self._held_scales is None
                            else self._held_scales.detach())
        return self._scales

    @property
    def shape(self) -> tuple[int, int]:
        return self.rows, self.cols

    @property
    def device(self) -> torch.device:
        return self._buffer.device

    def __repr__(self) -> str:
        return f"Fp4Tensor({self.rows} x {self.cols}, {self.format}, tensor_scale={self.tensor_scale}, {self.device})"


def _layout(rows: int, cols: int, fmt: str) -> tuple[int, int, int]:
    """Bytes of a row of codes, 128-row groups and chunks per group of the scales."""
    per_chunk = 128 if fmt == "mxfp4" else 64
    return (cols + 31) // 32 * 16, (rows + 127) // 128, (cols + per_chunk - 1) // per_chunk


def fp4_empty(rows: int, cols: int, format: str = "nvfp4", tensor_scale: float = 1.0, device="cuda") -> Fp4Tensor:
    """An uninitialised 4-bit matrix (the target of ``quantize_fp4_``)."""
    _check_format(format)
    if rows < 0 or cols < 1:
        raise ValueError(f"a 4-bit matrix has at least one column, got [{rows}, {cols}]")
    scale = _check_tensor_scale(format, tensor_scale)
    return Fp4Tensor._uninitialised(torch.empty(0, dtype=torch.uint8, device=device), rows, cols, format, scale)


def fp4_tensor_scale(amax: float) -> float:
    """The smallest power of two t with amax <= 6 * 448 * t: the finest nvfp4 tensor scale
    at which no block of a matrix with entries up to ``amax`` saturates."""
    amax = float(amax)
    if not math.isfinite(amax) or amax < 0:
        raise ValueError(f"amax must be finite and not negative, got {amax}")
    if amax == 0:
        return 1.0
    m, e = math.frexp(amax / 2688.0)        # m in [0.5, 1)
    return 2.0 ** max(-64, min(64, e - 1 if m == 0.5 else e))


def _check_scales_together(x_scale: float, w_scale: float) -> None:
    if math.isinf(ctypes.c_float(x_scale * w_scale).value):
        raise ValueError(f"the tensor scales {x_scale} and {w_scale} multiply to more than fp32 holds")


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


def _rows_to_write(out: torch.Tensor) -> torch.Tensor:
    try:
        return out if out.dim() == 2 else out.view(-1, out.shape[-1])
    except RuntimeError:
        raise ValueError("out's leading dimensions must collapse to rows without a copy") from None


# ---------------------------------------------------------------------------
# quantisation
# ---------------------------------------------------------------------------
def quantize_fp4_(out: Fp4Tensor, x: torch.Tensor) -> Fp4Tensor:
    """Quantise x [..., cols] BF16 into ``out`` (its format and tensor scale, a power of two)."""
    require_cuda(out._buffer, x)
    _check_tensor_scale(out.format, out.tensor_scale)
    x2 = _rows_of(x)
    if x2.shape != (out.rows, out.cols):
        raise ValueError(f"x has shape {tuple(x2.shape)}, the 4-bit matrix {out.shape}")
    call("h3_quantize_fp4", out.d_codes, out.d_scales, packed(x2), _FORMAT[out.format], out.tensor_scale,
         stream_of(x))
    return out


def quantize_fp4(x: torch.Tensor, format: str = "nvfp4", tensor_scale: float = 1.0) -> Fp4Tensor:
    """x [..., cols] BF16 as a 4-bit matrix of its rows."""
    code = _check_format(format)
    scale = _check_tensor_scale(format, tensor_scale)
    fast = host() and host().quantize_fp4(x, code, scale)
    if fast:
        CALLS["n"] += 1
        return Fp4Tensor._of(*fast, format, scale)
    require_cuda(x)
    x2 = _rows_of(x)
    rows, cols = x2.shape
    if cols < 1:
        raise ValueError("a 4-bit matrix has at least one column")
    out = Fp4Tensor._uninitialised(x, rows, cols, format, scale)
    call("h3_quantize_fp4", out.d_codes, out.d_scales, packed(x2), code, scale, stream_of(x))
    return out


def dequantize_fp4_(out: torch.Tensor, q: Fp4Tensor) -> torch.Tensor:
    require_cuda(out, q._buffer)
    if out.shape != q.shape:
        raise ValueError(f"out has shape {tuple(out.shape)}, the 4-bit matrix {q.shape}")
    call("h3_dequantize_fp4", packed(out), q.d_codes, q.d_scales, _FORMAT[q.format], q.tensor_scale,
         stream_of(out))
    return out


def dequantize_fp4(q: Fp4Tensor) -> torch.Tensor:
    """The values a 4-bit matrix stands for, [rows, cols] BF16: exact, but rounded where the
    tensor scale is no power of two."""
    if host():
        out = host().dequantize_fp4(q._buffer, q.d_codes, q.d_scales, q.rows, q.cols, _FORMAT[q.format],
                                    q.tensor_scale)
        if out is not None:
            CALLS["n"] += 1
            return out
    return dequantize_fp4_(q._buffer.new_empty((q.rows, q.cols), dtype=torch.bfloat16), q)


def pack_fp4(codes: torch.Tensor, scales: torch.Tensor, format: str, cols: int | None = None,
             tensor_scale: float = 1.0) -> Fp4Tensor:
    """A 4-bit matrix from row-major parts, as checkpoints store them: ``codes`` uint8
    [rows, ceil(cols/2)] (column 2i in the low nibble of byte i) and ``scales`` uint8 (or
    e4m3, without signs) [rows, ceil(cols/block)].  A set-up step: lays the scales out once, in
    torch, and looks at them on the host."""
    _check_format(format)
    if scales.dtype != torch.uint8 and scales.element_size() == 1:
        scales = scales.view(torch.uint8)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError("codes and scales must be bytes")
    if codes.dim() != 2 or scales.dim() != 2 or codes.shape[0] != scales.shape[0]:
        raise ValueError("codes and scales are matrices of the same rows")
    if codes.device != scales.device:
        raise ValueError("codes and scales must be on the same device")
    rows = codes.shape[0]
    cols = 2 * codes.shape[1] if cols is None else int(cols)
    block = FP4_BLOCK[format]
    blocks = (cols + block - 1) // block
    if cols < 1 or codes.shape[1] != (cols + 1) // 2 or scales.shape[1] != blocks:
        raise ValueError(f"{cols} columns need {(cols + 1) // 2} code bytes and {blocks} scales a row, got "
                         f"{codes.shape[1]} and {scales.shape[1]}")
    if format == "nvfp4" and bool((scales >= 128).any()):
        raise ValueError("nvfp4 scales have no sign: their bytes are below 128")
    out = Fp4Tensor._uninitialised(codes, rows, cols, format, tensor_scale)
    out.codes.zero_()
    out.codes[:, : codes.shape[1]] = codes
    if cols % 2:
        out.codes[:, cols // 2] &= 0x0F
    chunks_m, chunks_k = out.scales.shape[:2]
    padded = torch.zeros(chunks_m * 128, chunks_k * 4, dtype=torch.uint8, device=codes.device)
    padded[:rows, :blocks] = scales
    # row 128 a + 32 j + i, block 4 c + b -> chunk [a][c], byte 16 i + 4 j + b
    out.scales.copy_(padded.view(chunks_m, 4, 32, chunks_k, 4).permute(0, 3, 2, 1, 4).reshape(out.scales.shape))
    return out


def unpack_fp4(q: Fp4Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``pack_fp4``'s parts back: codes [rows, ceil(cols/2)] and scales [rows, ceil(cols/block)]."""
    blocks = (q.cols + FP4_BLOCK[q.format] - 1) // FP4_BLOCK[q.format]
    a, c = q.scales.shape[:2]
    scales = q.scales.view(a, c, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(a * 128, c * 4)
    return q.codes[:, : (q.cols + 1) // 2].clone(), scales[: q.rows, :blocks].contiguous()


# ---------------------------------------------------------------------------
# projection
# ---------------------------------------------------------------------------
def _fused_rows(weight: Fp4Tensor) -> int:
    return FUSED_ROWS if weight.rows <= FUSED_OUTS else 0


def linear_fp4_(out: torch.Tensor, x: torch.Tensor | Fp4Tensor, weight: Fp4Tensor, bias: torch.Tensor | None = None,
                x_tensor_scale: float = 1.0) -> torch.Tensor:
    """out [..., N] BF16 = x W^T (+ bias), both in ``weight``'s 4-bit format, fp32
    accumulation, one rounding.  ``x`` BF16 [..., K] is quantised on the way in (with
    ``x_tensor_scale`` for nvfp4), or given as an ``Fp4Tensor`` (with its own scale; out is
    then [M, N]) when several projections share it.  The product of the two tensor scales has to be below 2^128."""
    o2 = _rows_to_write(out)
    if isinstance(x, Fp4Tensor):
        require_cuda(out, x._buffer, weight._buffer, bias)
        if x.format != weight.format:
            raise ValueError(f"x is {x.format}, the weight {weight.format}")
        if x.cols != weight.cols:
            raise ValueError(f"x has {x.cols} columns, the weight {weight.cols}")
        _check_scales_together(x.tensor_scale, weight.tensor_scale)
        call("h3_linear_fp4_quantized", packed(o2), x.d_codes, x.d_scales, weight.d_codes, weight.d_scales,
             packed(bias), x.cols, _FORMAT[weight.format], x.tensor_scale, weight.tensor_scale, stream_of(out))
        return out
    x2 = _rows_of(x)
    rows, cols = x2.shape
    if cols != weight.cols:
        raise ValueError(f"x has {cols} columns, the weight {weight.cols}")
    require_cuda(out, x, weight._buffer, bias)
    scale = _check_tensor_scale(weight.format, x_tensor_scale)
    _check_scales_together(scale, weight.tensor_scale)
    work = None
    if rows > _fused_rows(weight):
        pitch, groups, chunks = _layout(rows, cols, weight.format)
        work = x.new_empty(rows * pitch + groups * chunks * 512, dtype=torch.uint8)   # x in 4 bits
    call("h3_linear_fp4", packed(o2), packed(x2), packed(work), weight.d_codes, weight.d_scales, packed(bias),
         _FORMAT[weight.format], scale, weight.tensor_scale, stream_of(x))
    return out


def linear_fp4(x: torch.Tensor | Fp4Tensor, weight: Fp4Tensor, bias: torch.Tensor | None = None,
               x_tensor_scale: float = 1.0) -> torch.Tensor:
    """``linear_fp4_`` into a new tensor."""
    if host() and not isinstance(x, Fp4Tensor):
        out = host().linear_fp4(x, weight._buffer, weight.d_codes, weight.d_scales, weight.rows, weight.cols, bias,
                                _FORMAT[weight.format], _check_tensor_scale(weight.format, x_tensor_scale),
                                weight.tensor_scale, _fused_rows(weight))
        if out is not None:
            CALLS["n"] += 1
            return out
    lead = (x.rows,) if isinstance(x, Fp4Tensor) else x.shape[:-1]
    out = weight._buffer.new_empty((*lead, weight.rows), dtype=torch.bfloat16)
    return linear_fp4_(out, x, weight, bias, x_tensor_scale)
