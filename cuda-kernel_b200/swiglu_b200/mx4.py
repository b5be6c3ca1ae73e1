"""Four-bit (MXFP4) matrices: rounding, reading back, and products with them.

A matrix ``[..., rows, cols]`` is held as two contiguous uint8 tensors: codes
``[..., rows, 16 * ceil(cols / 32)]`` and scales ``[..., rows, ceil(cols / 32)]``. Each block of
32 values along a row is 16 bytes of e2m1 codes (value 2i in the low half of byte i) times the
power of two ``2 ** (scale - 127)``; scale 255 makes the block NaN. A ragged last block is
filled up with zero codes.

The ``*_out`` calls write buffers the caller owns, launch on the current CUDA stream of the
tensors' device and allocate nothing; the others allocate their outputs. Inference only:
no tensor may require gradients. Every call fails with ``RuntimeError`` before it launches
when an argument does not fit.
"""
from __future__ import annotations

import torch

from . import _lib
from .binding import _check, _stream

BLOCK = 32
_TYPES = {torch.float16: _lib.SWB_F16, torch.bfloat16: _lib.SWB_BF16, torch.float32: _lib.SWB_F32}


def blocks(cols: int) -> int:
    """Blocks (scales) of a row of ``cols`` values."""
    return -(-cols // BLOCK)


# The current stream's handle by device index; the public torch.cuda.current_stream builds a
# Stream object each time, 2 of a small call's 10 microseconds.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _call(device: torch.device, fn, *args) -> None:
    index = device.index
    if index == torch.cuda.current_device():
        status = fn(*args, _raw_stream(index) if _raw_stream else _stream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _stream(device))
    if status:
        _lib.check(status)


def _rows(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, cols, pitch) of a tensor whose rows are contiguous and evenly spaced."""
    cols = t.size(-1)
    if t.is_contiguous():
        return (t.numel() // cols if cols else 0), cols, cols
    if not (t.dim() == 2 and (cols <= 1 or t.stride(1) == 1) and t.stride(0) >= cols):
        raise RuntimeError(f"{name} must be contiguous, or a matrix with contiguous rows")
    return t.size(0), cols, t.stride(0)


def _check_packed(codes: torch.Tensor, scales: torch.Tensor, lead: tuple, cols: int, device: torch.device) -> None:
    """codes and scales of a matrix of shape (*lead, cols)."""
    n = -(-cols // BLOCK)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise RuntimeError("codes and scales must be uint8")
    if not (codes.is_contiguous() and scales.is_contiguous()):
        raise RuntimeError("codes and scales must be contiguous")
    if codes.device != device or scales.device != device:
        raise RuntimeError("buffers must share a device")
    if codes.shape != (*lead, n * 16) or scales.shape != (*lead, n):
        raise RuntimeError("codes and scales do not fit the matrix")


def mx4_empty(*shape: int, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Uninitialised (codes, scales) for a matrix of ``shape``."""
    n = blocks(shape[-1])
    return (torch.empty((*shape[:-1], n * 16), dtype=torch.uint8, device=device or "cuda"),
            torch.empty((*shape[:-1], n), dtype=torch.uint8, device=device or "cuda"))


def _values(x: torch.Tensor) -> tuple[int, int, int]:
    """(rows, cols, pitch) of a tensor to round."""
    _check(x.is_cuda and x.dtype in _TYPES and x.dim() >= 1, "x must be a CUDA FP16, BF16 or FP32 tensor")
    _check(not x.requires_grad, "inference only: disable gradients")
    return _rows(x, "x")


def mx4_quantize_out(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor) -> None:
    """Rounds fp16, bf16 or fp32 ``x`` [..., cols] to ``codes`` and ``scales`` (swb_mx4_quantize).

    A block's scale is ``2 ** (floor(log2(max |x|)) - 2)``, at least 2^-127; values go to the
    nearest code, ties to the even one, larger ones to 6. A block that holds a NaN or an
    infinity becomes NaN as a whole. A matrix may have spaced rows (``x.stride(0) > cols``).
    """
    rows, cols, pitch = _values(x)
    _check_packed(codes, scales, x.shape[:-1], cols, x.device)
    _call(x.device, _lib.lib().swb_mx4_quantize, _TYPES[x.dtype], x.data_ptr(), pitch, codes.data_ptr(),
          scales.data_ptr(), rows, cols)


def mx4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Allocating form of ``mx4_quantize_out``: (codes, scales)."""
    rows, cols, pitch = _values(x)
    codes, scales = mx4_empty(*x.shape, device=x.device)
    _call(x.device, _lib.lib().swb_mx4_quantize, _TYPES[x.dtype], x.data_ptr(), pitch, codes.data_ptr(),
          scales.data_ptr(), rows, cols)
    return codes, scales


def mx4_dequantize_out(codes: torch.Tensor, scales: torch.Tensor, out: torch.Tensor) -> None:
    """The values of ``codes`` and ``scales`` into ``out`` [..., cols] (swb_mx4_dequantize); fp16
    rounds what its range does not hold."""
    _check(out.is_cuda and out.dtype in _TYPES and out.dim() >= 1, "out must be a CUDA FP16, BF16 or FP32 tensor")
    _check(not out.requires_grad, "inference only: disable gradients")
    rows, cols, pitch = _rows(out, "out")
    _check_packed(codes, scales, out.shape[:-1], cols, out.device)
    _call(out.device, _lib.lib().swb_mx4_dequantize, _TYPES[out.dtype], codes.data_ptr(), scales.data_ptr(),
          out.data_ptr(), pitch, rows, cols)


def mx4_dequantize(codes: torch.Tensor, scales: torch.Tensor, cols: int | None = None,
                   dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """Allocating wrapper of ``mx4_dequantize_out``; ``cols`` defaults to whole blocks."""
    _check(scales.dim() >= 1, "scales must hold rows of blocks")
    cols = scales.size(-1) * BLOCK if cols is None else cols
    out = torch.empty((*scales.shape[:-1], cols), dtype=dtype, device=codes.device)
    mx4_dequantize_out(codes, scales, out)
    return out


def _product_arguments(out, like, tokens, rows, bias, residual):
    if out.shape != (tokens, rows) or not out.is_contiguous():
        raise RuntimeError("out must be contiguous [tokens, rows]")
    if out.requires_grad:
        raise RuntimeError("inference only: disable gradients")
    for t, shape in ((bias, (rows,)), (residual, (tokens, rows))):
        if t is not None:
            if t.dtype != like or t.device != out.device or not t.is_contiguous() or t.shape != shape:
                raise RuntimeError("bias must be [rows], residual [tokens, rows], contiguous and of the tokens' type")
            if t.requires_grad:
                raise RuntimeError("inference only: disable gradients")


def mx4_project_out(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, out: torch.Tensor,
                    bias: torch.Tensor | None = None, residual: torch.Tensor | None = None) -> None:
    """out[t] = W x[t] (+ bias) (+ residual[t]) with a four-bit W [rows, cols] (swb_mx4_project).

    x: [tokens, cols] fp16 or bf16, rows contiguous; bias [rows] and residual [tokens, rows] of
    x's type; out: [tokens, rows] of x's type or fp32. ``residual`` may be ``out`` itself.
    """
    _check(x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and x.dim() == 2,
           "x must be a CUDA FP16 or BF16 matrix")
    _check(not x.requires_grad, "inference only: disable gradients")
    _check(codes.dim() == 2 and out.device == x.device and out.dtype in (x.dtype, torch.float32),
           "out must have x's type or FP32, on x's device")
    tokens, rows = x.size(0), codes.size(0)
    cols, pitch = x.size(1), x.stride(0) if tokens > 1 else x.size(1)
    _check((cols <= 1 or x.stride(1) == 1) and pitch >= cols, "x must have contiguous rows")
    _check_packed(codes, scales, (rows,), cols, x.device)
    _product_arguments(out, x.dtype, tokens, rows, bias, residual)
    flags = (_lib.SWB_RESIDUAL if residual is not None else 0) | \
            (_lib.SWB_HALF_OUT if out.dtype == x.dtype else 0)
    _call(x.device, _lib.lib().swb_mx4_project, _TYPES[x.dtype], codes.data_ptr(), scales.data_ptr(), x.data_ptr(),
          pitch, None if bias is None else bias.data_ptr(), None if residual is None else residual.data_ptr(),
          out.data_ptr(), tokens, rows, cols, flags)


def mx4_project(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None,
                residual: torch.Tensor | None = None, dtype: torch.dtype | None = None) -> torch.Tensor:
    """Allocating wrapper of ``mx4_project_out``; ``dtype``: x's type (default) or fp32."""
    _check(x.dim() == 2 and codes.dim() == 2, "x and codes must be matrices")
    out = torch.empty((x.size(0), codes.size(0)), dtype=dtype or x.dtype, device=x.device)
    mx4_project_out(x, codes, scales, out, bias, residual)
    return out


def mx4_matmul_out(x_codes: torch.Tensor, x_scales: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                   out: torch.Tensor, bias: torch.Tensor | None = None,
                   residual: torch.Tensor | None = None) -> None:
    """out[t] = W x[t] (+ bias) (+ residual[t]), both sides in four bits (swb_mx4_matmul).

    x: [tokens, cols] and W: [rows, cols] as codes and scales of the same number of blocks (codes
    beyond a ragged cols are zero, as ``mx4_quantize`` leaves them); out: [tokens, rows] fp16 or
    bf16, the type of bias [rows] and residual [tokens, rows]. ``residual`` may be ``out`` itself.
    """
    _check(out.is_cuda and out.dtype in (torch.float16, torch.bfloat16), "out must be a CUDA FP16 or BF16 matrix")
    _check(x_codes.dim() == 2 and codes.dim() == 2 and x_scales.dim() == 2, "codes must be matrices")
    tokens, rows, cols = x_codes.size(0), codes.size(0), x_scales.size(1) * BLOCK
    _check_packed(x_codes, x_scales, (tokens,), cols, out.device)
    _check_packed(codes, scales, (rows,), cols, out.device)
    _product_arguments(out, out.dtype, tokens, rows, bias, residual)
    _call(out.device, _lib.lib().swb_mx4_matmul, _TYPES[out.dtype], x_codes.data_ptr(), x_scales.data_ptr(),
          codes.data_ptr(), scales.data_ptr(), None if bias is None else bias.data_ptr(),
          None if residual is None else residual.data_ptr(), out.data_ptr(), tokens, rows, cols,
          _lib.SWB_RESIDUAL if residual is not None else 0)


def mx4_matmul(x_codes: torch.Tensor, x_scales: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
               bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
               dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """Allocating wrapper of ``mx4_matmul_out``."""
    _check(x_codes.dim() == 2 and codes.dim() == 2, "codes must be matrices")
    out = torch.empty((x_codes.size(0), codes.size(0)), dtype=dtype, device=x_codes.device)
    mx4_matmul_out(x_codes, x_scales, codes, scales, out, bias, residual)
    return out
