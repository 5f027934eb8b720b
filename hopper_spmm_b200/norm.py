"""The RMS norm in front of products with weights in few bits, and its result in 8 bits (b200spmm_rms_norm of the C ABI).

    y = rms_norm(x, w)                                     # 16 or 32 bits, as x
    y, h = rms_norm(x, w, residual=h)                      # h = x + h, in a new tensor
    y, h = rms_norm(x, w, residual=h, sum_out=h, dtype=torch.float8_e4m3fn, group=128)   # h in place, y an Fp8Matrix
    Int4Matrix(...).linear(y)

The reference has no such operator (its element types are fp16 and tf32, src/common.h:14-43).
"""
from __future__ import annotations

from . import _capi as capi
from .fp4 import _lib, _on

GROUPS = (32, 64, 128)  # columns that may share a scale, beside a whole row


class Fp8Matrix:
    """A rows x cols matrix in e4m3: ``values`` float8_e4m3fn [rows, cols] times ``scales`` float32, [rows, 1] for a scale of each row (``group``
    None) or [rows, groups of a row] for one of every ``group`` (32, 64 or 128) neighbours begun.  CUDA tensors; rows of ``values`` may lie apart,
    ``scales`` is contiguous."""

    __slots__ = ("values", "scales", "group")

    def __init__(self, values, scales, group: int | None = None):
        import torch
        if group is not None and group not in GROUPS:
            raise ValueError("group must be None (a row), 32, 64 or 128")
        if getattr(values, "dtype", None) != torch.float8_e4m3fn or values.dim() != 2:
            raise ValueError("values must be a two-dimensional float8_e4m3fn tensor")
        rows, cols = values.shape
        groups = 1 if group is None else (cols + group - 1) // group
        if getattr(scales, "dtype", None) != torch.float32 or tuple(scales.shape) != (rows, groups) or not scales.is_contiguous():
            raise ValueError(f"scales must be a contiguous float32 tensor of shape {(rows, groups)}")
        if scales.device != values.device:
            raise ValueError("values and scales must be on one device")
        self.values, self.scales, self.group = values, scales, group

    rows = property(lambda self: self.values.shape[0])
    cols = property(lambda self: self.values.shape[1])

    @property
    def device(self):
        return self.values.device


def _fp8(values, scales, group):
    """Arrays that were made for it."""
    m = object.__new__(Fp8Matrix)
    m.values, m.scales, m.group = values, scales, group
    return m


_codes = {}


def _code_of(dtype):
    if not _codes:
        import torch
        _codes.update({torch.float32: capi.T_F32, torch.float16: capi.T_F16, torch.bfloat16: capi.T_BF16, torch.float8_e4m3fn: capi.T_E4M3})
    try:
        return _codes[dtype]
    except (KeyError, TypeError):
        raise TypeError("dtype must be float32, float16, bfloat16 or float8_e4m3fn") from None


def rms_norm(X, weight=None, eps: float = 1e-6, residual=None, sum_out=None, dtype=None, group: int | None = None, out=None, stream=None):
    """y = h / sqrt(mean(h²) + eps) * weight for the rows of X [rows, cols] (float32, float16 or bfloat16), h = X, or X + ``residual``
    (X's type or float32), computed in fp32 and rounded once.

    ``dtype``: y's (X's; with ``out``, its type); float8_e4m3fn gives an Fp8Matrix, with a scale of each row or, with ``group``, of so many columns.
    ``weight``: [cols], any of the three types.  Returns y, or with a residual (y, h), h in the residual's type in a new tensor or in ``sum_out``,
    which may be ``residual`` itself, or X.  ``out``: a tensor, or an Fp8Matrix, for y; a tensor may be X.  Inputs that require a gradient
    while gradients are recorded, or have a tangent, are refused: there is none.  What is written in place is new to autograd."""
    if stream is not None:
        mine = (out.values, out.scales) if isinstance(out, Fp8Matrix) else (out,)
        with _on(stream, *(t for t in (X, weight, residual, sum_out, *mine) if t is not None)):
            return rms_norm(X, weight, eps, residual, sum_out, dtype, group, out)
    eights = type(out) is Fp8Matrix
    if dtype is None:
        code = capi.T_E4M3 if eights else _code_of(out.dtype if out is not None else getattr(X, "dtype", None))
    else:
        code = _code_of(dtype)
    if (code == capi.T_E4M3) != eights and out is not None:
        raise ValueError("out must be an Fp8Matrix for float8_e4m3fn, else a tensor")
    if eights and group is None:
        group = out.group
    if group is not None and (code != capi.T_E4M3 or group not in GROUPS):
        raise ValueError("group must be None, 32, 64 or 128, and is for float8_e4m3fn alone")
    if eights and out.group != group:
        raise ValueError("out has scales for another group")
    y, scales, h = _lib().rms_norm(X, weight, eps, residual, sum_out, out.values if eights else out, out.scales if eights else None, code, group or 0)
    if type(y) is int:
        raise capi.SpmmError(y, "b200spmm_rms_norm")
    if code == capi.T_E4M3:
        y = out if eights else _fp8(y, scales, group)
    return y if residual is None else (y, h)
