"""Matrices of 4-bit integers with scales and zeros of groups, times a few columns (b200spmm_int4_product of the C ABI).

Beside the 4-bit floating-point forms (``Fp4Matrix``), whose scales are of 16 or 32 neighbours, stands the form that most checkpoints in 4 bits
have: (code - zero) * scale for every 32, 64, 128 ... neighbours of a row.  The reference has neither (src/common.h:14-43).

    W = Int4Matrix(rows, cols, 128, values=values, scales=scales, zeros=zeros)
    y = W.linear(x)                       # x [n, cols] float16 or bfloat16, token by token: [n, rows]
    y = W.linear(rms_norm(x, w, dtype=torch.float8_e4m3fn))   # activations in 8 bits
    C = W.matmul(B)                       # B [cols, n]: [rows, n], as Fp4Matrix.matmul and SpmmPlan.spmm
"""
from __future__ import annotations

from . import _capi as capi
from .fp4 import _lib, _on, _type_code
from .norm import Fp8Matrix


class Int4Matrix:
    """A rows x cols matrix of 4-bit integers.  ``group``: neighbours of a row that share a scale, a power of two from 32 on, or None for a whole row.
    ``values`` uint8 [rows, pitch]: two codes from 0 to 15 to a byte, the lower half first, pitch 16 bytes for every 32 columns begun.  ``scales``
    float16 or bfloat16 [groups of a row, rows].  ``zeros`` uint8 [groups of a row, rows], 0 to 15; None: 8 everywhere.  All contiguous, on one CUDA
    device; they are kept, not copied: their values may change, and a call refuses them once they have another storage, type or shape."""

    __slots__ = ("rows", "cols", "group", "_arrays", "_m")

    def __init__(self, rows: int, cols: int, group: int | None = 128, *, values, scales, zeros=None):
        self._m = _lib().int4_matrix(values, scales, zeros, rows, cols, group or 0)
        self._arrays = (values, scales, zeros)
        self.rows, self.cols, self.group = rows, cols, group

    values = property(lambda self: self._arrays[0])
    scales = property(lambda self: self._arrays[1])
    zeros = property(lambda self: self._arrays[2])

    @property
    def device(self):
        return self.values.device

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self._arrays if t is not None)

    def _product(self, B, out, dtype, stream, first):
        code = _type_code(dtype) if dtype is not None else _type_code(out.dtype) if out is not None else capi.T_F32
        eights = type(B) is Fp8Matrix
        if stream is not None:
            with _on(stream, *(t for t in (*self._arrays, out, *((B.values, B.scales) if eights else (B,))) if t is not None)):
                return self._product(B, out, dtype, None, first)
        if eights:
            out = _lib().int4_product(self._m, B.values, B.scales, B.group or 0, out, code, first)
        else:
            out = _lib().int4_product(self._m, B, None, 0, out, code, first)
        if type(out) is int:
            raise capi.SpmmError(out, "b200spmm_int4_product")
        return out

    def linear(self, X, out=None, dtype=None, stream=None):
        """Y = X Wᵀ, [n, rows], for a few tokens that lie row by row: X [n, cols] float16 or bfloat16, or an Fp8Matrix.  Y in ``dtype`` (float32; with
        ``out``, its type); sums in fp32.  The matrix is read once for every 40 rows of X, of which there may be 65,535.  Asynchronous; there is no gradient: X may
        not require one while gradients are recorded, nor have a tangent."""
        return self._product(X, out, dtype, stream, True)

    def matmul(self, B, C_out=None, dtype=None, stream=None):
        """C = W B, [rows, n], for B [cols, n] float16 or bfloat16, or an Fp8Matrix of n rows, whose transpose is meant; else as ``linear``.  B and C may lie
        row by row or column by column (``x.t()``)."""
        return self._product(B, C_out, dtype, stream, False)
