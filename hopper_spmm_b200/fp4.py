"""Dense matrices in 4 bits a value, and their products (b200spmm_fp4_* of the C ABI).

Beside the sparse forms of a weight matrix (``SpmmPlan``) stands the other way to make one smaller, fewer bits: e2m1 values with
one scale per block of 16 (``nvfp4``) or 32 (``mxfp4``) neighbours of a row.  The reference has no such form (src/common.h:14-43).

    W = fp4_quantize(weights)                      # [rows, cols] float32 / float16 / bfloat16, once
    C = W.matmul(B)                                # B [cols, n] float16 or bfloat16: [rows, n], as SpmmPlan.spmm
    C = W.matmul(fp4_quantize(X))                  # X [n, cols], both operands in 4 bits
    W.matmul(x.t(), y.t(), dtype=y.dtype)          # activations that lie token by token, x [n, cols], y [n, rows]

As everywhere in this package, what computes runs in libb200spmm.so; there is no fallback.
"""
from __future__ import annotations

import contextlib

from . import _capi as capi

FORMATS = {"nvfp4": capi.NVFP4, "mxfp4": capi.MXFP4}
_BLOCK = {"nvfp4": 16, "mxfp4": 32}

_native = None


def _lib():
    """The native half of these calls; like the library itself it has no fallback."""
    global _native
    if _native is None:
        import torch  # noqa: F401  (the module links against torch's libraries)
        capi.lib()
        try:
            from . import _torch_binding
        except ImportError as e:
            raise RuntimeError("hopper_spmm_b200/_torch_binding.so is missing or unusable: build it with "
                               "`python -m hopper_spmm_b200.build`") from e
        _native = _torch_binding
    return _native


_types = {}


def _type_code(dtype):
    if not _types:
        import torch
        _types.update({torch.float32: capi.T_F32, torch.float16: capi.T_F16, torch.bfloat16: capi.T_BF16})
    try:
        return _types[dtype]
    except (KeyError, TypeError):
        raise TypeError("dtype must be float32, float16 or bfloat16") from None


@contextlib.contextmanager
def _on(stream, *tensors):
    """Work and new tensors on `stream`, which the caching allocator is told about for the tensors of the call."""
    import torch
    if any(getattr(t, "device", stream.device) != stream.device for t in tensors):
        raise ValueError("the stream and the tensors must be on one device")
    with torch.cuda.stream(stream):
        yield
    for t in tensors:
        if t is not None:
            t.record_stream(stream)


class Fp4Matrix:
    """A rows x cols matrix in 4 bits.  ``values`` uint8 [rows, pitch], ``scales`` uint8 and ``tensor_scale`` float32 [1] are CUDA
    tensors in the layout that include/b200_spmm.h describes: give them (a checkpoint in that layout), or leave them
    out for a matrix that ``fp4_quantize(..., out=)`` fills."""

    __slots__ = ("format", "_m")  # the format's name; values, scales, tensor_scale, rows, cols, the format's code

    def __init__(self, rows: int, cols: int, format: str = "nvfp4", *, values=None, scales=None, tensor_scale=None, device=None):
        import torch
        if format not in FORMATS:
            raise ValueError(f"format must be one of {', '.join(FORMATS)}")
        rows, cols = int(rows), int(cols)
        if rows < 0 or cols < 0 or rows > 0x7FFFFFFF - 128 or cols > 0x7FFFFFFF - 256:
            raise ValueError("rows and cols must lie between 0 and 2^31")
        blk = _BLOCK[format]
        pitch, n_scales = (cols + 31) // 32 * 16, (rows + 127) // 128 * ((cols + 4 * blk - 1) // (4 * blk)) * 512
        if values is None and scales is None:
            if tensor_scale is not None:
                raise ValueError("values and scales are given together")
            device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
            values = torch.empty((rows, pitch), dtype=torch.uint8, device=device)
            scales = torch.empty(n_scales, dtype=torch.uint8, device=device)
            tensor_scale = torch.empty(1, dtype=torch.float32, device=device)
        elif values is None or scales is None or (tensor_scale is None and format == "nvfp4"):
            raise ValueError("values, scales and, for nvfp4, tensor_scale are given together")
        else:
            if tensor_scale is None:
                tensor_scale = torch.ones(1, dtype=torch.float32, device=values.device)
            if (values.dtype != torch.uint8 or values.numel() != rows * pitch or scales.dtype != torch.uint8 or
                    scales.numel() != n_scales or tensor_scale.dtype != torch.float32 or tensor_scale.numel() != 1 or
                    not (values.is_contiguous() and scales.is_contiguous())):
                raise ValueError(f"a {rows} x {cols} {format} matrix takes contiguous uint8 values of {rows * pitch} bytes and scales of "
                                 f"{n_scales} bytes, and one float32 tensor_scale")
        self.format = format
        self._m = (values, scales, tensor_scale, rows, cols, FORMATS[format])

    values = property(lambda self: self._m[0])
    scales = property(lambda self: self._m[1])
    tensor_scale = property(lambda self: self._m[2])
    rows = property(lambda self: self._m[3])
    cols = property(lambda self: self._m[4])

    @property
    def device(self):
        return self.values.device

    @property
    def nbytes(self) -> int:
        return self.values.numel() + self.scales.numel() + 4

    def dequantize(self, out=None, dtype=None, stream=None):
        """The values it stands for, [rows, cols] in ``dtype`` (float32; with ``out``, its type)."""
        code = _type_code(dtype) if dtype is not None else _type_code(out.dtype) if out is not None else capi.T_F32
        if stream is not None:
            with _on(stream, self.values, self.scales, self.tensor_scale, out):
                return self.dequantize(out, dtype)
        out = _lib().fp4_dequantize(*self._m, out, code)
        if type(out) is int:
            raise capi.SpmmError(out, "b200spmm_fp4_dequantize")
        return out

    def matmul(self, B, C_out=None, dtype=None, stream=None, sync: bool = True):
        """This matrix times B: a float16 or bfloat16 tensor [cols, n] (mxfp4: bfloat16), or an Fp4Matrix of n rows with
        blocks along the same columns, whose transpose is meant.  Returns C [rows, n] in ``dtype`` (float32; with
        ``C_out``, its type).  B and C may lie row by row or column by column (``x.t()``)."""
        code = _type_code(dtype) if dtype is not None else _type_code(C_out.dtype) if C_out is not None else capi.T_F32
        if stream is not None:
            mine = (self.values, self.scales, self.tensor_scale, C_out)
            with _on(stream, *mine, *((B.values, B.scales, B.tensor_scale) if isinstance(B, Fp4Matrix) else (B,))):
                C_out = self.matmul(B, C_out, dtype, None, False)
            if sync:
                self.sync(stream)
            return C_out
        if isinstance(B, Fp4Matrix):
            if B.format != self.format:
                raise ValueError("both matrices must have the same format")
            C_out, where = _lib().fp4_product(*self._m, *B._m, C_out, code), "b200spmm_fp4_product"
        else:
            if self.format == "mxfp4" and str(getattr(B, "dtype", None)) == "torch.float16":
                raise ValueError("an mxfp4 matrix takes bfloat16: its scales go beyond the range of float16")
            C_out, where = _lib().fp4_dense_product(*self._m, B, C_out, code), "b200spmm_fp4_dense_product"
        if type(C_out) is int:
            raise capi.SpmmError(C_out, where)
        if sync:
            self.sync()
        return C_out

    def sync(self, stream=None):
        """Waits for ``stream`` (the current one) and raises if a product on this device ran out of time: on whatever stream it
        was, for a thread is told of it on every stream that it uses.  Not while the stream is captured (pass ``sync=False`` there)."""
        import torch
        s = (stream or torch.cuda.current_stream(self.values.device)).cuda_stream
        capi.check(capi.lib().b200spmm_fp4_status(self.values.device.index, s), "b200spmm_fp4_status")


def _matrix(rows, cols, format, values, scales, tensor_scale) -> Fp4Matrix:
    """Arrays that were made for it (the checks of Fp4Matrix cost as much as a launch)."""
    m = object.__new__(Fp4Matrix)
    m.format = format
    m._m = (values, scales, tensor_scale, rows, cols, FORMATS[format])
    return m


def _format_code(format):
    try:
        return FORMATS[format]
    except (KeyError, TypeError):
        raise ValueError(f"format must be one of {', '.join(FORMATS)}") from None


def _quantized(X, format, tensor_scale, by_rows, by_cols):
    made = _lib().fp4_quantize_new(X, tensor_scale, _format_code(format), by_rows, by_cols)
    if type(made) is int:
        raise capi.SpmmError(made, "b200spmm_fp4_quantize")
    return made


def fp4_quantize(X, format: str = "nvfp4", axis: int = 1, tensor_scale=None, out: Fp4Matrix | None = None, stream=None) -> Fp4Matrix:
    """X in 4 bits.  ``axis`` 1: blocks along X's rows, a matrix of X's shape; 0: along its columns, and the matrix is X's
    transpose (the axis that a product sums over has to be the matrix's rows).  ``tensor_scale``: for nvfp4 (mxfp4 has none), a
    positive float32 tensor of one element, say a calibrated one, in place of a pass over X for its largest value.  It is rounded
    up to a power of two, which is the scale that X gets: codes and block scales are those for that one, not for the number as
    it was given.  ``out``: a matrix to fill, else a new one."""
    if axis not in (0, 1):
        raise ValueError("axis must be 0 or 1")
    if stream is not None:
        with _on(stream, X, tensor_scale, *(() if out is None else (out.values, out.scales, out.tensor_scale))):
            return fp4_quantize(X, format, axis, tensor_scale, out)
    if out is None:
        made = _quantized(X, format, tensor_scale, axis == 1, axis == 0)
        return _matrix(X.shape[1 - axis], X.shape[axis], format, *made)
    if out.format != format:
        raise ValueError(f"out must be a matrix of {format}")
    st = _lib().fp4_quantize(X, tensor_scale, *out._m, axis == 0)
    if st is not None:
        raise capi.SpmmError(st, "b200spmm_fp4_quantize")
    return out


def fp4_quantize_both(X, format: str = "nvfp4", tensor_scale=None, stream=None) -> tuple[Fp4Matrix, Fp4Matrix]:
    """``fp4_quantize(X, axis=1)`` and ``fp4_quantize(X, axis=0)`` from one read of X (nvfp4 without ``tensor_scale`` reads it for its
    largest value before): what training needs.  For Y = X Wᵀ the forward pass sums over X's columns, the weights' gradient dYᵀ X
    over its rows:

        X, Xt = fp4_quantize_both(x);  W, Wt = fp4_quantize_both(w);  dY, dYt = fp4_quantize_both(dy)
        y, dx, dw = X.matmul(W), dY.matmul(Wt), dYt.matmul(Xt)
    """
    if stream is not None:
        with _on(stream, X, tensor_scale):
            return fp4_quantize_both(X, format, tensor_scale)
    made = _quantized(X, format, tensor_scale, True, True)
    r, c = X.shape
    return _matrix(r, c, format, *made[:3]), _matrix(c, r, format, *made[3:])
