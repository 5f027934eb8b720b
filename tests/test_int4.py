"""Matrices of 4-bit integers without a GPU: refusals, which come before any device is touched, and the reference that the GPU tests go by."""
import ctypes as C

import pytest
import torch

import hopper_spmm_b200 as hs
from hopper_spmm_b200 import _capi as capi

NO_GPU = not torch.cuda.is_available()


def matrix(**kw):
    p = dict(rows=128, cols=64, group=32, scale_dtype=capi.T_F16, device=0, values=4096, scales=4096, zeros=4096)
    p.update(kw)
    return capi.Int4(**p)


def call(m=None, B=4096, ldb=64, n=64, b_dtype=capi.T_F16, b_t=1, scales=None, group=0, C_=4096, ldc=128, c_dtype=capi.T_F16, c_t=1):
    m = matrix() if m is None else m
    return capi.lib().b200spmm_int4_product(C.byref(m) if m else None, B, ldb, n, b_dtype, b_t, scales, group, C_, ldc, c_dtype, c_t, None)


def test_refusals_come_before_any_device_is_touched():
    bad = capi.ERR_INVALID_ARG
    for kw in (dict(group=16), dict(group=48), dict(group=-32), dict(scale_dtype=capi.T_F32), dict(scale_dtype=3), dict(values=0), dict(scales=0), dict(scales=4097)):
        assert call(matrix(**kw)) == bad, kw
    assert call(matrix(values=4104)) == call(matrix(rows=2**31)) == call(matrix(cols=2**31)) == capi.ERR_UNSUPPORTED
    assert call(False) == call(n=-1) == call(B=0) == call(B=4097) == call(ldb=63) == call(b_dtype=4) == call(C_=0) == call(C_=4097) == call(ldc=127) == call(c_dtype=3) == bad
    assert call(n=65536) == call(b_dtype=capi.T_F32) == capi.ERR_UNSUPPORTED
    assert call(scales=4096) == call(group=32) == bad  # for 8 bits alone
    eights = dict(b_dtype=capi.T_E4M3, scales=4096)
    assert call(**dict(eights, scales=0)) == call(**eights, b_t=0) == call(**eights, group=16) == call(**eights, group=256) == call(**eights, ldb=63) == call(**dict(eights, scales=4098)) == bad
    if NO_GPU:
        for st in (call(), call(**eights), call(**eights, group=64), call(matrix(group=0)), call(matrix(zeros=0)), call(n=0), call(matrix(device=-1)), call(b_t=0, c_t=0, ldc=64)):
            assert st == capi.ERR_NO_DEVICE


def test_python_refusals():
    v, s, z = torch.zeros(5, 48, dtype=torch.uint8), torch.ones(3, 5).half(), torch.zeros(3, 5, dtype=torch.uint8)
    make = lambda rows=5, cols=70, group=32, **kw: hs.Int4Matrix(rows, cols, group, **dict(dict(values=v, scales=s, zeros=z), **kw))  # noqa: E731
    for kw in (dict(values=v[:4]), dict(values=v.int()), dict(values=v.t().contiguous().t()), dict(values=None)):
        with pytest.raises(ValueError, match="values must be"):
            make(**kw)
    for kw in (dict(scales=s.float()), dict(scales=s.t().contiguous()), dict(scales=s[:2]), dict(scales=s.t().contiguous().t())):
        with pytest.raises(ValueError, match="scales must be"):
            make(**kw)
    for kw in (dict(zeros=z.int()), dict(zeros=z[:2]), dict(zeros=3)):
        with pytest.raises(ValueError, match="zeros must be"):
            make(**kw)
    for group in (16, 33, 96, -32):
        with pytest.raises(ValueError, match="group must be"):
            make(group=group)
    with pytest.raises(ValueError, match="rows and cols"):
        make(rows=-1)
    with pytest.raises(ValueError, match="CUDA device"):
        make()
    with pytest.raises(ValueError, match="no backward"):
        make(scales=s.clone().requires_grad_())
