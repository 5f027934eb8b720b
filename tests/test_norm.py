"""The RMS norm without a GPU: its refusals, which come before any device is touched."""
import ctypes as C

import pytest
import torch

import hopper_spmm_b200 as hs
from hopper_spmm_b200 import _capi as capi

NO_GPU = not torch.cuda.is_available()
E4M3 = torch.float8_e4m3fn


def call(**kw):
    p = dict(rows=4, cols=64, x_dtype=capi.T_F16, r_dtype=capi.T_F16, w_dtype=capi.T_F16, out_dtype=capi.T_F16, group=0, device=0, x=4096, residual=4096, weight=4096,
             sum=8192, out=8192, scales=8192, ldx=64, ldr=64, lds=64, ldo=64, eps=1e-6)
    p.update(kw)
    return capi.lib().b200spmm_rms_norm(C.byref(capi.RmsNorm(**p)), None)


@pytest.mark.parametrize("kw", [dict(x_dtype=3), dict(x_dtype=7), dict(out_dtype=4), dict(r_dtype=capi.T_BF16), dict(r_dtype=3), dict(w_dtype=3), dict(x=0), dict(x=4097), dict(ldx=63),
                                dict(residual=4097), dict(ldr=63), dict(sum=4097), dict(lds=63), dict(residual=0), dict(out=0), dict(out=4097), dict(ldo=63), dict(weight=4097),
                                dict(eps=-1.0), dict(eps=float("nan")), dict(group=32), dict(out_dtype=capi.T_E4M3, group=16), dict(out_dtype=capi.T_E4M3, group=48),
                                dict(out_dtype=capi.T_E4M3, scales=0), dict(out_dtype=capi.T_E4M3, scales=4098), dict(out_dtype=capi.T_E4M3, ldo=63)], ids=str)
def test_refusals_come_before_any_device_is_touched(kw):
    assert call(**kw) == capi.ERR_INVALID_ARG


def test_other_refusals():
    assert capi.lib().b200spmm_rms_norm(None, None) == capi.ERR_INVALID_ARG
    assert call(cols=2**31) == capi.ERR_UNSUPPORTED
    if NO_GPU:
        for kw in ({}, dict(residual=0, sum=0), dict(weight=0), dict(out_dtype=capi.T_E4M3, group=64), dict(rows=0), dict(device=-1)):
            assert call(**kw) == capi.ERR_NO_DEVICE


def test_python_refusals():
    x = torch.randn(4, 64)
    for bad in (x, x.half(), 3):
        with pytest.raises((ValueError, TypeError)):
            hs.rms_norm(bad)
    with pytest.raises(ValueError, match="X must be"):
        hs.rms_norm(x)
    with pytest.raises(TypeError):
        hs.rms_norm(x, dtype=torch.float64)
    with pytest.raises(ValueError, match="group"):
        hs.rms_norm(x, group=32)
    with pytest.raises(ValueError, match="group"):
        hs.rms_norm(x, dtype=E4M3, group=48)
    v, s = torch.zeros(4, 70).to(E4M3), torch.zeros(4, 3)
    m = hs.Fp8Matrix(v, s, 32)
    assert (m.rows, m.cols, m.group) == (4, 70, 32)
    with pytest.raises(ValueError, match="out must be"):
        hs.rms_norm(x, out=m, dtype=torch.float16)
    with pytest.raises(ValueError, match="out must be"):
        hs.rms_norm(x, out=x, dtype=E4M3)
    with pytest.raises(ValueError, match="another group"):
        hs.rms_norm(x, out=m, group=64)
    for args in ((v, s), (v, s, 48), (v, s, 64), (x, s, 32), (v[0], s, 32), (v, s.double(), 32), (v, s.t().contiguous().t(), 32), (None, s, 32), (v, None, 32)):
        with pytest.raises(ValueError):
            hs.Fp8Matrix(*args)


def test_a_stream_of_another_device_is_refused():
    class Stream:
        device = torch.device("cuda", 1)
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="one device"):
        hs.rms_norm(x, stream=Stream())
    with pytest.raises(ValueError, match="one device"):
        hs.rms_norm(x, out=hs.Fp8Matrix(x.to(E4M3), torch.zeros(4, 1)), stream=Stream())
