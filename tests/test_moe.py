"""The mixture-of-experts layer without a GPU: refusals, which come before any device is touched."""
import ctypes as C

import pytest
import torch

import hopper_spmm_b200 as hs
from hopper_spmm_b200 import _capi as capi

NO_GPU = not torch.cuda.is_available()
E, H, I = 4, 64, 40


def codes(rows, cols, **kw):
    return capi.Int4(**dict(dict(rows=rows, cols=cols, group=32, scale_dtype=capi.T_F16, device=0, values=4096, scales=4096, zeros=4096), **kw))


def layer(int4=False, up=None, low=None, **kw):
    p = dict(experts=E, hidden=H, inner=I, top_k=2, renormalize=1, dtype=capi.T_F16, device=0, router=4096, ld_router=H)
    if int4:
        p.update(gate_up=C.pointer(up or codes(E * 2 * I, H)), down=C.pointer(low or codes(E * H, I)))
    else:
        p.update(gate_up_16=4096, down_16=4096, ld_gate_up=H, ld_down=I)
    p.update(kw)
    return capi.Moe(**p)


def forward(m=None, x=4096, ldx=H, tokens=3, y=4096, ldy=H, ids=None, shares=None, ws=4096, bytes_=1 << 20):
    return capi.lib().b200spmm_moe(C.byref(m if m is not None else layer()), x, ldx, tokens, y, ldy, ids, shares, ws, bytes_, None)


def experts(m=None, x=4096, tokens=3, ids=4096, id_bytes=4, shares=4096, ws=4096, bytes_=1 << 20):
    return capi.lib().b200spmm_moe_experts(C.byref(m if m is not None else layer()), x, H, tokens, ids, id_bytes, shares, 4096, H, ws, bytes_, None)


BAD = [dict(dtype=capi.T_F32), dict(dtype=3), dict(experts=0), dict(hidden=0), dict(inner=0), dict(top_k=0), dict(gate_up_16=0), dict(down_16=0), dict(ld_gate_up=H - 8), dict(ld_down=I - 8),
       dict(gate_up=C.pointer(codes(E * 2 * I, H))), dict(gate_up=C.pointer(codes(E * 2 * I, H)), gate_up_16=0)]


@pytest.mark.parametrize("kw", BAD, ids=lambda k: ",".join(k))
def test_refusals_of_a_layer(kw):
    size = C.c_uint64()
    for st in (forward(layer(**kw)), experts(layer(**kw)), capi.lib().b200spmm_moe_workspace(C.byref(layer(**kw)), 3, C.byref(size))):
        assert st == capi.ERR_INVALID_ARG


def test_other_refusals():
    bad, no = capi.ERR_INVALID_ARG, capi.ERR_UNSUPPORTED
    for kw in (dict(experts=1025), dict(top_k=33), dict(ld_gate_up=H + 4), dict(ld_down=I + 4), dict(gate_up_16=4104), dict(down_16=4098)):
        assert forward(layer(**kw)) == experts(layer(**kw)) == no, kw
    for kw in (dict(up=codes(E * 2 * I + 1, H)), dict(low=codes(E * H, I + 1)), dict(up=codes(E * 2 * I, H, group=16)), dict(low=codes(E * H, I, device=1)), dict(low=codes(E * H, I, values=0))):
        assert forward(layer(True, **kw)) == experts(layer(True, **kw)) == bad, kw
    for kw in (dict(router=0), dict(router=4097), dict(ld_router=H - 1), dict(top_k=5)):
        assert forward(layer(**kw)) == bad, kw
    assert forward(tokens=-1) == forward(x=0) == forward(x=4097) == forward(ldx=H - 1) == forward(y=0) == forward(ldy=H - 1) == forward(ws=0) == forward(ws=4100) == forward(bytes_=64) == bad
    assert forward(ids=4098) == forward(shares=4098) == experts(id_bytes=2) == experts(ids=0) == experts(ids=4098) == experts(ids=4100, id_bytes=8) == experts(shares=0) == experts(shares=4098) == bad
    assert forward(tokens=257) == experts(tokens=257) == no
    size = C.c_uint64()
    l = capi.lib()
    assert l.b200spmm_moe_workspace(C.byref(layer()), 3, None) == l.b200spmm_moe_workspace(C.byref(layer()), -1, C.byref(size)) == bad
    assert l.b200spmm_moe_workspace(C.byref(layer()), 257, C.byref(size)) == no
    assert l.b200spmm_moe_workspace(C.byref(layer()), 3, C.byref(size)) == capi.OK and size.value >= 3 * 2 * (H + I) * 4
    if NO_GPU:
        for st in (forward(), experts(), forward(layer(True)), forward(tokens=0), experts(layer(router=0, top_k=5)), forward(layer(device=-1))):
            assert st == capi.ERR_NO_DEVICE


def test_python_refusals():
    r, g, d = torch.zeros(E, H).half(), torch.zeros(E, 2 * I, H).half(), torch.zeros(E, H, I).half()
    make = lambda router=r, gate_up=g, down=d, top_k=2, **kw: hs.MoeLayer(router, gate_up, down, top_k=top_k, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="CUDA device"):
        make()
    for kw in (dict(router=r.float()), dict(router=torch.zeros(E, 2 * H).half()[:, ::2]), dict(router=r[:, :32])):
        with pytest.raises(ValueError, match="router must"):
            make(**kw)
    for kw in (dict(gate_up=g.float()), dict(gate_up=g[:, 1:]), dict(down=d[:3]), dict(down=d[:, :32])):
        with pytest.raises(ValueError, match="gate_up must"):
            make(**kw)
    for kw in (dict(gate_up=g[0]), dict(down=None)):
        with pytest.raises(ValueError, match="gate_up must"):
            make(**kw)
    odd = torch.zeros(E, H, I + 1).half()
    with pytest.raises(ValueError, match="16 bytes"):
        make(down=odd[:, :, :I])
    with pytest.raises(ValueError, match="one type"):
        make(down=d.bfloat16())
    for top in (0, 33, 5):
        with pytest.raises(ValueError, match="top_k"):
            make(top_k=top)
    with pytest.raises(ValueError, match="another number"):
        make(experts=5)
    with pytest.raises(ValueError, match="no backward"):
        make(router=r.clone().requires_grad_())
