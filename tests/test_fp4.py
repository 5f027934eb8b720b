"""4-bit matrices without a GPU: layout, argument checks, and the reference that the GPU tests go by."""
import ctypes as C

import pytest
import torch

import fp4_ref as ref
import hopper_spmm_b200 as hs
from hopper_spmm_b200 import _capi as capi

NO_GPU = not torch.cuda.is_available()


def sizes(rows, cols, fmt):
    out = [C.c_uint64() for _ in range(4)]
    st = capi.lib().b200spmm_fp4_sizes(rows, cols, fmt, *(C.byref(o) for o in out))
    return st, tuple(o.value for o in out)


@pytest.mark.parametrize("rows,cols", [(0, 0), (0, 5), (5, 0), (1, 1), (3, 16), (128, 32), (129, 33), (1000, 4095), (28672, 8192), (2**31 - 200, 2**31 - 300)])
def test_sizes(rows, cols):
    for fmt, name in ((capi.NVFP4, "nvfp4"), (capi.MXFP4, "mxfp4")):
        st, (pitch, values, scales, workspace) = sizes(rows, cols, fmt)
        blocks = -(-cols // ref.BLOCK[name])
        assert st == capi.OK and pitch == -(-cols // 32) * 16 and values == rows * pitch
        assert scales == -(-rows // 128) * -(-blocks // 4) * 512 and workspace > 0
    assert sizes(1, 1, 2)[0] == capi.ERR_INVALID_ARG and sizes(2**31, 1, 0)[0] == capi.ERR_UNSUPPORTED
    assert capi.lib().b200spmm_fp4_sizes(4, 4, 0, None, None, None, None) == capi.OK


def matrix(rows=128, cols=64, fmt=capi.NVFP4, values=4096, scales=4096, scale=4096, device=0):
    return capi.Fp4(rows, cols, fmt, device, values, scales, scale)


def calls(m=None, other=None, x=4096, ld=64, dtype=capi.T_F16, n=64, ws=4096):
    """Every entry with these arguments (addresses that nothing reads, for a refusal comes first)."""
    l, m = capi.lib(), m or matrix()
    p, q = C.byref(m), C.byref(other or matrix(n, m.cols, m.format))
    t = matrix(m.cols, m.rows, m.format)
    return {"quantize": l.b200spmm_fp4_quantize(x, ld, dtype, 0, None, p, ws, None),
            "both": l.b200spmm_fp4_quantize_both(x, ld, dtype, None, p, C.byref(t), ws, None),
            "dequantize": l.b200spmm_fp4_dequantize(p, x, ld, dtype, None),
            "product": l.b200spmm_fp4_product(p, q, x, ld, dtype, 0, None, 0, None),
            "dense": l.b200spmm_fp4_dense_product(p, x, ld, n, dtype, 0, x, ld, dtype, 0, None, 0, None)}


def test_refusals_come_before_any_device_is_touched():
    bad = capi.ERR_INVALID_ARG
    for name, st in calls(matrix(fmt=7)).items():
        assert st == bad, name
    for m in (matrix(values=0), matrix(scales=0), matrix(scale=0), matrix(scale=4098)):
        assert set(calls(m).values()) == {bad}
    assert set(calls(matrix(values=4104)).values()) == {capi.ERR_UNSUPPORTED} == set(calls(matrix(scales=4100)).values())
    assert set(calls(x=0).values()) == {bad} == set(calls(x=4097).values()) == set(calls(ld=63).values()) == set(calls(dtype=3).values())
    assert calls(matrix(rows=2**31))["dequantize"] == capi.ERR_UNSUPPORTED
    # shapes, formats and types that do not go together
    assert calls(other=matrix(64, 65))["product"] == bad == calls(other=matrix(64, 64, device=1))["product"]
    assert calls(other=matrix(64, 64, capi.MXFP4))["product"] == capi.ERR_UNSUPPORTED
    assert calls(dtype=capi.T_F32)["dense"] == capi.ERR_UNSUPPORTED
    assert calls(matrix(fmt=capi.MXFP4), dtype=capi.T_F16)["dense"] == capi.ERR_UNSUPPORTED
    assert calls(ws=0)["quantize"] == bad == calls(ws=0)["both"] == calls(ws=4098)["quantize"]
    assert calls(n=-1, other=matrix(64, 64))["dense"] == bad
    l, m = capi.lib(), matrix()
    assert l.b200spmm_fp4_quantize(4096, 64, capi.T_F16, 0, None, None, 4096, None) == bad
    assert l.b200spmm_fp4_quantize_both(4096, 64, capi.T_F16, None, C.byref(m), C.byref(m), 4096, None) == bad  # not each other's transpose
    assert l.b200spmm_fp4_dequantize(None, 4096, 64, capi.T_F16, None) == bad
    assert l.b200spmm_fp4_product(C.byref(m), C.byref(m), 4096, 128, capi.T_F16, 0, 4097, 100, None) == bad
    size = C.c_uint64()
    assert l.b200spmm_fp4_product_workspace(C.byref(m), None, 0, 8, 0, None) == bad
    assert l.b200spmm_fp4_product_workspace(C.byref(m), None, 0, -1, 0, C.byref(size)) == bad


@pytest.mark.skipif(not NO_GPU, reason="a device is present")
def test_no_device_is_an_error_not_a_fallback():
    assert set(calls().values()) == {capi.ERR_NO_DEVICE}
    assert capi.lib().b200spmm_fp4_status(0, None) == capi.ERR_NO_DEVICE
    assert set(calls(matrix(device=-1)).values()) >= {capi.ERR_NO_DEVICE}


def test_python_refusals():
    x = torch.randn(4, 64)
    for bad in (x, x.half(), x.cuda() if not NO_GPU else None, 3):
        if bad is not None and getattr(bad, "is_cuda", False):
            continue
        with pytest.raises(ValueError, match="X must be a two-dimensional CUDA tensor"):
            hs.fp4_quantize(bad)
        with pytest.raises(ValueError, match="X must be a two-dimensional CUDA tensor"):
            hs.fp4_quantize_both(bad, "mxfp4")
    with pytest.raises(ValueError, match="format"):
        hs.fp4_quantize(x, "fp4")
    with pytest.raises(ValueError, match="axis"):
        hs.fp4_quantize(x, axis=2)
    with pytest.raises(ValueError, match="format"):
        hs.Fp4Matrix(4, 4, "int4")
    with pytest.raises(ValueError, match="rows and cols"):
        hs.Fp4Matrix(-1, 4)
    u8 = lambda n: torch.zeros(n, dtype=torch.uint8)
    one = torch.ones(1)
    for kw in ({"values": u8(64)}, {"values": u8(64), "scales": u8(512)}, {"tensor_scale": one}, {"values": u8(63), "scales": u8(512), "tensor_scale": one},
               {"values": u8(64), "scales": u8(511), "tensor_scale": one}, {"values": u8(64).int(), "scales": u8(512), "tensor_scale": one},
               {"values": u8(64), "scales": u8(512), "tensor_scale": one.double()}, {"values": u8(128)[::2], "scales": u8(512), "tensor_scale": one}):
        with pytest.raises(ValueError):
            hs.Fp4Matrix(4, 20, **kw)
    m = hs.Fp4Matrix(4, 20, values=u8(64), scales=u8(512), tensor_scale=one)  # in host memory: nothing can be done with it
    assert m.nbytes == 64 + 512 + 4 and m.device.type == "cpu"
    with pytest.raises(ValueError, match="CUDA device"):
        m.dequantize()
    with pytest.raises(ValueError, match="CUDA device"):
        m.matmul(torch.zeros(20, 3).half())
    with pytest.raises(ValueError, match="same format"):
        m.matmul(hs.Fp4Matrix(4, 20, "mxfp4", values=u8(64), scales=u8(512)))
    with pytest.raises(TypeError):
        m.matmul(torch.zeros(20, 3).half(), dtype=torch.float64)
    with pytest.raises(TypeError):
        m.dequantize(dtype=torch.int8)
    with pytest.raises(ValueError, match="bfloat16"):
        hs.Fp4Matrix(4, 20, "mxfp4", values=u8(64), scales=u8(512)).matmul(torch.zeros(20, 3).half())


def test_the_reference_rounds_as_the_types_do():
    # torch's own e4m3 for the table and for ties
    a = torch.cat([ref.e4m3_values(), (ref.e4m3_values()[1:] + ref.e4m3_values()[:-1]) / 2, torch.rand(4000, dtype=torch.float64) * 448])
    assert torch.equal(ref.e4m3_values()[ref.nearest(a, ref.e4m3_values())], a.float().to(torch.float8_e4m3fn).double())
    # ties of e2m1 go to even codes
    v = torch.tensor(ref.E2M1, dtype=torch.float64)
    assert ref.nearest((v[1:] + v[:-1]) / 2, v).tolist() == [0, 2, 2, 4, 4, 6, 6]
    # the tensor's exponent at the ends and next to a power of two
    for amax, k in ((2688.0, 0), (2688.0 * (1 + 2**-23), 1), (1344.0, -1), (1e-44, -126), (3.4e38, 117), (0.0, 0)):
        assert ref.tensor_exponent(torch.tensor([[amax, 0.0]], dtype=torch.float32)) == k


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_the_reference_stores_what_it_reads(fmt):
    x = torch.randn(200, 77, generator=torch.Generator().manual_seed(1)) * 3
    code, byte, k = ref.quantize(x, fmt)
    values, scales = ref.pack(code, byte, fmt)
    c, b = ref.unpack(values, scales, 200, 77, fmt)
    assert torch.equal(c, code) and torch.equal(b, byte)
    # Off by at most half the widest gap between codes, 4 to 6, which is one scale, or by what is beyond 6.  nvfp4: the scale is amax / 6 (1 + d) with
    # |d| <= 2^-4 (half a step of e4m3), so one scale is at most amax 17 / 96, and amax lies at most 6 / (1 - 2^-4) - 6 = 0.4 scales beyond 6.
    # mxfp4: amax lies in [4, 8) scales, so one scale is at most amax / 4, and what is beyond 6, under 2 of 8, under amax / 4.
    off = (ref.values(code, byte, k, fmt) - x.double()).abs()
    blk = ref.BLOCK[fmt]
    top = torch.nn.functional.pad(x.abs(), (0, -77 % blk)).view(200, -1, blk).amax(2).repeat_interleave(blk, 1)[:, :77]
    assert (off <= top.double() * (17 / 96 if fmt == "nvfp4" else 1 / 4) * 1.0001).all()


def test_a_stream_of_another_device_is_refused():
    class Stream:
        device = torch.device("cuda", 1)
    x, one = torch.zeros(4, 20), torch.ones(1)
    m = hs.Fp4Matrix(4, 20, values=torch.zeros(64, dtype=torch.uint8), scales=torch.zeros(512, dtype=torch.uint8), tensor_scale=one)
    for call in (lambda: hs.fp4_quantize(x, stream=Stream()), lambda: hs.fp4_quantize_both(x, stream=Stream()), lambda: hs.fp4_quantize(x, out=m, stream=Stream()),
                 lambda: m.dequantize(stream=Stream()), lambda: m.matmul(x.t().half(), stream=Stream()), lambda: m.matmul(m, stream=Stream())):
        with pytest.raises(ValueError, match="one device"):
            call()


def test_the_arrays_of_a_matrix_are_not_exchanged():
    m = hs.Fp4Matrix(4, 20, values=torch.zeros(64, dtype=torch.uint8), scales=torch.zeros(512, dtype=torch.uint8), tensor_scale=torch.ones(1))
    for name in ("values", "scales", "tensor_scale", "rows", "cols"):
        with pytest.raises(AttributeError):
            setattr(m, name, getattr(m, name))


def test_the_starving_of_products_takes_a_limit_and_an_operand():
    starve = capi.lib().b200spmm_kat_fp4_starve
    assert starve(2_000_000_001, 0) == starve(1, 2) == starve(1, -1) == capi.ERR_INVALID_ARG
    assert starve(5_000_000, 1) == starve(0, 0) == capi.OK


def test_no_kernel_reads_through_the_read_only_path():
    # What the kernels read may be written while they start (they wait for it inside); a load through the read-only path, or one that the compiler
    # may take for such (const and restrict), could be moved before that wait.
    import glob
    import os
    import re
    csrc = os.path.join(os.path.dirname(os.path.abspath(hs.__file__)), "csrc")
    files = sorted(glob.glob(os.path.join(csrc, "fp4*")))
    assert len(files) >= 10
    for f in files:
        with open(f) as source:
            found = re.findall(r"__ldg\w*|__restrict\w*|\w*global_nc\w*|ld\.global\.nc", source.read())
        assert not found, (f, found)


@pytest.mark.parametrize("sms", [148, 132, 7])
def test_few_columns_are_shared_out_evenly(sms):
    # no round goes through all of k for a few tiles left over: all rounds together have room for less than one tile a round more than there are
    for rows in [1, 16, 17, 128, 1000, 2048, 4096, 14331, 28672, 30000, 32000, 32768, 50257, 57344, 128256, 151936, 256000, 1000003]:
        for cols in (1, 100, 4096):
            out = [C.c_uint32() for _ in range(4)]
            assert capi.lib().b200spmm_kat_fp4_narrow_share(rows, cols, sms, *(C.byref(o) for o in out)) == capi.OK
            blocks, rounds, at_once, slices = (o.value for o in out)
            tiles = -(-rows // 16)
            most = -(-tiles // blocks)  # of a block
            assert blocks == min(tiles, sms) and most <= rounds * at_once < most + rounds
            assert 1 <= slices <= max(1, -(-cols // 128)) and at_once * slices + 3 <= 32 and at_once * 16 <= 256
    assert capi.lib().b200spmm_kat_fp4_narrow_share(16, 16, 0, *(C.byref(o) for o in out)) == capi.ERR_INVALID_ARG


@pytest.mark.parametrize("rows,blocks", [(1, 1), (128, 4), (130, 5), (300, 33)])
def test_scales_that_lie_row_by_row_are_brought_into_order(rows, blocks):
    # the two lines that the documents give for checkpoints
    s = torch.randint(0, 127, (rows, blocks), dtype=torch.uint8, generator=torch.Generator().manual_seed(rows))
    R, G = -(-rows // 128), -(-s.shape[1] // 4)
    scales = torch.nn.functional.pad(s, (0, G * 4 - s.shape[1], 0, R * 128 - rows)).view(R, 4, 32, G, 4).permute(0, 3, 2, 1, 4).reshape(-1)
    assert torch.equal(scales, ref.pack(torch.zeros(rows, blocks * 16, dtype=torch.uint8), s, "nvfp4")[1])
