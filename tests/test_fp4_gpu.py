"""4-bit matrices on the GPU: stored bytes against the definition in 64 bits, products against 64-bit products of what the
matrices stand for."""
import ctypes as C

import pytest
import torch

import fp4_ref as ref
import hopper_spmm_b200 as hs
from hopper_spmm_b200 import _capi as capi

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
FORMATS = ["nvfp4", "mxfp4"]
IDS = {F32: "f32", F16: "f16", BF16: "bf16"}.get


def normal(r, c, seed, dtype=F32, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(r, c, generator=g, device="cuda") * spread
    x[:, ::37] *= 20
    return x.to(dtype)


def check_quantized(m, x, k=None):
    """m holds exactly what x is in 4 bits, byte for byte (rows of scales past the last may hold anything)."""
    code, byte, k = ref.quantize(x, m.format, k)
    assert (m.rows, m.cols) == tuple(x.shape)
    values, _ = ref.pack(code, byte, m.format)
    assert torch.equal(m.values, values), f"{int((m.values != values).sum())} bytes of values differ"
    R, G = x.shape[0], (byte.shape[1] + 3) // 4 * 4
    got = m.scales[ref.scale_index(R, G).cuda()]
    assert torch.equal(got[:, :byte.shape[1]], byte), "scales differ"
    assert not got[:, byte.shape[1]:].any(), "scales behind a row's last are not zero"
    assert float(m.tensor_scale) == 2.0 ** k


SHAPES = [(1, 1), (1, 16), (3, 17), (2, 8190), (130, 64), (257, 129), (33, 1000), (64, 31), (300, 515), (1024, 2048)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_quantize_is_the_definition_byte_for_byte(shape, dtype, fmt):
    x = normal(*shape, seed=sum(shape), dtype=dtype)
    check_quantized(hs.fp4_quantize(x, fmt), x)
    check_quantized(hs.fp4_quantize(x, fmt, axis=0), x.t())
    a, b = hs.fp4_quantize_both(x, fmt)
    check_quantized(a, x)
    check_quantized(b, x.t())


@pytest.mark.parametrize("fmt", FORMATS)
def test_strides_offsets_and_transposed_views(fmt):
    whole = normal(300, 701, 5, F16)
    for x in (whole[:, 8:600], whole[3:, 1:98], whole[::2, :], whole[:, :1], whole[:1, 3:], whole.t()[5:77, :], whole.t()[:, 9:17]):
        check_quantized(hs.fp4_quantize(x, fmt), x)
        check_quantized(hs.fp4_quantize(x, fmt, axis=0), x.t())
        a, b = hs.fp4_quantize_both(x, fmt)
        check_quantized(a, x)
        check_quantized(b, x.t())


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS)
@pytest.mark.parametrize("fmt", FORMATS)
def test_values_on_and_next_to_the_borders_between_codes(fmt, dtype):
    # every border times every digit of a scale, and its neighbours in the type, in blocks whose largest value sets the scale
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda")
    rows = []
    for digits in range(8, 16):
        for e in (-9, -3, 0, 4):
            s = digits / 8 * 2.0 ** e
            v = (borders * s).to(dtype)
            inf = torch.full_like(v, torch.inf)
            for w in (v, torch.nextafter(v, inf), torch.nextafter(v, -inf)):
                rows.append(torch.cat([w, torch.tensor([6 * s, -6 * s], device="cuda").to(dtype)]))
    x = torch.stack(rows)
    x = torch.cat([x, -x.flip(1)], 1)
    check_quantized(hs.fp4_quantize(x, fmt), x)
    check_quantized(hs.fp4_quantize(x, fmt, axis=0), x.t())
    if fmt == "nvfp4":
        for scale, k in ((1.0, 0), (0.3, -1), (2.0 ** -8, -8)):
            given = torch.tensor([scale], device="cuda")
            check_quantized(hs.fp4_quantize(x, fmt, tensor_scale=given), x, k)
            for m, y in zip(hs.fp4_quantize_both(x, fmt, tensor_scale=given), (x, x.t())):
                check_quantized(m, y, k)


@pytest.mark.parametrize("fmt", FORMATS)
def test_ends_of_the_range_zeros_infinities_and_nan(fmt):
    x = normal(64, 192, 3)
    cases = {"zeros": torch.zeros_like(x), "minus zeros": -torch.zeros_like(x), "tiny": x * 1e-42, "smallest": x * 2.0 ** -126,
             "huge": x.clamp(-1, 1) * 3.4e38, "a zero block": torch.cat([x[:, :64] * 0, x[:, 64:]], 1), "wide": x * 10.0 ** torch.linspace(-40, 38, 192, device="cuda").clamp(-37, 36)}
    bad = x.clone()
    bad[3, 5], bad[7, 100], bad[9, 191] = torch.inf, -torch.inf, torch.nan
    cases["infinities and NaN"] = bad
    cases["all NaN"] = torch.full_like(x, torch.nan)
    for name, y in cases.items():
        for m, z in [(hs.fp4_quantize(y, fmt), y), (hs.fp4_quantize(y, fmt, axis=0), y.t()), *zip(hs.fp4_quantize_both(y, fmt), (y, y.t()))]:
            check_quantized(m, z)
            want = ref.matrix_values(m).float()
            assert torch.equal(m.dequantize().nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0)), name


def test_a_given_tensor_scale_that_is_too_small_saturates():
    x = normal(40, 100, 8, spread=1e30)
    given = torch.tensor([1e-30], device="cuda")
    k = int(torch.frexp(given)[1])
    m = hs.fp4_quantize(x, tensor_scale=given)
    check_quantized(m, x, k)
    assert torch.isfinite(m.dequantize()).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS)
def test_dequantize_rounds_the_exact_value_once(dtype, fmt):
    for r, c in [(1, 1), (5, 33), (129, 250), (200, 1024)]:
        m = hs.fp4_quantize(normal(r, c, r + c), fmt)
        want = ref.matrix_values(m)
        assert torch.equal(m.dequantize(dtype=dtype), want.to(dtype))
        room = torch.full((r, c + 9), -7.0, dtype=dtype, device="cuda")
        assert m.dequantize(room[:, 3:3 + c]) .data_ptr() == room[:, 3:].data_ptr()
        assert torch.equal(room[:, 3:3 + c], want.to(dtype)) and (room[:, :3] == -7).all() and (room[:, 3 + c:] == -7).all()


def outputs(rows, n, dtype):
    """Ways C may lie: new; row by row; inside a larger one, off any alignment; column by column."""
    yield None
    yield torch.full((rows, n), torch.nan, dtype=dtype, device="cuda")
    yield torch.full((rows + 2, n + 5), torch.nan, dtype=dtype, device="cuda")[1:-1, 3:3 + n]
    yield torch.full((n, rows), torch.nan, dtype=dtype, device="cuda").t()
    yield torch.full((n + 1, rows + 7), torch.nan, dtype=dtype, device="cuda")[1:, 5:5 + rows].t()


PRODUCTS = [(1, 1, 1), (1, 1, 16), (128, 16, 256), (130, 17, 300), (5, 300, 64), (257, 33, 513), (300, 64, 96), (513, 65, 1000), (384, 129, 2080), (128, 256, 4096),
            (1000, 257, 777), (16, 2000, 512), (700, 700, 31)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_of_two_matrices(m, n, k, fmt):
    A, B = hs.fp4_quantize(normal(m, k, 1), fmt), hs.fp4_quantize(normal(n, k, 2, spread=1e-3), fmt)
    a, b = ref.matrix_values(A), ref.matrix_values(B)
    for dtype in (F32, F16, BF16):
        for out in outputs(m, n, dtype):
            got = A.matmul(B, out, dtype=dtype)
            assert got is out or out is None
            ref.check_product(got, a, b.t(), 64)


DENSE = [(1, 1, 1), (1, 1, 16), (128, 8, 128), (130, 5, 300), (257, 1, 1000), (640, 16, 257), (300, 9, 4096), (4000, 8, 130), (129, 24, 2080), (500, 33, 512), (300, 64, 100), (384, 192, 1024),
         (1000, 257, 777), (200, 511, 64)]


@pytest.mark.parametrize("fmt,dtype", [("nvfp4", F16), ("nvfp4", BF16), ("mxfp4", BF16)], ids=str)
@pytest.mark.parametrize("m,n,k", DENSE)
def test_product_with_a_dense_matrix(m, n, k, fmt, dtype):
    A = hs.fp4_quantize(normal(m, k, 1, spread=0.02), fmt)
    a = ref.matrix_values(A)
    x = normal(k, n, 2, dtype)
    wide = normal(k + 1, n + 11, 3, dtype)
    for B in (x, x.t().contiguous().t(), wide[1:, 3:3 + n], wide.t().contiguous()[4:4 + n, 1:].t()):
        for out_type, out in [(F32, None), (dtype, None)] + [(dtype, o) for o in outputs(m, n, dtype)]:
            got = A.matmul(B, out, dtype=out_type)
            ref.check_product(got, a, B.double(), 16)
