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


# ---------------------------------------------------------------- masks of a kind: infinities, NaN, empty rows, padding

@pytest.mark.parametrize("fmt", FORMATS)
def test_nan_blocks_infinities_and_empty_rows(fmt):
    a, b = normal(300, 400, 1), normal(70, 400, 2)
    a[5, 17], a[299, 399], a[7] = torch.nan, torch.inf, 0.0
    b[3, 100], b[64] = -torch.inf, 0.0
    A, B = hs.fp4_quantize(a, fmt), hs.fp4_quantize(b, fmt)
    for m, n in ((A, B), (B, A), (A, hs.fp4_quantize(b[:9], fmt))):
        x, y = ref.matrix_values(m), ref.matrix_values(n)
        ref.check_product(m.matmul(n), x, y.t(), 64)
    for n in (1, 9, 70):
        dense = normal(400, n, 3, BF16)
        dense[10, 0] = torch.inf
        want = ref.matrix_values(A) @ dense.double()
        got = A.matmul(dense)
        # (an infinity times a code of 0 is NaN, as in any product)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
        clean = dense.clone()
        clean[10, 0] = 1.0
        ref.check_product(A.matmul(clean), ref.matrix_values(A), clean.double(), 16)


@pytest.mark.parametrize("fmt", FORMATS)
def test_what_lies_in_the_padding_of_scales_does_not_matter(fmt):
    # rows of scales past the last row, full of NaN
    x = normal(133, 200, 4)
    m = hs.fp4_quantize(x, fmt)
    rows = ref.scale_index(256, (m.scales.numel() // 512 // 2) * 4).cuda()[133:]
    m.scales[rows.reshape(-1)] = 255 if fmt == "mxfp4" else 127
    a = ref.matrix_values(m)
    for n in (3, 40, 150):
        other = hs.fp4_quantize(normal(n, 200, 5), fmt)
        ref.check_product(m.matmul(other), a, ref.matrix_values(other).t(), 64)
        ref.check_product(other.matmul(m), ref.matrix_values(other), a.t(), 64)
        dense = normal(200, n, 6, BF16)
        ref.check_product(m.matmul(dense), a, dense.double(), 16)
    assert torch.equal(m.dequantize(), a.float())


@pytest.mark.parametrize("n", [2, 20, 100])
def test_scales_over_the_whole_range(n):
    # mxfp4: every power of two that bf16 and fp32 have room for beside the sum; nvfp4: every e4m3 scale and a tensor scale of any number
    g = torch.Generator().manual_seed(n)
    for fmt in FORMATS:
        code = torch.randint(0, 16, (150, 1000), generator=g, dtype=torch.uint8)
        blocks = -(-1000 // ref.BLOCK[fmt])
        byte = torch.randint(0, 127, (150, blocks), generator=g, dtype=torch.uint8)
        if fmt == "mxfp4":  # rows of one size each, 2^-127 to 2^100
            byte = (torch.arange(150)[:, None] * 227 // 149 + torch.randint(0, 2, (150, blocks), generator=g)).to(torch.uint8)
        values, scales = ref.pack(code, byte, fmt)
        m = hs.Fp4Matrix(150, 1000, fmt, values=values.cuda(), scales=scales.cuda(), tensor_scale=torch.tensor([0.0371], device="cuda"))
        a = ref.matrix_values(m)
        dense = normal(1000, n, 9, BF16)
        got, want = m.matmul(dense), a @ dense.double()
        # (one rounding more: the tensor's scale is no power of two)
        bound = (a.abs() @ dense.double().abs()) * (80 * 2.0 ** -22 + 2.0 ** -23) + 2.0 ** -148
        assert ((got.double() - want).abs() <= bound).all()
        other = hs.fp4_quantize(normal(n, 1000, 8), fmt)
        got, b = m.matmul(other), ref.matrix_values(other)
        bound = (a.abs() @ b.abs().t()) * (80 * 2.0 ** -22 + 2.0 ** -23) + 2.0 ** -148
        assert ((got.double() - a @ b.t()).abs() <= bound).all()


# ---------------------------------------------------------------- streams, graphs, workspaces, repetition

def test_the_same_call_gives_the_same_bits():
    A, B, x = hs.fp4_quantize(normal(1500, 2048, 1)), hs.fp4_quantize(normal(700, 2048, 2)), normal(2048, 300, 3, F16)
    for f in (lambda: A.matmul(B), lambda: A.matmul(x), lambda: A.matmul(x[:, :7]), lambda: hs.fp4_quantize(x).values):
        first = f()
        for _ in range(3):
            assert torch.equal(f(), first)


@pytest.mark.parametrize("fmt", FORMATS)
def test_without_a_workspace(fmt):
    # 74 and some tiles: the last ones are cut along k where there is room for their sums
    A, x = hs.fp4_quantize(normal(300 * 64, 4096, 1), fmt), normal(4096, 256, 2, BF16)
    B = hs.fp4_quantize(x.t().contiguous(), fmt)
    want = A.matmul(x)
    m = capi.Fp4(A.rows, A.cols, capi.MXFP4 if fmt == "mxfp4" else capi.NVFP4, 0, A.values.data_ptr(), A.scales.data_ptr(), A.tensor_scale.data_ptr())
    b = capi.Fp4(B.rows, B.cols, m.format, 0, B.values.data_ptr(), B.scales.data_ptr(), B.tensor_scale.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    for bytes_ in (0, 64):
        ws = torch.empty(64, dtype=torch.uint8, device="cuda")
        got = torch.empty_like(want)
        assert capi.lib().b200spmm_fp4_dense_product(C.byref(m), x.data_ptr(), x.stride(0), 256, capi.T_BF16, 0, got.data_ptr(), 256, capi.T_F32, 0,
                                                     ws.data_ptr(), bytes_, stream) == capi.OK
        ref.check_product(got, ref.matrix_values(A), x.double(), 16)
        assert capi.lib().b200spmm_fp4_product(C.byref(m), C.byref(b), got.data_ptr(), 256, capi.T_F32, 0, ws.data_ptr(), bytes_, stream) == capi.OK
        ref.check_product(got, ref.matrix_values(A), ref.matrix_values(B).t(), 64)
        # a B that starts on any element goes in passes of 16 columns then
        odd = normal(4096, 41, 5, BF16)[:, 1:34]
        out = torch.empty(A.rows, 33, device="cuda")
        assert capi.lib().b200spmm_fp4_dense_product(C.byref(m), odd.data_ptr(), odd.stride(0), 33, capi.T_BF16, 0, out.data_ptr(), 33, capi.T_F32, 0,
                                                     ws.data_ptr(), bytes_, stream) == capi.OK
        ref.check_product(out, ref.matrix_values(A), odd.double(), 16)
    assert capi.lib().b200spmm_fp4_status(0, stream) == capi.OK


def test_empty_products_and_matrices():
    for fmt in FORMATS:
        none, some = hs.fp4_quantize(torch.empty(0, 40, device="cuda"), fmt), hs.fp4_quantize(normal(5, 40, 1), fmt)
        assert none.matmul(some).shape == (0, 5) and some.matmul(none).shape == (5, 0) and none.dequantize().shape == (0, 40)
        assert some.matmul(torch.empty(40, 0, dtype=BF16, device="cuda")).shape == (5, 0)
        flat = hs.fp4_quantize(torch.empty(5, 0, device="cuda"), fmt)
        assert float(flat.tensor_scale) == 1
        assert torch.equal(flat.matmul(flat), torch.zeros(5, 5, device="cuda"))
        assert torch.equal(flat.matmul(torch.empty(0, 3, dtype=BF16, device="cuda"), dtype=BF16), torch.zeros(5, 3, dtype=BF16, device="cuda"))
        both = hs.fp4_quantize_both(torch.empty(5, 0, device="cuda"), fmt)
        assert (both[1].rows, both[1].cols) == (0, 5)


def test_out_matrices_and_results_are_filled_in_place():
    m = hs.Fp4Matrix(100, 300)
    for seed in (1, 2):
        x = normal(100, 300, seed)
        assert hs.fp4_quantize(x, out=m) is m
        check_quantized(m, x)
        t = hs.Fp4Matrix(300, 100, device=x.device)
        check_quantized(hs.fp4_quantize(x, axis=0, out=t), x.t())
    with pytest.raises(ValueError, match="shape"):
        hs.fp4_quantize(normal(101, 300, 1), out=m)
    with pytest.raises(ValueError, match="mxfp4"):
        hs.fp4_quantize(normal(100, 300, 1), "mxfp4", out=m)


def test_refusals_on_the_gpu():
    x = normal(40, 64, 1)
    m = hs.fp4_quantize(x)
    for bad in (x.double(), x.int(), x[None], x[:, ::2], x.expand(40, 64)[:1].expand(40, 64), x.cpu()):
        with pytest.raises(ValueError, match="X must be"):
            hs.fp4_quantize(bad)
    for scale in (torch.ones(2, device="cuda"), torch.ones(1), torch.ones(1, dtype=F16, device="cuda"), 1.0):
        with pytest.raises(ValueError, match="tensor_scale"):
            hs.fp4_quantize(x, tensor_scale=scale)
    for bad in (x.t(), x.half(), normal(64, 3, 1), normal(64, 6, 1, F16)[:, ::2], normal(64, 3, 1, F16).cpu(), None):
        with pytest.raises(ValueError):
            m.matmul(bad)
    b = normal(64, 9, 1, F16)
    for bad in (torch.empty(40, 8, device="cuda"), torch.empty(40, 9), torch.empty(40, 9, dtype=F16, device="cuda"), torch.empty(40, 18, device="cuda")[:, ::2],
                torch.empty(40, 1, device="cuda").expand(40, 9)):
        with pytest.raises(ValueError, match="C has"):
            m.matmul(b, bad, dtype=F32)
    with pytest.raises(ValueError, match="number of columns"):
        m.matmul(hs.fp4_quantize(normal(3, 65, 1)))
    with pytest.raises(ValueError, match="bfloat16"):
        hs.fp4_quantize(x, "mxfp4").matmul(b)
    with pytest.raises(capi.SpmmError) as e:
        hs.Fp4Matrix(40, 64, values=torch.zeros(40 * 32 + 8, dtype=torch.uint8, device="cuda")[8:], scales=m.scales, tensor_scale=m.tensor_scale).dequantize()
    assert e.value.status == capi.ERR_UNSUPPORTED


def test_two_streams_at_once():
    W, x = hs.fp4_quantize(normal(4096, 2048, 1)), normal(2048, 600, 2, F16)
    X = hs.fp4_quantize(x.t().contiguous())
    want = [(W.matmul(x[:, :5]), W.matmul(x), W.matmul(X), hs.fp4_quantize(x).values)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for s in streams:
            got.append((W.matmul(x[:, :5], stream=s, sync=False), W.matmul(x, stream=s, sync=False), W.matmul(X, stream=s, sync=False),
                        hs.fp4_quantize(x, stream=s).values))
    for s in streams:
        W.sync(s)
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want[0]):
            assert torch.equal(a, b)


def test_captured_calls_replay_on_new_inputs():
    W = hs.fp4_quantize(normal(3000, 1024, 1))
    x = normal(200, 1024, 2, BF16)
    scale = torch.tensor([0.25], device="cuda")

    def step():
        X = hs.fp4_quantize(x)
        y = W.matmul(X, sync=False)
        z = W.matmul(x.t()[:, :6], sync=False)
        a, b = hs.fp4_quantize_both(x, tensor_scale=scale)
        return y, z, W.matmul(x.t(), dtype=BF16, sync=False), a.dequantize(), b.dequantize(dtype=F16)

    graphs = []
    for _ in range(2):  # two graphs, whose workspaces are their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for seed in (3, 4):
        x.copy_(normal(200, 1024, seed, BF16))
        want = step()
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


def test_the_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch, hopper_spmm_b200 as hs
x = torch.randn(300, 512, device="cuda").half()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    W = hs.fp4_quantize(x)
    y, z, v = W.matmul(W, sync=False), W.matmul(x.t()[:, :3], sync=False), W.matmul(x.t(), sync=False)
g.replay()
torch.cuda.synchronize()
V = hs.fp4_quantize(x)
assert torch.equal(y, V.matmul(V)) and torch.equal(z, V.matmul(x.t()[:, :3])) and torch.equal(v, V.matmul(x.t()))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_two_layers_in_4_bits(tokens, fmt):
    # up, down, with the activations brought to 4 bits between them: each step against the definition on the values it was given
    W1, W2 = normal(700, 260, 1, BF16, 0.05), normal(260, 700, 2, BF16, 0.05)
    x = normal(tokens, 260, 3, BF16)
    Q1, Q2 = hs.fp4_quantize(W1, fmt), hs.fp4_quantize(W2, fmt)
    X = hs.fp4_quantize(x, fmt)
    check_quantized(X, x)
    h = X.matmul(Q1, dtype=BF16)
    ref.check_product(h, ref.matrix_values(X), ref.matrix_values(Q1).t(), 64)
    h = torch.relu(h)
    H = hs.fp4_quantize(h, fmt)
    check_quantized(H, h)
    y = H.matmul(Q2)
    ref.check_product(y, ref.matrix_values(H), ref.matrix_values(Q2).t(), 64)
    # the second layer with 16-bit activations
    z = torch.empty(tokens, 260, dtype=BF16, device="cuda")
    Q2.matmul(h.t(), z.t())
    ref.check_product(z.t(), ref.matrix_values(Q2), h.t().double(), 16)


@pytest.mark.parametrize("fmt", FORMATS)
def test_gradients_of_a_linear_layer(fmt):
    n, k, m = 90, 150, 210
    x, w, dy = normal(n, k, 1), normal(m, k, 2, spread=0.1), normal(n, m, 3, spread=0.01)
    (X, Xt), (W, Wt), (dY, dYt) = (hs.fp4_quantize_both(t, fmt) for t in (x, w, dy))
    v = ref.matrix_values
    dx, dw = dY.matmul(Wt), dYt.matmul(Xt)
    ref.check_product(dx, v(dY), v(Wt).t(), 64)
    ref.check_product(dw, v(dYt), v(Xt).t(), 64)
    # against differences of the loss <dy, x wᵀ>, with the values that each product's operands stand for: linear in x and in w, so that a step
    # of any size gives the gradient along it
    g = torch.Generator(device="cuda").manual_seed(5)
    of_x = lambda t: (v(dY) * (t @ v(Wt))).sum()
    of_w = lambda t: (v(dYt).t() * (v(Xt).t() @ t.t())).sum()
    for loss, at, grad in ((of_x, x, dx), (of_w, w, dw)):
        step = torch.randn(at.shape, generator=g, device="cuda", dtype=torch.float64)
        difference = float(loss(at.double() + step) - loss(at.double()))
        got = float((grad.double() * step).sum())
        # fp32 sums of at most 210 products, each addition off by 2^-22 of the sum of magnitudes
        size = float(((v(dY).abs() @ v(Wt).abs().t() if grad is dx else v(dYt).abs() @ v(Xt).abs().t()) * step.abs()).sum())
        assert abs(got - difference) <= size * 16 * 2.0 ** -22 + 1e-9 * size


def test_offsets_past_32_bits():
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    rows, cols = 70100, 131072  # 4.6 GB of codes; C of it with 8 columns, x of 18 GB
    g = torch.Generator(device="cuda").manual_seed(1)
    values = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8, device="cuda")
    scales = torch.randint(40, 60, (-(-rows // 128) * (cols // 64) * 512,), generator=g, dtype=torch.uint8, device="cuda")
    m = hs.Fp4Matrix(rows, cols, values=values, scales=scales, tensor_scale=torch.ones(1, device="cuda"))
    last = torch.arange(rows - 40, rows)
    code = torch.stack([values[-40:] & 15, values[-40:] >> 4], 2).view(40, cols)
    n = cols // 16
    base = (last // 128) * (n // 4) * 512 + (last % 32) * 16 + (last // 32 % 4) * 4
    where = base[:, None] + (torch.arange(n) // 4 * 512 + torch.arange(n) % 4)[None, :]
    a = ref.values(code, scales[where.cuda()], 0, "nvfp4")
    for k in (3, 40):
        x = normal(cols, k, 2, F16)
        ref.check_product(m.matmul(x)[-40:], a, x.double(), 16)
    other = hs.fp4_quantize(normal(100, cols, 3))
    ref.check_product(m.matmul(other)[-40:], a, ref.matrix_values(other).t(), 64)
    ref.check_product(other.matmul(m)[:, -40:], ref.matrix_values(other), a.t(), 64)
    out = m.dequantize(dtype=F16)
    assert torch.equal(out[-40:], a.half())
    again = hs.fp4_quantize(out, tensor_scale=torch.ones(1, device="cuda"))
    code, byte, _ = ref.quantize(out[-40:], "nvfp4", 0)
    assert torch.equal(again.values[-40:], ref.pack(code, byte, "nvfp4")[0]) and torch.equal(again.scales[where.cuda()], byte)
    del again
    t = hs.fp4_quantize(out, axis=0, tensor_scale=torch.ones(1, device="cuda"))
    code, byte, _ = ref.quantize(out[:, -9:].t().contiguous(), "nvfp4", 0)
    assert torch.equal(t.values[-9:], ref.pack(code, byte, "nvfp4")[0])


@pytest.mark.parametrize("fmt", FORMATS)
def test_sums_of_fp32_results(fmt):
    # An MMA cuts its sum off to fp32, at most 2^-23 of it, and sums in fp32 are taken over from the tensor core after at most 32 of them (512
    # values of k; the product of two 4-bit matrices and one of few columns: their MMAs cover 64 and 16 and are followed below).  Over a run of
    # random values the sum grows with the root, the mean of which is 2/3 of its last value: 32 * 2/3 * 2^-23, and the errors of different
    # runs, of either sign, add like the runs themselves.  16 rounded additions of runs: at most 16 * 2^-24 more.
    k = 8192
    w = normal(700, k, 1, spread=k ** -0.5)
    W = hs.fp4_quantize(w, fmt)
    a = ref.matrix_values(W)
    for n in (40, 100, 300):
        for dtype in (F16, BF16) if fmt == "nvfp4" else (BF16,):
            x = normal(k, n, 2, dtype)
            want = a @ x.double()
            error = float((W.matmul(x, dtype=F32).double() - want).norm() / want.norm())
            assert error <= (32 * 2 / 3 + 8) * 2.0 ** -23, (n, dtype, error)


@pytest.mark.parametrize("fmt", FORMATS)
def test_operands_larger_than_the_cache(fmt):
    # What is read from memory arrives in another order than it was asked for; every run has the same sums.  (With the sides exchanged tiles
    # are others, k is cut elsewhere, and fp32 sums add up in another order: that result has its own bound.)
    rows, cols = 40100, 32768
    g = torch.Generator(device="cuda").manual_seed(1)
    values = torch.randint(0, 256, (rows, cols // 2), generator=g, dtype=torch.uint8, device="cuda")
    low, high, per = (40, 60, 64) if fmt == "nvfp4" else (118, 128, 128)
    scales = torch.randint(low, high, (-(-rows // 128) * (cols // per) * 512,), generator=g, dtype=torch.uint8, device="cuda")
    whole = {"tensor_scale": torch.ones(1, device="cuda")} if fmt == "nvfp4" else {"format": fmt}
    m = hs.Fp4Matrix(rows, cols, values=values, scales=scales, **whole)
    other = hs.fp4_quantize(normal(100, cols, 3), fmt)
    dense = F16 if fmt == "nvfp4" else BF16
    x = other.dequantize(dtype=dense).t()
    at = torch.arange(0, rows, 97, device="cuda")
    a = m.dequantize()[at].double()
    for n in (20, 100):
        small = other if n == 100 else hs.fp4_quantize(normal(n, cols, 4), fmt)
        got, other_way = m.matmul(small), small.matmul(m)
        ref.check_product(got[at], a, ref.matrix_values(small).t(), 64)
        ref.check_product(other_way[:, at], ref.matrix_values(small), a.t(), 64)
        for _ in range(6):
            assert torch.equal(m.matmul(small), got) and torch.equal(small.matmul(m), other_way)
    for n, dtype in ((3, dense), (40, dense), (100, dense), (100, F32)):
        got = m.matmul(x[:, :n], dtype=dtype)
        ref.check_product(got[at], a, x[:, :n].double(), 16)
        for _ in range(6):
            assert torch.equal(m.matmul(x[:, :n], dtype=dtype), got)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
def test_tensor_scales_at_the_ends_of_their_range(dtype):
    # the result is an ordinary number, the other operand makes up for the scale; 64 products of magnitudes that fp32 holds
    for whole, size in ((2.0 ** -126, 1e35), (2.0 ** 127, 1e-37), (1.5 * 2.0 ** -140, 1e35), (1.5 * 2.0 ** 125, 1e-37)):
        if dtype == F16:
            size = 100.0 if size > 1 else 1e-5
        W = hs.fp4_quantize(normal(200, 64, 1, spread=4), tensor_scale=torch.ones(1, device="cuda"))
        a = ref.matrix_values(W)
        W.tensor_scale.fill_(whole)
        for n in (1, 16, 40, 300):
            g = torch.Generator(device="cuda").manual_seed(n)
            x = (torch.randn(64, n, generator=g, device="cuda") * size).to(dtype)
            got, want, mag = W.matmul(x).double(), a @ x.double() * whole, a.abs() @ x.double().abs() * whole
            # sums of at most 16 additions and two roundings of the scales, in fp32, whose numbers end at 2^-149; where they end is infinity
            bound = mag * 18 * 2.0 ** -22 + 2.0 ** -148
            inf = want.abs() > 3.4e38
            assert torch.equal(got.isinf(), inf) and not got.isnan().any()
            assert bool(((got - want).abs() <= bound)[~inf].all()), (whole, n)


@pytest.mark.parametrize("n", [1, 3, 9, 16, 17])
def test_columns_that_start_on_any_element(n):
    # few and many of them: read one by one, or copied first
    for k in (1000, 2050, 17000):
        W = hs.fp4_quantize(normal(300, k, 1))
        a = ref.matrix_values(W)
        whole = normal(k + 1, 2 * n + 3, 2, BF16)
        for x in (whole[1:, 1:n + 1], whole[:k, 1::2][:, :n].contiguous(), whole[:k, 3:3 + n], whole.t().contiguous()[1:n + 1, 1:].t()):
            ref.check_product(W.matmul(x), a, x.double(), 16)
            ref.check_product(W.matmul(x, dtype=BF16), a, x.double(), 16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS)
@pytest.mark.parametrize("cols, first", [(700, 0), (702, 0), (704, 2), (704, 4), (708, 1), (701, 0)])
def test_rows_that_start_on_8_4_or_2_bytes(cols, first, dtype, fmt):
    x = normal(261, cols, 5, dtype)[:, first:]
    x[7, 70] = torch.inf
    check_quantized(hs.fp4_quantize(x, fmt), x)
    check_quantized(hs.fp4_quantize(x, fmt, axis=0), x.t())
    a, b = hs.fp4_quantize_both(x, fmt)
    check_quantized(a, x)
    check_quantized(b, x.t())
    one = x[3:4]
    check_quantized(hs.fp4_quantize(one, fmt), one)


# ---------------------------------------------------------------- waits that run out

@pytest.fixture
def starve():
    yield capi.lib().b200spmm_kat_fp4_starve
    assert capi.lib().b200spmm_kat_fp4_starve(0, 0) == capi.OK
    torch.cuda.synchronize()
    capi.lib().b200spmm_fp4_status(0, torch.cuda.current_stream().cuda_stream)  # (every stream that was launched to is told of every failure)


STARVED = [(300, 4096, 1, F16, F16), (300, 128, 16, BF16, F32), (40000, 512, 3, F16, F32), (300, 1000, 40, BF16, BF16), (700, 2048, 300, F16, F16), (700, 2048, 300, BF16, F32)]


@pytest.mark.parametrize("operand", [0, 1])
@pytest.mark.parametrize("m,k,n,dtype,out", STARVED, ids=str)
def test_a_starved_product_with_dense_columns_ends_and_says_so(m, k, n, dtype, out, operand, starve):
    # A failure made on the host: boxes of half the rows, so that no stage is ever complete.  Every role has to leave its waits, the barriers
    # between them included, and the next product is an ordinary one.
    W, x = hs.fp4_quantize(normal(m, k, 1)), normal(k, n, 2, dtype)
    for B in (x, x.t().contiguous().t()):
        assert starve(5_000_000, operand) == capi.OK
        W.matmul(B, dtype=out, sync=False)
        assert starve(0, 0) == capi.OK
        if operand == 1 and n <= 16:  # few columns have no box of B
            W.sync()
        else:
            with pytest.raises(capi.SpmmError) as e:
                W.sync()
            assert e.value.status == capi.ERR_DEVICE_TIMEOUT
        W.sync()  # said once
        ref.check_product(W.matmul(B, dtype=out), ref.matrix_values(W), B.double(), 16)


@pytest.mark.parametrize("operand", [0, 1])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,k,n", [(300, 4096, 8), (300, 1000, 50), (700, 2048, 300), (257, 100, 65)])
def test_a_starved_product_of_two_matrices_ends_and_says_so(m, k, n, fmt, operand, starve):
    A, B = hs.fp4_quantize(normal(m, k, 1), fmt), hs.fp4_quantize(normal(n, k, 2), fmt)
    assert starve(5_000_000, operand) == capi.OK
    A.matmul(B, sync=False)
    assert starve(0, 0) == capi.OK
    with pytest.raises(capi.SpmmError) as e:
        A.sync()
    assert e.value.status == capi.ERR_DEVICE_TIMEOUT
    A.sync()
    ref.check_product(A.matmul(B), ref.matrix_values(A), ref.matrix_values(B).t(), 64)


def starved_product(starve, W, x, stream, limit_ns=5_000_000, out=None):
    assert starve(limit_ns, 0) == capi.OK
    y = W.matmul(x, out, stream=stream, sync=False)
    assert starve(0, 0) == capi.OK
    return y


def status(stream):
    return capi.lib().b200spmm_fp4_status(0, stream.cuda_stream)


def test_asking_for_one_stream_does_not_hide_a_failure_from_others(starve):
    import threading
    W, x = hs.fp4_quantize(normal(300, 512, 1)), normal(512, 8, 2, F16)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    W.matmul(x)
    torch.cuda.synchronize()
    starved_product(starve, W, x, a)
    torch.cuda.synchronize()
    assert status(b) == capi.ERR_DEVICE_TIMEOUT  # somewhere on the device, and said once
    assert status(b) == capi.OK
    assert status(a) == capi.ERR_DEVICE_TIMEOUT  # ... and still to who launched it
    assert status(a) == capi.OK
    W.matmul(x, stream=torch.cuda.Stream())  # a stream of which the thread has known nothing until it was told
    # two threads on one stream: either is told
    ready, asked, told = threading.Barrier(2), threading.Event(), {}

    def other():
        W.matmul(x, stream=a, sync=False)
        ready.wait()
        asked.wait()
        told["other"] = [status(a), status(a)]
    t = threading.Thread(target=other)
    t.start()
    ready.wait()
    starved_product(starve, W, x, a)
    told["this"] = [status(a), status(a)]
    asked.set()
    t.join()
    assert told["this"] == told["other"] == [capi.ERR_DEVICE_TIMEOUT, capi.OK]
    # who comes later is not told what others have read
    t = threading.Thread(target=lambda: told.update(late=[status(a), status(b)]))
    t.start()
    t.join()
    assert told["late"] == [capi.OK, capi.OK]
    W.matmul(x, stream=a)


def test_every_replay_of_a_starved_product_is_reported(starve):
    W, x = hs.fp4_quantize(normal(300, 512, 1)), normal(512, 40, 2, F16)
    out = W.matmul(x)
    s, other, g = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        starved_product(starve, W, x, None, out=out)
    for on in (s, other, s):
        with torch.cuda.stream(on):
            g.replay()
        assert status(on) == capi.ERR_DEVICE_TIMEOUT
    assert status(s) == capi.OK and status(other) == capi.ERR_DEVICE_TIMEOUT  # (the third one, for who asks there)
    del g
    assert status(torch.cuda.current_stream()) == capi.ERR_DEVICE_TIMEOUT
    W.matmul(x)


def test_waiting_for_a_product_waits_for_its_stream_alone():
    W, x = hs.fp4_quantize(normal(300, 512, 1)), normal(512, 8, 2, F16)
    want = W.matmul(x)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert torch.cuda.current_stream() == torch.cuda.default_stream()
    torch.cuda._sleep(2_000_000_000)  # about a second
    with torch.cuda.stream(s):
        got = W.matmul(x)
    assert not torch.cuda.default_stream().query(), "waited for another stream"
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_waiting_while_another_thread_captures():
    import threading
    W, x = hs.fp4_quantize(normal(300, 512, 1)), normal(512, 8, 2, F16)
    want, room, mine = W.matmul(x), torch.empty(300, 8, device="cuda"), torch.empty(300, 8, device="cuda")
    side, g, went = torch.cuda.Stream(), torch.cuda.CUDAGraph(), {}
    torch.cuda.synchronize()

    def other():
        try:
            with torch.cuda.stream(side):
                W.matmul(x, mine)
            went["ok"] = True
        except Exception as e:  # noqa: BLE001
            went["error"] = e
    with torch.cuda.graph(g):
        W.matmul(x, room, sync=False)
        t = threading.Thread(target=other)
        t.start()
        t.join()
    assert went == {"ok": True}
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(room, want) and torch.equal(mine, want)


def test_waiting_for_a_stream_that_is_captured_is_refused():
    W, x = hs.fp4_quantize(normal(300, 512, 1)), normal(512, 8, 2, F16)
    want, out, g = W.matmul(x), torch.empty(300, 8, device="cuda"), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        with pytest.raises(capi.SpmmError) as e:
            W.matmul(x, out)
    assert e.value.status == capi.ERR_UNSUPPORTED
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# What an MMA drops of a sum is anywhere between nothing and 2^-23 of it, half of that on the average.  Over a run of MMAs of random values the sum
# grows with the root, and the mean of its size is 2/3 of its last: runs of r MMAs leave r/3 * 2^-23 of the run.  Runs, and what they leave, add
# like one another; their rounded additions, of either sign, leave less than one 2^-23 more.
def left_by_runs(mmas):
    return (mmas / 3 + 1) * 2.0 ** -23


@pytest.mark.parametrize("fmt,dtype", [("nvfp4", F16), ("nvfp4", BF16), ("mxfp4", BF16)], ids=str)
@pytest.mark.parametrize("rows", [700, 28672])
def test_sums_of_fp32_results_of_few_columns(rows, fmt, dtype):
    # whatever share of k a warp has (all rows are multiplied; some hundred are looked at): 512 values of k, 16 an MMA, a run
    k = 8192
    W = hs.fp4_quantize(normal(rows, k, 1, spread=k ** -0.5), fmt)
    at = torch.arange(0, rows, max(1, rows // 700), device="cuda")
    a = W.dequantize()[at].double()
    for n in (1, 8, 16):
        x = normal(k, n, 2, dtype)
        want = a @ x.double()
        error = float((W.matmul(x)[at].double() - want).norm() / want.norm())
        assert error <= left_by_runs(32), (n, error)


@pytest.mark.parametrize("fmt", FORMATS)
def test_sums_of_fp32_results_of_two_matrices(fmt):
    # all of k in one accumulator, 64 values of it an MMA
    k = 8192
    W = hs.fp4_quantize(normal(700, k, 1, spread=k ** -0.5), fmt)
    a = ref.matrix_values(W)
    for n in (8, 50, 300):
        X = hs.fp4_quantize(normal(n, k, 2), fmt)
        want = a @ ref.matrix_values(X).t()
        error = float((W.matmul(X).double() - want).norm() / want.norm())
        assert error <= left_by_runs(k // 64), (n, error)


@pytest.mark.parametrize("fmt,dtype", [("nvfp4", F16), ("mxfp4", BF16)], ids=str)
@pytest.mark.parametrize("rows", [28672, 31000, 32777, 34000, 66300, 128256])
def test_few_columns_of_matrices_of_many_rows(rows, fmt, dtype):
    # blocks with one to several rounds of tiles, of different sizes
    W = hs.fp4_quantize(normal(rows, 300, 1), fmt)
    a = ref.matrix_values(W)
    for n in (1, 7, 16):
        x = normal(300, n, 2, dtype)
        for out in (F32, dtype):
            ref.check_product(W.matmul(x, dtype=out), a, x.double(), 16)
            ref.check_product(W.matmul(x.t().contiguous().t(), dtype=out), a, x.double(), 16)


@pytest.mark.filterwarnings("ignore:ComplexHalf")
def test_a_tensor_with_a_pending_negation_is_refused():
    # the imaginary part of a conjugate: torch keeps the numbers as they were and a mark that they are to be negated
    z = torch.complex(normal(40, 1, 1), normal(40, 1, 2))
    x = z.conj().imag
    assert x.is_neg() and not x.resolve_neg().is_neg()
    for call in (lambda: hs.fp4_quantize(x), lambda: hs.fp4_quantize(x, axis=0), lambda: hs.fp4_quantize_both(x, "mxfp4")):
        with pytest.raises(ValueError, match="X must be"):
            call()
    check_quantized(hs.fp4_quantize(x.resolve_neg()), x.resolve_neg())
    W = hs.fp4_quantize(normal(1, 40, 3))
    y = torch.complex(normal(40, 1, 1).half(), normal(40, 1, 2).half()).conj().imag
    with pytest.raises(ValueError, match="B must be"):
        W.matmul(y)
    ref.check_product(W.matmul(y.resolve_neg()), ref.matrix_values(W), y.resolve_neg().double(), 16)
    c = torch.complex(normal(1, 1, 1), normal(1, 1, 2)).conj().imag
    with pytest.raises(ValueError, match="C has"):
        W.matmul(y.resolve_neg(), c, dtype=F32)
    with pytest.raises(ValueError, match="C has"):
        hs.fp4_quantize(normal(1, 1, 3)).dequantize(c)
