"""Products of matrices of 4-bit integers on the GPU against 64-bit products of what they stand for."""
import pytest
import torch

import hopper_spmm_b200 as hs
import int4_ref as ref
from hopper_spmm_b200 import _capi as capi

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
IDS = {F32: "f32", F16: "f16", BF16: "bf16"}.get


def normal(r, c, seed, dtype=F32, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(r, c, generator=g, device="cuda") * spread
    x[:, ::37] *= 20
    return x.to(dtype)


def span(m, x_group=None):
    return min(128, m.group or 128, x_group or 128)


def outputs(rows, n, dtype):
    """Ways a result of rows x n may lie: new; row by row; inside a larger one, off any alignment; column by column."""
    yield None
    yield torch.full((rows, n), torch.nan, dtype=dtype, device="cuda")
    yield torch.full((rows + 2, n + 5), torch.nan, dtype=dtype, device="cuda")[1:-1, 3:3 + n]
    yield torch.full((n + 1, rows + 7), torch.nan, dtype=dtype, device="cuda")[1:, 5:5 + rows].t()


# rows, columns, n: less than a tile, ends inside tiles, steps, groups and 16 bytes; several rounds of a block (4,800 tiles and more); columns that do not fit as a whole
SIZES = [(1, 1, 1), (1, 31, 2), (15, 33, 8), (17, 100, 3), (130, 250, 9), (64, 2080, 16), (500, 777, 17), (333, 1500, 33), (2368, 512, 5), (48 * 148 * 16 + 5, 64, 4), (100, 9000, 8),
         (40, 30001, 7), (70, 4096, 40)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("group", [32, 64, 128, 256, None], ids=str)
@pytest.mark.parametrize("rows,cols,n", SIZES)
def test_product(rows, cols, n, group, dtype):
    m = ref.matrix(rows, cols, group, rows + cols, BF16 if dtype == F16 else F16, zeros=(rows + n) % 2 == 0)
    a, x = ref.values_of(m), normal(n, cols, 3, dtype)
    for out in (F32, dtype):
        y = m.linear(x, dtype=out)
        assert y.dtype == out
        ref.check_product(y.t(), a, x.double().t(), span(m))
        ref.check_product(m.matmul(x.t(), dtype=out), a, x.double().t(), span(m))
    assert torch.equal(m.linear(x), m.linear(x, dtype=F32))


@pytest.mark.parametrize("x_group", [None, 32, 64, 128], ids=str)
@pytest.mark.parametrize("group", [32, 64, 128, None], ids=str)
@pytest.mark.parametrize("rows,cols,n", [(1, 1, 1), (17, 100, 3), (130, 250, 9), (64, 2080, 16), (333, 1500, 33), (2368, 512, 5), (40, 30001, 7)])
def test_product_with_8_bits(rows, cols, n, group, x_group):
    m = ref.matrix(rows, cols, group, rows + cols, zeros=n % 2 == 0)
    X = hs.rms_norm(normal(n, cols, 3, BF16), dtype=E4M3, group=x_group)
    x = X.values.double() * X.scales.double().repeat_interleave(x_group or cols, 1)[:, :cols]
    for out in (F32, F16, BF16):
        ref.check_product(m.linear(X, dtype=out).t(), ref.values_of(m), x.t(), span(m, x_group))
    assert torch.equal(m.matmul(X), m.linear(X).t())
    # rows that lie apart, off any alignment
    wide = torch.zeros(n, cols + 9, device="cuda").to(E4M3)
    wide[:, 3:3 + cols] = X.values
    assert torch.equal(m.linear(hs.Fp8Matrix(wide[:, 3:3 + cols], X.scales, x_group)), m.linear(X))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("rows,cols,n", [(130, 250, 9), (64, 2080, 16), (2368, 512, 1), (300, 1000, 33)])
def test_strides_offsets_and_results(rows, cols, n, dtype):
    m = ref.matrix(rows, cols, 64, 1)
    a = ref.values_of(m)
    wide = normal(n + 3, cols + 11, 3, dtype)
    for x in (wide[1:1 + n, 8:8 + cols], wide[1:1 + n, 3:3 + cols], wide.t().contiguous()[3:3 + cols, 2:2 + n].t(), wide[:n, :cols].contiguous()):
        want = x.double().t()
        ref.check_product(m.linear(x).t(), a, want, 64)
        for out in outputs(n, rows, dtype):
            y = m.linear(x, out, dtype=dtype)
            assert y is out or out is None
            ref.check_product(y.t(), a, want, 64)
        for out in outputs(rows, n, F32):
            y = m.matmul(x.t(), out)
            assert y is out or out is None
            ref.check_product(y, a, want, 64)
    # what lies around a result stays
    room = torch.full((n + 2, rows + 9), -7.0, dtype=dtype, device="cuda")
    m.linear(wide[:n, :cols], room[1:-1, 4:4 + rows])
    room[1:-1, 4:4 + rows] = -7
    assert (room == -7).all()


def test_columns_that_come_piece_by_piece_in_every_round():
    # more tiles than a block has warps, and columns that do not fit as a whole
    m, x = ref.matrix(148 * 16 * 17 + 3, 4100, 64, 1), normal(33, 4100, 2, F16)
    ref.check_product(m.linear(x).t(), ref.values_of(m), x.double().t(), 64)


def test_infinities_and_nan():
    m = ref.matrix(200, 300, 64, 1, BF16)
    s = m.scales
    s[2, 17], s[0, 199], s[4, 3] = torch.nan, torch.inf, torch.inf
    a = ref.values_of(m)
    x = normal(9, 300, 2, BF16)
    want = a @ x.double().t()
    got = m.linear(x).t()
    # a scale multiplies the sum over its group: an infinite one makes infinities of what, value by value, were infinities of either sign (NaN)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)) and torch.isnan(got[17]).all()
    fine = torch.isfinite(want).all(1)
    assert fine.sum() == 197
    ref.check_product(got[fine], a[fine], x.double().t(), 64)
    s.nan_to_num_(nan=1.0, posinf=1.0)
    # an infinity or a NaN in one column is that column's alone
    x[3, 77], x[5, 299] = torch.inf, torch.nan
    got = m.linear(x).t()
    good = [0, 1, 2, 4, 6, 7, 8]
    ref.check_product(got[:, good], ref.values_of(m), x.double().t()[:, good], 64)
    assert not torch.isfinite(got[:, 3]).any() and torch.isnan(got[:, 5]).all()
    # zero columns and zero rows
    x[:] = 0
    assert not m.linear(x).any()


def test_zeros_above_15_count_by_their_low_bits():
    m = ref.matrix(50, 200, 32, 1)
    x = normal(4, 200, 2, F16)
    want = m.linear(x)
    other = hs.Int4Matrix(50, 200, 32, values=m.values, scales=m.scales, zeros=m.zeros + 48)
    assert torch.equal(other.linear(x), want)


def test_sums_over_long_rows_are_as_exact_as_over_short_ones():
    # all of one sign: an addition that cut off would show
    for cols, group in ((65536, 128), (65536, None)):
        v = torch.full((64, cols // 2), 0xFF, dtype=torch.uint8, device="cuda")
        groups = cols // group if group else 1
        m = hs.Int4Matrix(64, cols, group, values=v, scales=torch.full((groups, 64), 0.0137, dtype=F16, device="cuda"))
        x = (torch.rand(3, cols, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") + 0.5).half()
        want = ref.values_of(m) @ x.double().t()
        # 8 additions of the MMA in 2^-22 at most, and each warp's 512 / 28 roundings in fp32
        assert (m.linear(x).t().double() / want - 1).abs().max() < 8 * 2.0 ** -22 + (512 / 28 + 1 + 28) * 2.0 ** -24


def test_offsets_that_pass_32_bits():
    rows, cols = 1_100_000, 8192
    v = torch.zeros(rows, cols // 2, dtype=torch.uint8, device="cuda")
    s = torch.ones(64, rows, dtype=F16, device="cuda")
    z = torch.zeros(64, rows, dtype=torch.uint8, device="cuda")
    v[-37:] = torch.randint(0, 256, (37, cols // 2), device="cuda", dtype=torch.uint8)
    z[:, -37:] = torch.randint(0, 16, (64, 37), device="cuda", dtype=torch.uint8)
    m = hs.Int4Matrix(rows, cols, 128, values=v, scales=s, zeros=z)
    x = normal(2, cols, 1, F16)
    y = m.linear(x)
    assert not y[:, :-37].any()
    ref.check_product(y[:, -37:].t(), ref.values_of(m, slice(rows - 37, rows)), x.double().t(), 128)


def test_empty():
    x = torch.empty(0, 64, dtype=F16, device="cuda")
    m = ref.matrix(40, 64, 32, 1)
    assert m.linear(x).shape == (0, 40) and m.matmul(x.t()).shape == (40, 0)
    none = ref.matrix(0, 64, 32, 1)
    assert none.linear(normal(3, 64, 1, F16)).shape == (3, 0)
    for group in (32, None):
        flat = ref.matrix(40, 0, group, 1)
        assert torch.equal(flat.linear(torch.empty(3, 0, dtype=BF16, device="cuda"), dtype=BF16), torch.zeros(3, 40, dtype=BF16, device="cuda"))


def test_refusals_on_the_gpu():
    m = ref.matrix(40, 64, 32, 1)
    x = normal(8, 64, 1, F16)
    for bad in (x.float(), x[:, :63], x[None], normal(8, 128, 1, F16)[:, ::2], x.cpu(), x[:1].expand(8, 64), x.to(E4M3), None):
        with pytest.raises(ValueError, match="X must be"):
            m.linear(bad)
    with pytest.raises(ValueError, match="B must be"):
        m.matmul(x)
    X = hs.rms_norm(x, dtype=E4M3, group=32)
    with pytest.raises(ValueError, match="8-bit"):
        m.linear(hs.Fp8Matrix(X.values[:, :32], X.scales[:, :1].contiguous(), 32))
    with pytest.raises(ValueError, match="8-bit"):
        m.linear(hs.Fp8Matrix(X.values.t().contiguous().t(), X.scales, 32))
    for bad in (torch.empty(8, 39, device="cuda"), torch.empty(8, 40), torch.empty(8, 80, device="cuda")[:, ::2], torch.empty(8, 1, device="cuda").expand(8, 40)):
        with pytest.raises(ValueError, match="C has"):
            m.linear(x, bad)
    with pytest.raises(TypeError):
        m.linear(x, dtype=torch.float64)
    with pytest.raises(ValueError, match="no backward"):
        m.linear(x.clone().requires_grad_())
    with pytest.raises(capi.SpmmError) as e:
        hs.Int4Matrix(40, 64, 32, values=torch.zeros(40 * 32 + 8, dtype=torch.uint8, device="cuda")[8:].view(40, 32), scales=m.scales, zeros=m.zeros).linear(x)
    assert e.value.status == capi.ERR_UNSUPPORTED
    v, s, z = ref.arrays(40, 64, 32, 1)
    with pytest.raises(ValueError, match="one device"):
        hs.Int4Matrix(40, 64, 32, values=v, scales=s.cpu(), zeros=z)


def test_scales_that_are_not_the_values_are_refused():
    m, X = ref.matrix(40, 64, 32, 1), hs.rms_norm(normal(8, 64, 1, F16), dtype=E4M3, group=32)
    scales = X.scales
    for bad in (scales[:, :1].contiguous(), scales[:7], scales.half(), scales.t().contiguous().t(), scales.cpu(), scales[0], None):
        X.scales = bad
        with pytest.raises(ValueError, match="scales|X must"):
            m.linear(X)
    X.scales, X.group = scales, None
    with pytest.raises(ValueError, match="scales"):
        m.linear(X)
    X.group, X.scales = 32, scales.clone().requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        m.linear(X)


@pytest.mark.parametrize("which", range(3))
def test_kept_tensors_that_have_become_others_are_refused(which):
    kept = ref.arrays(40, 64, 32, 1)
    m, x = hs.Int4Matrix(40, 64, 32, values=kept[0], scales=kept[1], zeros=kept[2]), normal(8, 64, 1, F16)
    want, t = m.linear(x), kept[which]
    old = t.data
    for new in (old.clone(), old.float(), old.t(), old[:1], old.cpu()):
        t.data = new
        with pytest.raises(ValueError, match="anew"):
            m.linear(x)
    t.data = old
    assert torch.equal(m.linear(x), want)
    t.mul_(1)  # (its values may change: they are read by every call)
    assert torch.equal(m.linear(x), want)
    t.resize_(4000, 1000)
    with pytest.raises(ValueError, match="anew"):
        m.linear(x)


def test_kept_scales_that_come_to_want_a_gradient_are_refused():
    kept = ref.arrays(40, 64, 32, 1)
    m, x = hs.Int4Matrix(40, 64, 32, values=kept[0], scales=kept[1], zeros=kept[2]), normal(8, 64, 1, F16)
    want = m.linear(x)
    kept[1].requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        m.linear(x)
    with torch.no_grad():
        assert torch.equal(m.linear(x), want)


def test_the_same_call_gives_the_same_bits_on_every_stream_and_in_graphs():
    m, x = ref.matrix(4000, 2048, 64, 1), normal(9, 2048, 2, BF16)
    X = hs.rms_norm(x, dtype=E4M3, group=64)
    want = (m.linear(x), m.linear(X), m.matmul(x[:1].t()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [(m.linear(x, stream=s), m.linear(X, stream=s), m.matmul(x[:1].t(), stream=s)) for s in streams * 3]
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            X = hs.rms_norm(x, dtype=E4M3, group=64)
            out = (m.linear(x), m.linear(X), m.matmul(x[:1].t()))
        graphs.append((g, out))
    for seed in (5, 6):
        x.copy_(normal(9, 2048, seed, BF16))
        X = hs.rms_norm(x, dtype=E4M3, group=64)
        want = (m.linear(x), m.linear(X), m.matmul(x[:1].t()))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_the_matrix_is_that_of_its_arrays():
    # arrays that are written after the matrix was made count as they are at the call; nothing is kept of them
    m, x = ref.matrix(300, 500, 32, 1), normal(3, 500, 2, F16)
    m.linear(x)
    v, s, z = ref.arrays(300, 500, 32, 9)
    m.values.copy_(v)
    m.scales.copy_(s)
    m.zeros.copy_(z)
    ref.check_product(m.linear(x).t(), ref.values_of(m), x.double().t(), 32)
    assert m.nbytes == v.numel() + 2 * s.numel() + z.numel() and m.device == v.device


# columns whose scales as a whole leave no room for a step of them (a column of 53,248 with scales of 32 has 6.6 KB of them); more tiles than a block has warps, with columns and scales that
# come piece by piece in every round
@pytest.mark.parametrize("rows,cols,n,group,x_group", [(40, 53_248, 33, 64, 32), (50, 53_248, 40, 128, 32), (33, 53_250, 80, 32, 32), (40, 65_536, 24, 128, 32), (20, 200_001, 8, None, 32),
                                                       (20, 131_072, 16, 64, 32), (40, 100_000, 40, 128, 64), (40, 100_100, 40, 128, None), (148 * 16 * 17 + 3, 4100, 33, 64, 32)])
def test_long_columns_in_8_bits(rows, cols, n, group, x_group):
    m = ref.matrix(rows, cols, group, rows + n)
    X = hs.rms_norm(normal(n, cols, 3, BF16), dtype=E4M3, group=x_group)
    x = X.values.double() * X.scales.double().repeat_interleave(x_group or cols, 1)[:, :cols]
    y = m.linear(X)
    ref.check_product(y.t(), ref.values_of(m), x.t(), span(m, x_group))
    # one column at a time has all its scales beside it
    for j in (0, n - 1):
        one = hs.Fp8Matrix(X.values[j:j + 1], X.scales[j:j + 1], x_group)
        ref.check_product(m.linear(one).t(), ref.values_of(m), x[j:j + 1].t(), span(m, x_group))


# ---------------------------------------------------------------- what autograd is told

def test_tangents_are_refused():
    from torch.autograd import forward_ad
    m, x = ref.matrix(40, 64, 32, 1), normal(8, 64, 1, F16)
    X = hs.rms_norm(x, dtype=E4M3, group=32)
    v, s, z = ref.arrays(40, 64, 32, 1)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        of_dual = hs.Fp8Matrix(X.values, X.scales, 32)
        of_dual.scales = dual(X.scales)
        for call in (lambda: m.linear(dual(x)), lambda: m.matmul(dual(x.t())), lambda: m.linear(of_dual), lambda: m.linear(x, dual(torch.empty(8, 40, device="cuda"))),
                     lambda: hs.Int4Matrix(40, 64, 32, values=v, scales=dual(s), zeros=z)):
            with pytest.raises(ValueError, match="no backward"):
                call()


def test_autograd_is_told_of_results_that_are_written_in_place():
    m, x = ref.matrix(40, 64, 32, 1), normal(8, 64, 1, F16)
    for call, shape in ((m.linear, (8, 40)), (lambda x, y: m.matmul(x.t(), y), (40, 8))):
        y = torch.zeros(shape, device="cuda")
        loss = (torch.ones(shape, device="cuda", requires_grad=True) * y).sum()
        assert call(x, y) is y
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        before = x._version, y._version
        call(x, y)
        assert (x._version, y._version) == (before[0], before[1] + 1)
