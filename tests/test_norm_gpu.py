"""The RMS norm on the GPU against its formula in 64 bits."""
import pytest
import torch

import hopper_spmm_b200 as hs

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
IDS = {F32: "f32", F16: "f16", BF16: "bf16", E4M3: "e4m3", None: "none"}.get
# h is one rounding off.  The sum of squares, all positive, is off by the depth of its additions: up to 40 for a thread (8 values times 4, or times 5 of a
# row of 40,000), 10 in the tree; its root by half of that; then the mean's division, eps, the root, the reciprocal, two products: 25 + 1 + 6 < 40 halves of a step.
NEAR = 40 * 2.0 ** -24


def normal(r, c, seed, dtype=F32, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(r, c, generator=g, device="cuda") * spread
    x[:, ::37] *= 20
    return x.to(dtype)


def reference(x, w, eps, r=None):
    h = x.double() + (0 if r is None else r.double())
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + eps)
    return y if w is None else y * w.double()


def check_values(y, want):
    # half a step of the type, of numbers that are NEAR; below its normal numbers half of the smallest step
    t = torch.finfo(y.dtype)
    bound = want.abs() * (t.eps / 2 * (1 + NEAR) + NEAR) + t.tiny * t.eps / 2
    assert y.shape == want.shape and ((y.double() - want).abs() <= bound).all(), float(((y.double() - want).abs() - bound).max())


def check_eights(m, want):
    rows, cols = want.shape
    group = m.group or cols
    top = torch.nn.functional.pad(want.abs(), (0, -cols % group)).view(rows, -1, group).amax(2)
    scale = top / 448
    assert ((m.scales.double() - scale).abs() <= scale * (NEAR + 2.0 ** -24) + 2.0 ** -149).all()
    s = m.scales.double().repeat_interleave(group, 1)[:, :cols]
    v = m.values.double()
    assert torch.equal(v[s == 0], torch.zeros_like(v[s == 0]))
    q = torch.where(s > 0, want / torch.where(s > 0, s, 1.0), 0.0)
    # half the step of the binade that q lies in, and what y, the reciprocal and the product are off (at the top, what the scale is off)
    step = torch.exp2((torch.frexp(q.abs())[1] - 1).clamp(min=-6).double() - 3)
    assert (v.abs() <= 448).all()
    assert ((v - q).abs() <= step / 2 + q.abs() * (2 * NEAR + 3 * 2.0 ** -24)).all()


SHAPES = [(1, 1), (1, 4096), (3, 17), (5, 250), (130, 256), (2, 1023), (33, 1032), (700, 2049), (4, 8192), (600, 8192), (9, 5000), (2, 32768), (3, 40000), (1, 40003)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm(shape, dtype):
    x, w = normal(*shape, 1, dtype), normal(1, shape[1], 2, dtype, 0.3)[0]
    for r in (None, normal(*shape, 3, dtype, 2.0), normal(*shape, 3, F32, 2.0)):
        want = reference(x, w, 1e-6, r)
        for out in (dtype, F32):
            y = hs.rms_norm(x, w, residual=r, dtype=out)
            if r is not None:
                y, h = y
                assert torch.equal(h, (x.float() + r.float()).to(r.dtype))
            check_values(y, want)
        for group in (None, 32, 64, 128):
            y = hs.rms_norm(x, w, residual=r, dtype=E4M3, group=group)
            if r is not None:
                y, h = y
                assert torch.equal(h, (x.float() + r.float()).to(r.dtype))
            check_eights(y, want)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=IDS)
def test_without_a_weight_and_with_one_of_another_type(dtype):
    x = normal(40, 777, 1, dtype)
    check_values(hs.rms_norm(x), reference(x, None, 1e-6))
    for kind in (F32, F16, BF16):
        w = normal(1, 777, 2, kind)[0]
        check_values(hs.rms_norm(x, w, 1e-3, dtype=F32), reference(x, w, 1e-3))
        check_eights(hs.rms_norm(x, w, 1e-3, dtype=E4M3, group=64), reference(x, w, 1e-3))


@pytest.mark.parametrize("cols", [200, 2000, 33000])
def test_strides_offsets_and_results_in_place(cols):
    big, other = normal(30, cols + 50, 1, BF16), normal(61, cols + 9, 2, BF16)
    w = normal(1, cols + 3, 3, BF16)[0, 3:]
    for x, r in ((big[:, 8:8 + cols], other[:30, :cols]), (big[3:21, 1:1 + cols], other[::2, 7:7 + cols][:18]), (big[::3, 4:4 + cols], other[1:21:2, 2:2 + cols])):
        want = reference(x, w, 1e-6, r)
        h_want = (x.float() + r.float()).to(BF16)
        room = torch.full((x.shape[0] + 2, cols + 11), -7.0, dtype=BF16, device="cuda")
        for at in (0, 3, 8):
            room.fill_(-7)
            out = room[1:-1, at:at + cols]
            y, h = hs.rms_norm(x, w, residual=r, out=out)
            assert y is out and torch.equal(h, h_want)
            check_values(y, want)
            room[1:-1, at:at + cols] = -7
            assert (room == -7).all()  # nothing beside it was written
        # the sum in the residual's place, the result in X's
        x2, r2 = x.clone(), r.clone()
        y, h = hs.rms_norm(x2, w, residual=r2, sum_out=r2, out=x2)
        assert y is x2 and h is r2 and torch.equal(r2, h_want)
        check_values(x2, want)
        # the sum in X's place
        x2 = x.clone()
        y, h = hs.rms_norm(x2, w, residual=r, sum_out=x2)
        assert h is x2 and torch.equal(x2, h_want)
        check_values(y, want)
        # 8 bits into arrays that are there, off any alignment
        bytes_ = torch.zeros(x.shape[0], cols + 5, device="cuda").to(E4M3)
        m = hs.Fp8Matrix(bytes_[:, 3:3 + cols], torch.empty(x.shape[0], (cols + 31) // 32, device="cuda"), 32)
        got, _ = hs.rms_norm(x, w, residual=r, out=m)
        assert got is m
        check_eights(m, want)
        assert not bytes_[:, :3].float().any() and not bytes_[:, 3 + cols:].float().any()


@pytest.mark.parametrize("cols", [64, 5000, 40000])
def test_zeros_infinities_and_nan(cols):
    x = normal(8, cols, 1)
    x[1] = 0
    x[2, 5] = torch.nan
    x[3, cols - 1] = torch.inf
    x[4, :40] = 0
    w = torch.ones(cols, device="cuda")
    w[7] = 0
    y = hs.rms_norm(x, w)
    good = torch.tensor([0, 1, 4, 5, 6, 7], device="cuda")
    check_values(y[good], reference(x[good], w, 1e-6))
    assert torch.isnan(y[2]).all() and torch.isnan(y[3, cols - 1]) and not y[3, :cols - 1].any()  # as the formula: finite / infinity is 0
    assert torch.isnan(hs.rms_norm(x[1:2], w, 0.0)).all()  # 0 / 0
    for group in (None, 32, 128):
        m = hs.rms_norm(x, w, dtype=E4M3, group=group)
        check_eights(hs.Fp8Matrix(m.values[good], m.scales[good], group), reference(x[good], w, 1e-6))
        assert not m.scales[1].any()
        assert torch.isnan(m.scales[2]).all() and not m.values[2].float().any()
        assert torch.isnan(m.scales[3, -1]) and not m.values[3].float().any()
        assert group is None or cols <= group or not m.scales[3, 0]


@pytest.mark.parametrize("cols", [100, 5000, 40000])
@pytest.mark.parametrize("spread", [1e-44, 1e-30, 1e-17, 1e15, 1e19, 1e36])
def test_squares_beyond_the_range_of_32_bits(spread, cols):
    x = normal(6, cols, 1, F32, 1.0).clamp(-4, 4) * spread
    r = normal(6, cols, 2, F32, 1.0).clamp(-4, 4) * spread
    w = normal(1, cols, 3)[0]
    for eps in (0.0, 1e-6, 1e-38):
        h32 = (x + r).double()  # (one rounding of h, which near the smallest numbers is no longer relative)
        want = reference(h32, w, float(torch.tensor(eps, dtype=F32)))
        y, h = hs.rms_norm(x, w, eps, residual=r)
        assert torch.equal(h, x + r)
        if spread * 1e-6 > 2.0 ** -126 or eps == 0.0:
            check_values(y, want)
            check_eights(hs.rms_norm(x, w, eps, residual=r, dtype=E4M3, group=64)[0], want)
        assert torch.isfinite(y).all()


def test_many_rows_and_the_same_bits_again():
    x, w = normal(20000, 96, 1, F16), normal(1, 96, 2, F16)[0]
    m = hs.rms_norm(x, w, dtype=E4M3)
    check_eights(m, reference(x, w, 1e-6))
    for _ in range(3):
        again = hs.rms_norm(x, w, dtype=E4M3)
        assert torch.equal(again.values.view(torch.uint8), m.values.view(torch.uint8)) and torch.equal(again.scales, m.scales)


def test_rows_whose_offsets_pass_32_bits():
    # 2^31 elements and some before the last row
    x = torch.empty(70000, 32768, dtype=F16, device="cuda")
    x[-3:] = normal(3, 32768, 1, F16)
    x[:-3] = 0
    m = hs.rms_norm(x, dtype=E4M3)
    check_eights(hs.Fp8Matrix(m.values[-3:], m.scales[-3:]), reference(x[-3:], None, 1e-6))
    assert not m.scales[:-3].any()


def test_empty():
    for shape in ((0, 64), (5, 0), (0, 0)):
        x = torch.empty(shape, dtype=F16, device="cuda")
        y, h = hs.rms_norm(x, torch.empty(shape[1], device="cuda"), residual=x)
        assert y.shape == h.shape == x.shape
        m = hs.rms_norm(x, dtype=E4M3, group=32)
        assert m.values.shape == x.shape and m.scales.shape == (shape[0], (shape[1] + 31) // 32)


def test_refusals_on_the_gpu():
    x = normal(8, 64, 1)
    w = torch.ones(64, device="cuda")
    for bad in (x.double(), x[None], x[:, ::2], x.t(), x[:1].expand(8, 64), x.cpu(), x.to(E4M3), torch.randn(8, 64, dtype=torch.complex64, device="cuda").conj().imag):
        with pytest.raises((ValueError, TypeError)):
            hs.rms_norm(bad, dtype=F32)
    for bad in (w[:63], w.cpu(), w.double(), w[None], torch.ones(128, device="cuda")[::2]):
        with pytest.raises(ValueError, match="weight"):
            hs.rms_norm(x, bad)
    for bad in (x[:7], x.half(), x.cpu(), x.t().contiguous().t(), x[:1].expand(8, 64)):
        with pytest.raises(ValueError, match="residual"):
            hs.rms_norm(x, residual=bad)
        with pytest.raises(ValueError, match="sum_out"):
            hs.rms_norm(x, residual=x, sum_out=bad)
    with pytest.raises(ValueError, match="sum_out"):
        hs.rms_norm(x, sum_out=x)
    for bad in (x[:7], x.cpu(), x.t().contiguous().t()):
        with pytest.raises(ValueError, match="out has"):
            hs.rms_norm(x, out=bad)
    with pytest.raises(ValueError, match="eps"):
        hs.rms_norm(x, eps=-1e-6)
    with pytest.raises(ValueError, match="out has"):
        hs.rms_norm(x, out=hs.Fp8Matrix(x.to(E4M3)[:4], torch.empty(4, 1, device="cuda")))


def test_inputs_that_want_a_gradient():
    x, w = normal(4, 64, 1), torch.nn.Parameter(torch.ones(64, device="cuda"))
    with pytest.raises(ValueError, match="no backward"):
        hs.rms_norm(x, w)
    with pytest.raises(ValueError, match="no backward"):
        hs.rms_norm(x.clone().requires_grad_())
    with torch.no_grad():
        check_values(hs.rms_norm(x, w), reference(x, w, 1e-6))
    with torch.inference_mode():
        check_values(hs.rms_norm(x, w), reference(x, w, 1e-6))


def test_streams_and_graphs():
    x, w, r = normal(64, 4096, 1, BF16), normal(1, 4096, 2, BF16)[0], normal(64, 4096, 3, BF16)

    def step():
        y, h = hs.rms_norm(x, w, residual=r)
        return (y, h, *(lambda m: (m.values.view(torch.uint8), m.scales))(hs.rms_norm(h, w, dtype=E4M3, group=128)))

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams * 3:
        y, h = hs.rms_norm(x, w, residual=r, stream=s)
        m = hs.rms_norm(h, w, dtype=E4M3, group=128, stream=s)
        s.synchronize()
        for a, b in zip((y, h, m.values.view(torch.uint8), m.scales), want):
            assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for seed in (5, 6):
        x.copy_(normal(64, 4096, seed, BF16))
        want = step()
        for g, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b)


# ---------------------------------------------------------------- what autograd is told

def test_tangents_are_refused():
    from torch.autograd import forward_ad
    x, w, r = normal(4, 64, 1), torch.ones(64, device="cuda"), normal(4, 64, 2)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: hs.rms_norm(dual(x), w), lambda: hs.rms_norm(x, dual(w)), lambda: hs.rms_norm(x, w, residual=dual(r)), lambda: hs.rms_norm(x, w, out=dual(x.clone())),
                     lambda: hs.rms_norm(x, w, residual=r, sum_out=dual(r.clone()))):
            with pytest.raises(ValueError, match="no backward"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="no backward"):  # (it takes tangents along)
                call()
        check_values(hs.rms_norm(forward_ad.unpack_dual(dual(x)).primal, w), reference(x, w, 1e-6))
    check_values(hs.rms_norm(x, w), reference(x, w, 1e-6))


def saved_by(t):
    """A loss whose backward pass needs t."""
    return (torch.ones(t.shape, dtype=t.dtype, device=t.device, requires_grad=True) * t).sum()


def test_autograd_is_told_of_results_that_are_written_in_place():
    x, r, w = normal(4, 64, 1), normal(4, 64, 2), torch.ones(64, device="cuda")
    losses = saved_by(x), saved_by(r)
    hs.rms_norm(x, w, residual=r, sum_out=r, out=x)
    for loss in losses:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    m = hs.rms_norm(x, w, dtype=E4M3, group=32)
    before = m.values._version, m.scales._version, x._version
    loss = saved_by(m.scales)
    hs.rms_norm(x, w, out=m)
    assert (m.values._version, m.scales._version, x._version) == (before[0] + 1, before[1] + 1, before[2])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    # what is only read is as it was
    loss = saved_by(x)
    hs.rms_norm(x, w, residual=r)
    loss.backward()
    with torch.inference_mode():
        y = torch.empty_like(x)
        check_values(hs.rms_norm(x, w, out=y), reference(x, w, 1e-6))
    check_values(hs.rms_norm(x, w, out=y), reference(x, w, 1e-6))  # (its kind has no versions)


def test_rows_without_columns_have_scales_of_zero():
    x = torch.empty(5, 0, dtype=F16, device="cuda")
    m = hs.Fp8Matrix(x.to(E4M3), torch.full((5, 1), 7.0, device="cuda"))
    hs.rms_norm(x, out=m)
    assert not m.scales.any()
    assert not hs.rms_norm(x, dtype=E4M3).scales.any()


@pytest.mark.parametrize("cols", [100, 5000, 5002, 40000])
@pytest.mark.parametrize("spread,far", [(1e18, 1e25), (1e15, 1e35), (1e-13, 1e-30), (1e-12, 1e-28), (1e36, 1e36), (1e-30, 1e-25), (1e17, 1e-37), (1e-12, 1e36)])
def test_weights_as_far_from_one_as_the_values(spread, far, cols):
    # h w leaves fp32's range, y does not
    x = normal(6, cols, 1).clamp(-4, 4) * spread
    w = (normal(1, cols, 2)[0].clamp(-4, 4).abs() + 0.5) * far
    want = reference(x, w, 0.0)
    check_values(hs.rms_norm(x, w, 0.0), want)
    for group in (None, 32, 64, 128):
        check_eights(hs.rms_norm(x, w, 0.0, dtype=E4M3, group=group), want)
