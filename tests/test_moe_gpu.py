"""The mixture-of-experts layer on the GPU against its formula in 64 bits."""
import pytest
import torch

import hopper_spmm_b200 as hs
import int4_ref as ref
from fp4_ref import EPS, TINY
from hopper_spmm_b200 import _capi as capi

pytestmark = pytest.mark.gpu

F32, F16, BF16, E4M3 = torch.float32, torch.float16, torch.bfloat16, torch.float8_e4m3fn
IDS = {F32: "f32", F16: "f16", BF16: "bf16"}.get


def rand(*shape, seed, dtype=F32, spread=1.0):
    return (torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * spread).to(dtype)


def tokens_of(n, hidden, seed, dtype):
    x = rand(n, hidden, seed=seed)
    x[:, ::37] *= 20
    return x.to(dtype)


class Case:
    """A layer, and its experts in 64 bits."""

    def __init__(self, experts, hidden, inner, top, dtype, group=0, seed=1, renormalize=True, router=True, zeros=True):
        self.E, self.H, self.I, self.top, self.dtype, self.group, self.renormalize = experts, hidden, inner, top, dtype, group, renormalize
        self.router = rand(experts, hidden, seed=seed, dtype=dtype, spread=hidden ** -0.5) if router else None
        if group is None or group:
            self.gate_up = ref.matrix(experts * 2 * inner, hidden, group, seed + 1, dtype, zeros, spread=0.4 * hidden ** -0.5)
            self.down = ref.matrix(experts * hidden, inner, group, seed + 2, dtype, zeros, spread=0.4 * inner ** -0.5)
        else:
            # rows that start on 16 bytes, with something between them
            def weights(r, c, s):
                return rand(experts, r, (c + 7) // 8 * 8 + 8, seed=s, dtype=dtype, spread=c ** -0.5)[:, :, :c]
            self.gate_up, self.down = weights(2 * inner, hidden, seed + 1), weights(hidden, inner, seed + 2)
        self.layer = hs.MoeLayer(self.router, self.gate_up, self.down, top_k=top, renormalize=renormalize, experts=experts)

    def expert(self, e):
        if self.group is None or self.group:
            return ref.values_of(self.gate_up, slice(e * 2 * self.I, (e + 1) * 2 * self.I)), ref.values_of(self.down, slice(e * self.H, (e + 1) * self.H))
        return self.gate_up[e].double(), self.down[e].double()

    def check(self, y, x, ids, shares):
        """y against the formula for this routing, within what its roundings can be.

        A sum of K products takes K / 16 additions of the MMA (16-bit experts) or span / 16 of them and one rounding of fp32 for each span (codes), and up to 24 that join parts:
        `off` of the sum of magnitudes.  An inner value is off by what its gate (SiLU's slope is at most 1.1) and up are, and 2^-20 of itself for exp, the division and the product.
        It is multiplied as two 16-bit numbers, of which 2^-16 is lost (bf16) or 2^-22 (fp16), or, by codes and for bf16, as one of fp16: 2^-11; fp16, scaled, loses
        2^-38 of the pair's largest besides (half of its smallest step, 2^-25, of 2^14 or more; and so, 2^-39, do bf16 columns that are brought to fp16).  Two take twice the additions."""
        x, want, bound = x.double(), torch.zeros(x.shape, dtype=torch.float64, device="cuda"), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        span = 0 if self.group == 0 else min(128, self.group or 128)

        def off(k, planes):
            if span:
                return planes * span / 16 * 2.0 ** -22 + (-(-k // span) + 24 + 2) * 2.0 ** -24
            return (planes * -(-k // 16) + 24) * 2.0 ** -22

        one = span and self.dtype == BF16
        lost = 2.0 ** -11 if one else 2.0 ** -16 if self.dtype == BF16 else 2.0 ** -22
        for e in range(self.E):
            t, j = torch.where(ids == e)
            if len(t) == 0:
                continue
            gate_up, down = self.expert(e)
            (g, u), (mg, mu) = (x[t] @ gate_up.t()).split(self.I, 1), (x[t].abs() @ gate_up.abs().t()).split(self.I, 1)
            dg, du = mg * off(self.H, 1), mu * off(self.H, 1)
            if one:  # (of the weights' sum of magnitudes)
                far = x[t].abs().amax(1, keepdim=True) * gate_up.abs().sum(1) * 2.0 ** -39
                dg, du = dg + far[:, :self.I], du + far[:, self.I:]
            silu = g * torch.sigmoid(g)
            h = silu * u
            dh = 1.1 * dg * (u.abs() + du) + silu.abs() * du + h.abs() * 2.0 ** -20
            dh = dh + h.abs() * lost + h.abs().amax(1, keepdim=True) * 2.0 ** -38
            out, mag = h @ down.t(), h.abs() @ down.abs().t()
            d = mag * off(self.I, 1 if one else 2) + dh @ down.abs().t()
            s = shares[t, j].double()[:, None]
            want.index_add_(0, t, s * out)
            bound.index_add_(0, t, s.abs() * (d + out.abs() * (self.top + 1) * 2.0 ** -24))
        bound = bound + (want.abs() + bound) * EPS[y.dtype] + TINY[y.dtype]
        err = (y.double() - want).abs()
        assert y.shape == want.shape and not torch.isnan(y).any()
        worst = float((err / bound).max())
        assert worst <= 1, f"{worst:.2f} times the bound"

    def check_routing(self, x, ids, shares):
        """Choices by logits that are off by at most 8 roundings of their sum of magnitudes; shares by that, exp, the sum and the division."""
        logits, mag = x.double() @ self.router.double().t(), x.double().abs() @ self.router.double().abs().t()
        near = mag.amax(1, keepdim=True) * 8 * 2.0 ** -24
        ids = ids.long()
        mine = logits.gather(1, ids)
        assert (mine[:, :-1] >= mine[:, 1:] - 2 * near).all()
        rest = logits.clone().scatter_(1, ids, -torch.inf)
        assert (ids.sort(1)[0].diff(dim=1) > 0).all() and (mine.amin(1) >= rest.amax(1) - 2 * near[:, 0]).all()
        want = torch.softmax(logits, 1).gather(1, ids)
        want = want / want.sum(1, keepdim=True) if self.renormalize else want
        assert ((shares.double() / want - 1).abs() <= 4 * near + 2.0 ** -20).all()


# experts, hidden, inner, chosen, tokens
SIZES = [(4, 64, 40, 2, 1), (8, 256, 128, 3, 5), (10, 1000, 333, 4, 17), (64, 512, 96, 8, 3), (5, 130, 1000, 5, 40), (3, 2049, 64, 1, 9), (1, 72, 8, 1, 2), (300, 96, 24, 2, 33), (16, 4100, 70, 2, 12), (4, 48, 2500, 4, 70), (100, 64, 16, 6, 4),
         (300, 64, 16, 3, 2)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("group", [0, 32, 64, 128, None], ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_layer(size, group, dtype):
    experts, hidden, inner, top, n = size
    c = Case(experts, hidden, inner, top, dtype, group, seed=sum(size), renormalize=n % 2 == 1, zeros=hidden % 2 == 0)
    x = tokens_of(n, hidden, 9, dtype)
    y, ids, shares = c.layer.forward(x, return_routing=True)
    assert y.dtype == dtype and ids.dtype == torch.int32 and shares.dtype == F32
    c.check_routing(x, ids, shares)
    c.check(y, x, ids, shares)
    assert torch.equal(c.layer.forward(x), y)
    assert torch.equal(c.layer.experts(x, ids, shares), y)
    assert torch.equal(c.layer.experts(x, ids.long(), shares), y)


@pytest.mark.parametrize("group", [0, 64], ids=str)
def test_given_routing_with_masked_places(group):
    c = Case(6, 200, 88, 4, BF16, group, router=False)
    x = tokens_of(23, 200, 2, BF16)
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(-3, 9, (23, 4), generator=g, device="cuda")
    ids[5] = -1
    ids[6] = torch.tensor([2**33, -2**40, 6, -1], device="cuda")  # none of them an expert's
    ids[7] = 3  # the same expert four times
    shares = torch.rand(23, 4, generator=g, device="cuda") - 0.3
    shares[5] = torch.nan  # of nobody
    shares[6, 0] = torch.inf
    y = c.layer.experts(x, ids, shares)
    assert not y[5].any() and not y[6].any()
    c.check(y, x, torch.where((ids >= 0) & (ids < 6), ids, -1), shares.nan_to_num(posinf=0))
    small = torch.where((ids >= 0) & (ids < 6), ids, -1).int()
    assert torch.equal(c.layer.experts(x, small, shares), y)
    # nobody at all
    assert not c.layer.experts(x, torch.full_like(small, -1), shares).any()
    # what the rows of masked tokens hold does not matter, not even to others
    x[5] = torch.nan
    x[6] = torch.inf
    assert torch.equal(c.layer.experts(x, ids, shares), y)


@pytest.mark.parametrize("group", [0, 32], ids=str)
def test_all_tokens_to_one_expert(group):
    c = Case(5, 300, 72, 2, F16, group)
    x = tokens_of(256, 300, 2, F16)
    ids = torch.full((256, 2), 4, device="cuda", dtype=torch.int32)
    ids[:, 1] = -1
    shares = torch.ones(256, 2, device="cuda")
    c.check(c.layer.experts(x, ids, shares), x, ids, shares)
    y, i, s = c.layer.forward(x, return_routing=True)
    c.check_routing(x, i, s)
    c.check(y, x, i, s)


def test_the_largest_routing():
    c = Case(1024, 16, 8, 32, BF16)
    x = tokens_of(256, 16, 2, BF16)
    y, i, s = c.layer.forward(x, return_routing=True)
    c.check_routing(x, i, s)
    c.check(y, x, i, s)


def test_of_equal_logits_the_first_is_chosen_and_nan_is_the_largest():
    c = Case(40, 64, 16, 4, BF16)
    c.router[:] = c.router[0]  # all equal
    c.router[7] *= 2  # (but one)
    c.router[33] = c.router[7]
    x = tokens_of(6, 64, 2, BF16)
    _, ids, shares = c.layer.forward(x, return_routing=True)
    l = x.double() @ c.router.double().t()
    for t in range(6):
        assert ids[t].tolist() == ([7, 33, 0, 1] if l[t, 7] > l[t, 0] else [0, 1, 2, 3])
    x[0] = 0  # +0 and -0 are one
    x[1] = -0.0
    assert c.layer.forward(x, return_routing=True)[1][:2].tolist() == [[0, 1, 2, 3]] * 2
    # a token with a NaN is NaN as a whole, and no other is
    y = c.layer.forward(x)
    x[3, 5] = torch.nan
    z, ids, shares = c.layer.forward(x, return_routing=True)
    assert torch.isnan(z[3]).all() and torch.isnan(shares[3]).all() and ids[3].tolist() == [0, 1, 2, 3]
    others = [0, 1, 2, 4, 5]
    assert torch.equal(z[others], y[others])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
def test_inner_values_beyond_the_range_of_fp16_and_far_below_it(dtype):
    for spread in (300.0, 1e-4):
        c = Case(4, 128, 64, 2, dtype)
        c.gate_up.mul_(spread)
        c.down.mul_(1e-4 if spread > 1 else 1.0)
        x = tokens_of(7, 128, 2, dtype)
        ids, shares = torch.tensor([[0, 3]] * 7, device="cuda"), torch.full((7, 2), 0.5, device="cuda")
        c.check(c.layer.experts(x, ids, shares), x, ids, shares)


def test_strides_and_results_in_place():
    c = Case(6, 200, 80, 2, F16, 32)
    wide = tokens_of(20, 230, 2, F16)
    for x in (wide[:, 3:203], wide[::2, 8:208], wide[:1, 1:201]):
        y, ids, shares = c.layer.forward(x, return_routing=True)
        c.check(y, x, ids, shares)
        room = torch.full((x.shape[0] + 2, 217), -7.0, dtype=F16, device="cuda")
        out = room[1:-1, 5:205]
        assert c.layer.forward(x, out) is out and torch.equal(out, y)
        out.fill_(-7)
        assert (room == -7).all()
    router = torch.zeros(6, 211, dtype=F16, device="cuda")
    router[:, 3:203] = c.router
    other = hs.MoeLayer(router[:, 3:203], c.gate_up, c.down, top_k=2)
    x = wide[:, 3:203]
    assert torch.equal(other.forward(x), c.layer.forward(x))


def test_empty():
    c = Case(6, 200, 80, 2, F16, 32)
    x = torch.empty(0, 200, dtype=F16, device="cuda")
    y, ids, shares = c.layer.forward(x, return_routing=True)
    assert y.shape == (0, 200) and ids.shape == shares.shape == (0, 2)
    assert c.layer.experts(x, ids, shares).shape == (0, 200)


def test_refusals_on_the_gpu():
    c = Case(6, 200, 80, 2, F16, 32)
    x = tokens_of(4, 200, 2, F16)
    ids, shares = torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.ones(4, 2, device="cuda")
    for bad in (x.float(), x.bfloat16(), x[:, :199], x[None], x.t().contiguous().t(), x.cpu(), x[:1].expand(4, 200), None):
        with pytest.raises(ValueError, match="X must"):
            c.layer.forward(bad)
    for bad in (ids.float(), ids[:3], ids[:, :1], ids.cpu(), ids.t().contiguous().t(), 3):
        with pytest.raises(ValueError, match="ids must"):
            c.layer.experts(x, bad, shares)
    for bad in (shares.half(), shares[:3], shares.cpu(), 3):
        with pytest.raises(ValueError, match="shares must"):
            c.layer.experts(x, ids, bad)
    with pytest.raises(ValueError, match="together"):
        c.layer.experts(x, ids, None)
    for bad in (torch.empty(4, 199, dtype=F16, device="cuda"), torch.empty(4, 200, device="cuda"), torch.empty(4, 400, dtype=F16, device="cuda")[:, ::2]):
        with pytest.raises(ValueError, match="out must"):
            c.layer.forward(x, bad)
    with pytest.raises(ValueError, match="256 tokens"):
        c.layer.forward(tokens_of(257, 200, 2, F16))
    with pytest.raises(ValueError, match="no router"):
        hs.MoeLayer(None, c.gate_up, c.down, top_k=2, experts=6).forward(x)
    with pytest.raises(ValueError, match="number of experts"):
        hs.MoeLayer(None, c.gate_up, c.down, top_k=2)
    with pytest.raises(ValueError, match="both"):
        hs.MoeLayer(c.router, c.gate_up, torch.zeros(6, 200, 80, dtype=F16, device="cuda"), top_k=2)
    with pytest.raises(ValueError, match="rows"):
        hs.MoeLayer(c.router[:5], c.gate_up, c.down, top_k=2)
    with pytest.raises(ValueError, match="no backward"):
        c.layer.forward(x.clone().requires_grad_())


@pytest.mark.parametrize("group", [0, 64], ids=str)
def test_kept_tensors_that_have_become_others_are_refused(group):
    c = Case(6, 128, 64, 2, F16, group)
    x = tokens_of(4, 128, 2, F16)
    want = c.layer.forward(x)
    for t in c.layer._tensors():
        old = t.data
        for new in (old.clone(), old.float(), old.cpu(), old[:, :1]):  # (the first row of one is all of it)
            t.data = new
            with pytest.raises(ValueError, match="anew"):
                c.layer.forward(x)
        t.data = old
        assert torch.equal(c.layer.forward(x), want)
    c.router.requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        c.layer.forward(x)
    with torch.no_grad():
        assert torch.equal(c.layer.forward(x), want)


@pytest.mark.parametrize("group", [0, 64], ids=str)
def test_the_same_bits_on_every_stream_and_in_graphs(group):
    c = Case(16, 512, 256, 3, BF16, group)
    x = tokens_of(9, 512, 2, BF16)
    want = c.layer.forward(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [c.layer.forward(x, stream=s) for s in streams * 4]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c.layer.forward(x, return_routing=True)
        graphs.append((g, out))
    for seed in (5, 6):
        x.copy_(tokens_of(9, 512, seed, BF16))
        want = c.layer.forward(x, return_routing=True)
        for g, _ in graphs * 2:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_a_workspace_of_any_content():
    import ctypes as C
    c = Case(8, 256, 96, 3, F16)
    x = tokens_of(6, 256, 2, F16)
    want = c.layer.forward(x)
    m = capi.Moe(experts=8, hidden=256, inner=96, top_k=3, renormalize=1, dtype=capi.T_F16, device=0, router=c.router.data_ptr(), ld_router=256, gate_up_16=c.gate_up.data_ptr(),
                 down_16=c.down.data_ptr(), ld_gate_up=c.gate_up.stride(1), ld_down=c.down.stride(1))
    size = C.c_uint64()
    assert capi.lib().b200spmm_moe_workspace(C.byref(m), 6, C.byref(size)) == capi.OK
    for fill in (0, 255, 127):
        ws = torch.full((size.value + 64,), fill, dtype=torch.uint8, device="cuda")
        y = torch.empty_like(x)
        for _ in range(2):  # and as the last call left it
            assert capi.lib().b200spmm_moe(C.byref(m), x.data_ptr(), 256, 6, y.data_ptr(), 256, None, None, ws.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream) == capi.OK
            assert torch.equal(y, want)
        assert (ws[size.value:] == fill).all()


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("n", [1, 6, 33])
def test_a_decoding_step(n, dtype):
    # norm to 8 bits, a product with 4-bit integers, the residual and the norm again, the experts: each against the definition on the values it was given
    H = 384
    x, h, w1, w2 = tokens_of(n, H, 1, dtype), tokens_of(n, H, 2, dtype), rand(H, seed=3, dtype=dtype, spread=0.2) + 1, rand(H, seed=4, dtype=dtype, spread=0.2) + 1
    W = ref.matrix(H, H, 128, 5, dtype, spread=0.4 * H ** -0.5)
    c = Case(8, H, 200, 2, dtype, 64)
    a, h1 = hs.rms_norm(x, w1, residual=h, dtype=E4M3, group=128)
    assert torch.equal(h1, (x.float() + h.float()).to(dtype))
    y = W.linear(a, dtype=dtype)
    av = a.values.double() * a.scales.double().repeat_interleave(128, 1)[:, :H]
    ref.check_product(y.t(), ref.values_of(W), av.t(), 128)
    b, h2 = hs.rms_norm(y, w2, residual=h1)
    want = h1.double() + y.double()
    want = want / want.square().mean(1, keepdim=True).add(1e-6).sqrt() * w2.double()
    assert ((b.double() - want).abs() <= want.abs() * (EPS[dtype] + 2.0 ** -18) + TINY[dtype]).all()
    z, ids, shares = c.layer.forward(b, return_routing=True)
    c.check_routing(b, ids, shares)
    c.check(z, b, ids, shares)
    # the same as one graph
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a2, k1 = hs.rms_norm(x, w1, residual=h, dtype=E4M3, group=128)
        b2, k2 = hs.rms_norm(W.linear(a2, dtype=dtype), w2, residual=k1)
        z2 = c.layer.forward(b2)
    for _ in range(3):
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(z2, z) and torch.equal(k2, h2)


def test_sizes_that_no_block_has_room_for():
    def weights(*shape):
        return torch.zeros(*shape, dtype=F16, device="cuda")
    for hidden, inner in ((120_000, 8), (16, 60_000)):
        layer = hs.MoeLayer(weights(2, hidden), weights(2, 2 * inner, hidden), weights(2, hidden, inner), top_k=1)
        with pytest.raises(capi.SpmmError) as e:
            layer.forward(weights(3, hidden))
        assert e.value.status == capi.ERR_UNSUPPORTED
    # the largest that is promised, with as many pairs as there may be
    layer = hs.MoeLayer(None, weights(1024, 16, 24_000), weights(1024, 24_000, 8), top_k=32)
    ids = torch.zeros(256, 32, dtype=torch.int32, device="cuda")
    assert not layer.experts(weights(256, 24_000), ids, torch.ones(256, 32, device="cuda")).any()
    layer = hs.MoeLayer(None, weights(2, 24_000, 16), weights(2, 16, 12_000), top_k=32)
    assert not layer.experts(weights(256, 16), ids, torch.ones(256, 32, device="cuda")).any()


def test_the_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch, hopper_spmm_b200 as hs
E4M3 = torch.float8_e4m3fn
g0 = torch.Generator(device="cuda").manual_seed(1)
def rand(*s): return torch.randn(*s, generator=g0, device="cuda").half() * 0.1
x, w = rand(5, 256), rand(256)
W = hs.Int4Matrix(256, 256, 64, values=torch.randint(0, 256, (256, 128), device="cuda", dtype=torch.uint8), scales=rand(4, 256).abs())
layer = hs.MoeLayer(rand(4, 256), rand(4, 128, 256), rand(4, 256, 64), top_k=2)
def step():
    a = hs.rms_norm(x, w, dtype=E4M3, group=64)
    y = W.linear(a, dtype=torch.float16)
    return y, layer.forward(hs.rms_norm(y, w))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, step()))
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ---------------------------------------------------------------- long rows

@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("which", ["gate_up", "down"])
def test_sums_of_16_bit_experts_over_long_rows_are_as_exact_as_over_short_ones(which, dtype):
    # Two experts that give the same number: one from thousands of products 1 - 2^-14 = (1 + 2^-7) (1 - 2^-7), one from two terms.  The sum of 64 of them is a multiple of 2^-8 below 64, all sums
    # of those are multiples of 2^-9 below 2^15: exact in fp32.  But a sum of the MMA that runs on through the row meets each product's 2^-14 with 28 digits.  A gate of 32 or more is its own SiLU;
    # inner values are the same for both, or exact in 8 digits: the difference is zero.
    # Two pairs have room in a block, so there are 256 runs, and 12 tiles in each: most warps have whole rows.
    hidden, inner = (24_000, 96) if which == "gate_up" else (192, 12_000)
    near = 1 + 2.0 ** -7
    gate_up, down = torch.zeros(2, 2 * inner, hidden, dtype=dtype, device="cuda"), torch.zeros(2, hidden, inner, dtype=dtype, device="cuda")
    gate_up[:, :inner, 0] = 32
    if which == "gate_up":
        x = torch.full((256, hidden), near, dtype=dtype, device="cuda")
        gate_up[0, inner] = 1 - 2.0 ** -7
        gate_up[1, inner, 1], gate_up[1, inner, 2] = 23808, 4.5  # 24,000 (1 - 2^-7)
        down[:, 0, 0] = 1
    else:
        x = torch.ones(256, hidden, dtype=dtype, device="cuda")
        gate_up[:, inner:, 0] = near
        down[0, 0] = 1 - 2.0 ** -7
        down[1, 0, 1], down[1, 0, 2] = 11904, 2.25
    layer = hs.MoeLayer(None, gate_up, down, top_k=2)
    ids, shares = torch.arange(2, device="cuda", dtype=torch.int32).repeat(256, 1), torch.zeros(256, 2, device="cuda")
    shares[:, 0] = 1 / 16
    total = (1 - 2.0 ** -14) * (24_000 * 32 * near if which == "gate_up" else 12_000 * 32) / 16
    for one in (shares, shares.roll(1, 1)):
        y = layer.experts(x, ids, one)
        # (h and its two parts are off by 2^-16 at most, where they do not cancel)
        assert (y[:, 0].double() - total).abs().max() <= total * (EPS[dtype] + 2.0 ** -16) and not y[:, 1:].any()
    shares[:, 1] = -1 / 16
    assert not layer.experts(x, ids, shares).any()


@pytest.mark.parametrize("group", [32, 64, 128], ids=str)
@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
def test_inner_values_beside_codes_have_22_digits(dtype, group):
    # Two experts that differ in up's scales by a 128th, one taken from the other: what is left shows roundings of inner values that a layer's own result would hide.
    H, I = 128, 24
    c = Case(2, H, I, 2, dtype, group)
    for m, rows in ((c.gate_up, 2 * I), (c.down, H)):
        m.values[rows:] = m.values[:rows]
        m.zeros[:, rows:] = m.zeros[:, :rows]
        m.scales[:, rows:] = m.scales[:, :rows]
    c.gate_up.scales[:, 3 * I:] *= 1 + 2.0 ** -7
    x = rand(20, H, seed=2, dtype=dtype)
    ids, shares = torch.arange(2, device="cuda").repeat(20, 1), torch.tensor([1.0, -1.0], device="cuda").repeat(20, 1)
    y = c.layer.experts(x, ids, shares).double()
    want = bound = 0
    for e in range(2):
        # as Case.check, with 2^-22 of an inner value and 2^-38 of a token's largest for its two parts; the gates are the same, and so is what they are off
        gate_up, down = c.expert(e)
        (g, u), (_, mu) = (x.double() @ gate_up.t()).split(I, 1), (x.double().abs() @ gate_up.abs().t()).split(I, 1)
        off = group / 16 * 2.0 ** -22 + (-(-H // group) + 24 + 2) * 2.0 ** -24
        silu = g * torch.sigmoid(g)
        h = silu * u
        dh = silu.abs() * (mu * off + x.double().abs().amax(1, keepdim=True) * gate_up.abs().sum(1)[I:] * 2.0 ** -39)
        dh = dh + h.abs() * (2.0 ** -22 + 2.0 ** -23) + h.abs().amax(1, keepdim=True) * 2.0 ** -38
        want = want + (1 - 2 * e) * (h @ down.t())
        bound = bound + dh @ down.abs().t() + h.abs() @ down.abs().t() * (2 * group / 16 * 2.0 ** -22 + 27 * 2.0 ** -24)
    gate_up, down = c.expert(0)
    # (the gates' own error, and the exponential's, are those of the difference)
    g, mg = x.double() @ gate_up[:I].t(), x.double().abs() @ gate_up[:I].abs().t()
    du = (x.double() @ (gate_up[I:] - c.expert(1)[0][I:]).t()).abs()
    bound = bound + (du * (1.1 * mg * 2.0 ** -18 + (g * torch.sigmoid(g)).abs() * 2.0 ** -20)) @ down.abs().t()
    bound = bound + (want.abs() + bound) * EPS[dtype] + TINY[dtype]
    worst = ((y - want).abs() / bound).max().item()
    assert worst <= 1, f"{worst:.2f} times the bound"


# ---------------------------------------------------------------- logits

@pytest.mark.parametrize("tokens", [1, 3, 9])
@pytest.mark.parametrize("experts", [40, 100, 200, 500])  # each way of choosing
@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
def test_experts_are_told_apart_by_small_terms_beside_large_ones_that_cancel(dtype, experts, tokens):
    # Products of 2^14 and -2^14 in every eight of the row, and 2^-12 times whole numbers beside them: exact in 64 bits in any order, while in fp32 neighbours of 2^14 are 2^-10 apart.
    H = 512
    rank = torch.randperm(experts, generator=torch.Generator(device="cuda").manual_seed(experts), device="cuda")
    router = torch.zeros(experts, H, dtype=dtype, device="cuda")
    router[:, 0::8], router[:, 7::8] = 1, -1
    router[:, 3] = (rank % 8).to(dtype) * 2.0 ** -6
    router[:, 460] = (rank // 8).to(dtype) * 2.0 ** -3  # (up to 63)
    x = torch.zeros(tokens, H, dtype=dtype, device="cuda")
    x[:, 0::8] = x[:, 7::8] = 2.0 ** 14
    x[:, 3] = x[:, 460] = 2.0 ** -6
    layer = hs.MoeLayer(router, torch.zeros(experts, 16, H, dtype=dtype, device="cuda"), torch.zeros(experts, H, 8, dtype=dtype, device="cuda"), top_k=20)
    _, ids, shares = layer.forward(x, return_routing=True)
    logits = x.double() @ router.double().t()
    want = rank.argsort(descending=True)[:20]
    assert torch.equal(logits[0], rank.double() * 2.0 ** -12) and (ids == want).all()
    want = torch.softmax(logits.gather(1, ids.long()), 1)
    # each exponential is off by the 2 units of its last place that expf may be, the sum by 5 roundings, the quotient by one; the difference of two logits is exact in fp32
    assert ((shares.double() / want - 1).abs() <= 2 * 2.0 ** -22 + 6 * 2.0 ** -24).all()


def test_logits_beyond_the_range_of_32_bits():
    # products of 2^140, which are no infinities in 64 bits, beside ones of 2^90, which there are within their 53 digits
    router, x = torch.zeros(6, 64, dtype=BF16, device="cuda"), torch.zeros(2, 64, dtype=BF16, device="cuda")
    router[:, 5] = router[:, 11] = 2.0 ** 70
    router[:, 7] = torch.tensor([3, 1, 4, 1, 5, 9], device="cuda") * 2.0 ** 45
    router[3, 11] = 2.0 ** 71
    x[:, 5], x[:, 11], x[:, 7] = 2.0 ** 70, -2.0 ** 70, 2.0 ** 45
    layer = hs.MoeLayer(router, torch.zeros(6, 16, 64, dtype=BF16, device="cuda"), torch.zeros(6, 64, 8, dtype=BF16, device="cuda"), top_k=6)
    _, ids, shares = layer.forward(x, return_routing=True)
    assert ids.tolist() == [[5, 4, 2, 0, 1, 3]] * 2  # (the last one's logit is -2^140)
    assert shares.tolist() == [[1, 0, 0, 0, 0, 0]] * 2


# ---------------------------------------------------------------- what autograd is told

@pytest.mark.parametrize("group", [0, 64], ids=str)
def test_tangents_are_refused(group):
    from torch.autograd import forward_ad
    c = Case(6, 128, 64, 2, F16, group)
    x, ids, shares = tokens_of(4, 128, 2, F16), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.ones(4, 2, device="cuda")
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: c.layer.forward(dual(x)), lambda: c.layer.experts(x, ids, dual(shares)), lambda: c.layer.forward(x, dual(x.clone())),
                     lambda: hs.MoeLayer(dual(c.router), c.gate_up, c.down, top_k=2)):
            with pytest.raises(ValueError, match="no backward"):
                call()
        if not group:
            with pytest.raises(ValueError, match="no backward"):
                hs.MoeLayer(c.router, c.gate_up, dual(c.down), top_k=2)


def test_autograd_is_told_of_results_that_are_written_in_place():
    c = Case(6, 128, 64, 2, F16)
    x = tokens_of(4, 128, 2, F16)
    _, ids, shares = c.layer.forward(x, return_routing=True)
    for call in (c.layer.forward, lambda x, y: c.layer.experts(x, ids, shares, y)):
        y = torch.zeros_like(x)
        loss = (torch.ones_like(x, requires_grad=True) * y).sum()
        assert call(x, y) is y
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        before = x._version, y._version, ids._version, shares._version
        call(x, y)
        assert (x._version, y._version, ids._version, shares._version) == (before[0], before[1] + 1, *before[2:])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("group", [32, 64, 128], ids=str)
@pytest.mark.parametrize("n", [1, 5])
def test_inner_values_beside_codes_that_no_block_has_room_for(n, group, dtype):
    # a column's two halves are 290 KB
    c = Case(3, 72, 72_000, 2, dtype, group, router=False)
    x = tokens_of(n, 72, 9, dtype)
    ids, shares = torch.tensor([[0, 2]] * n, device="cuda"), torch.tensor([[0.75, -0.5]] * n, device="cuda")
    c.check(c.layer.experts(x, ids, shares), x, ids, shares)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("group", [0, 64], ids=str)
@pytest.mark.parametrize("tokens", [1, 9, 14, 16, 17, 40])
def test_inner_values_of_a_run_in_pieces(tokens, group, dtype):
    # 16 columns of 6,000 have no room as a whole, 8 or 9 do; hidden sizes with one round of a block's tiles, and with several
    for hidden in (200, 148 * 16 * 21 + 5):
        c = Case(2, hidden, 6000, 1, dtype, group, router=False)
        x = tokens_of(tokens, hidden, 9, dtype)
        ids, shares = (torch.arange(tokens, device="cuda") % 10 == 9).long()[:, None], torch.rand(tokens, 1, device="cuda")
        c.check(c.layer.experts(x, ids, shares), x, ids, shares)


# ---------------------------------------------------------------- codes: columns and inner values as scaled fp16

@pytest.mark.parametrize("group", [32, 64, 128, None], ids=str)
@pytest.mark.parametrize("spread", [1e-18, 1e-15, 1e-8, 1e-5, 1e5, 1e12, 1e16])
def test_tokens_far_from_one_beside_codes(spread, group):
    c = Case(4, 200, 72, 2, BF16, group)
    x = (tokens_of(9, 200, 2, F32) * spread).to(BF16)
    ids, shares = torch.tensor([[0, 3]] * 9, device="cuda"), torch.full((9, 2), 0.5, device="cuda")
    c.check(c.layer.experts(x, ids, shares), x, ids, shares)
    # and beside others of another size
    x[::2] /= spread
    c.check(c.layer.experts(x, ids, shares), x, ids, shares)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("group", [32, 64, 128], ids=str)
def test_inner_values_beyond_the_range_of_fp16_and_far_below_it_beside_codes(group, dtype):
    for spread in (300.0, 2.0 ** -8):
        c = Case(4, 128, 64, 2, dtype, group)
        c.gate_up.scales.mul_(spread)
        c.down.scales.mul_(1e-4 if spread > 1 else 1.0)
        x = tokens_of(7, 128, 2, dtype)
        ids, shares = torch.tensor([[0, 3]] * 7, device="cuda"), torch.full((7, 2), 0.5, device="cuda")
        c.check(c.layer.experts(x, ids, shares), x, ids, shares)


@pytest.mark.parametrize("tokens", [3, 9])  # (all as columns before the routing, or those of runs)
def test_values_up_to_31_binades_below_a_token_s_largest_are_exact_beside_codes(tokens):
    # a value of 2^30 that meets nothing but codes of zero takes no digit from the others
    c = Case(3, 128, 40, 2, BF16, 64)
    v, z = c.gate_up.values, c.gate_up.zeros
    v[:, 5] = (v[:, 5] & 0xF0) | z[0]  # column 10
    x = rand(tokens, 128, seed=2, dtype=BF16)
    ids, shares = torch.tensor([[0, 2]] * tokens, device="cuda"), torch.full((tokens, 2), 0.5, device="cuda")
    x[:, 10] = 0
    x = torch.where(x.abs() < 2.0 ** -3, 0.25, x)
    x[:, 10] = 0
    want = c.layer.experts(x, ids, shares)
    c.check(want, x, ids, shares)
    x[:, 10] = 2.0 ** 28
    # the sums are of the same numbers in the same order, but for a power of two
    assert torch.equal(c.layer.experts(x, ids, shares), want)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("group", [0, 32, 64, 128], ids=str)
@pytest.mark.parametrize("tokens", [3, 9])
def test_infinities_and_nan_in_a_token_are_its_own(tokens, group, dtype):
    c = Case(5, 200, 72, 2, dtype, group)
    x = tokens_of(tokens, 200, 2, dtype)
    ids = torch.tensor([[0, 3]] * tokens, device="cuda")  # the same runs for all
    shares = torch.full((tokens, 2), 0.5, device="cuda")
    want = c.layer.experts(x, ids, shares)
    x[0, 77], x[2, 199] = torch.nan, -torch.inf
    y = c.layer.experts(x, ids, shares)
    assert torch.isnan(y[0]).all() and not torch.isfinite(y[2]).any()
    others = [i for i in range(tokens) if i not in (0, 2)]
    assert torch.equal(y[others], want[others])
    z = c.layer.forward(x)
    assert torch.isnan(z[0]).all() and not torch.isfinite(z[2]).any() and torch.isfinite(z[others]).all()


# ---------------------------------------------------------------- the largest sizes

@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("group", [0, 32, 64, 128], ids=str)
@pytest.mark.parametrize("size", [(4, 64, 12_000, 2, 20), (2, 24_000, 16, 2, 20), (3, 72, 36_000, 1, 5), (3, 72_000, 8, 1, 5), (8, 4096, 14_336, 2, 32)], ids=str)
def test_few_columns_have_room_in_a_block(size, group, dtype):
    experts, hidden, inner, top, n = size
    c = Case(experts, hidden, inner, top, dtype, group, seed=sum(size))
    x = tokens_of(n, hidden, 9, dtype)
    y, ids, shares = c.layer.forward(x, return_routing=True)
    c.check_routing(x, ids, shares)
    c.check(y, x, ids, shares)
    assert torch.equal(c.layer.experts(x, ids, shares), y)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=IDS)
@pytest.mark.parametrize("group", [0, 64], ids=str)
@pytest.mark.parametrize("hidden,inner", [(24_000, 24), (40, 12_000)])
def test_one_column_has_room_beside_the_largest_routing(hidden, inner, group, dtype):
    c = Case(5, hidden, inner, 32, dtype, group, router=False)
    x = tokens_of(256, hidden, 2, dtype)
    g = torch.Generator(device="cuda").manual_seed(3)
    ids, shares = torch.randint(-1, 5, (256, 32), generator=g, device="cuda"), torch.rand(256, 32, generator=g, device="cuda") - 0.3
    c.check(c.layer.experts(x, ids, shares), x, ids, shares)
