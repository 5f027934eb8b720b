"""What a decoding step does around weights in few bits, as measurable cases.

``op`` of a case:

* ``norm``  the residual's addition and the RMS norm: h = x + r, y = h / sqrt(mean(h²) + eps) * w, as 16 bits or as e4m3 with a
            scale, max |y| / 448, for each row (``group`` 0) or for ``group`` neighbours of a row
* ``int4``  Y = X Wᵀ for a few rows of X, with W in 4-bit integers: (code - zero) * scale, one scale and one zero (8 where none are
            given) for ``group`` neighbours of a row of W; X in 16 bits or in e4m3 with scales
* ``moe``   a whole mixture-of-experts layer for a few tokens: softmax of the router's logits, the ``top`` largest (of equal ones the first),
            their shares scaled to 1, y = sum of share * down(silu(gate x) * up x); experts in 16 bits or in 4-bit integers.
            ``routed``: experts and shares are given instead, some of them masked (expert -1)

Sizes are those of the pruned layers that the library is benchmarked with (28672 x 8192, 14336 x 4096; 8 columns), generic ones and ragged ones.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
EPS = 1e-6
TOP = 448.0  # the largest number of e4m3


def _norm(name, rows, cols, dtype="bf16", residual="bf16", out="e4m3", group=0):
    """`residual`: its type, or "" for none."""
    c = {"op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "residual": residual, "out": out, "group": group}
    return dict(c, name=name) if name else c


def _int4(name, rows, cols, n, group=128, dtype="bf16", out="bf16", zeros=True, x_group=-1):
    """`x_group`: -1 X in `dtype`; 0 in e4m3 with a scale for each row; else with one for so many neighbours."""
    c = {"op": "int4", "rows": rows, "cols": cols, "n": n, "group": group, "dtype": dtype, "out": out, "zeros": zeros, "x_group": x_group}
    return dict(c, name=name) if name else c


def _moe(name, tokens, hidden, inner, experts, top, group=0, dtype="bf16", routed=False):
    """`group`: 0 for experts in `dtype`, else of their 4-bit integers (with zeros)."""
    c = {"op": "moe", "tokens": tokens, "hidden": hidden, "inner": inner, "experts": experts, "top": top, "group": group, "dtype": dtype, "routed": routed}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token before a product in 16 bits: nothing but latency
        _norm("norm_1x4096_bf16", 1, 4096, out="bf16"),
        # a batch of eight in decoding
        _norm("norm_8x8192_rows", 8, 8192, dtype="f16", residual="f16"),
        # a long prompt, scales as fine as the weights'
        _norm("norm_8192x8192_g128", 8192, 8192, group=128),
        # short prompts of ragged size, the residual kept in 32 bits
        _norm("norm_5001x4090_g32", 5001, 4090, residual="f32", group=32),
        # one token
        _int4("int4_n1", 28672, 8192, 1, dtype="f16", out="f16"),
        # decoding of eight sequences, activations as the norm leaves them
        _int4("int4_n8_e4m3", 28672, 8192, 8, zeros=False, x_group=128),
        # a small layer of a speculative model, a few tokens
        _int4("int4_small_n5_g32", 2048, 1024, 5, group=32),
        # a layer of odd shape, a batch of 33
        _int4("int4_ragged_n33_g64", 14331, 4090, 33, group=64, dtype="f16", out="f32"),
        # one token through a small layer in 16 bits
        _moe("moe_bf16_t1", 1, 2048, 1024, 64, 8),
        # decoding of eight sequences, experts in 4 bits
        _moe("moe_int4_t8", 8, 4096, 2048, 64, 8, group=128),
        # ... of 32: nearly every expert is chosen
        _moe("moe_int4_t32", 32, 4096, 2048, 128, 4, group=64, dtype="f16"),
        # experts chosen by the program, padded places among them, odd shape
        _moe("moe_f16_t17_routed", 17, 2056, 1008, 10, 3, dtype="f16", routed=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges; half of them have sizes of no particular form."""
    op = rng.choice(["norm", "int4", "int4", "moe", "moe"])
    step = rng.choice([1, 1, 8, 64])
    dtype = rng.choice(["f16", "bf16"])

    def size(lo, hi, unit=1):
        return max(lo, _log_int(rng, lo, hi) // max(step, unit) * max(step, unit))

    if op == "norm":
        dtype = rng.choice(["f32", "f16", "bf16"])
        out = rng.choice(["e4m3", "e4m3", dtype])
        return _norm(None, size(1, 8192), size(64, 8192), dtype, rng.choice(["", "f32", dtype]), out, rng.choice([0, 32, 64, 128]) if out == "e4m3" else 0)
    if op == "int4":
        return _int4(None, size(256, 28672), size(128, 8192), _log_int(rng, 1, 33), rng.choice([32, 64, 128]), dtype, rng.choice([dtype, "f32"]), rng.random() < 0.5,
                     rng.choice([-1, -1, 0, 32, 64, 128]))
    group = rng.choice([0, 32, 64, 128])
    unit = 1 if group else 8  # rows of 16-bit experts start on 16 bytes
    experts = rng.choice([4, 8, 10, 16, 32, 64] if group else [4, 8, 10, 16])
    return _moe(None, _log_int(rng, 1, 32), size(256, 4096, unit), size(128, 2048, unit), experts, rng.randint(1, min(8, experts)), group, dtype, rng.random() < 0.3)


# ------------------------------------------------------------------ inputs

def _normal(g, r, c, dtype, spread=1.0):
    """Normal values; every 64th column, at places of the seed, is 20 times as large: the outlier channels of activations."""
    x = torch.randn(r, c, generator=g, device="cuda")
    at = torch.randint(0, c, (max(1, c // 64),), generator=g, device="cuda")
    x[:, at] *= 20
    return (x * spread).to(dtype)


def _weights(g, rows, cols, group, dtype, zeros):
    """A matrix of normal values in 4-bit integers: ``values`` two codes a byte, low half first, rows padded to a multiple of 16 bytes;
    ``scales`` and ``zeros`` [groups, rows]."""
    groups = -(-cols // group)
    w = torch.randn(rows, groups * group, generator=g, device="cuda", dtype=torch.float16).view(rows, groups, group)
    if zeros:
        low, high = w.amin(2, keepdim=True).float(), w.amax(2, keepdim=True).float()
        scale = ((high - low) / 15).clamp(min=1e-6)
        zero = (-low / scale).round().clamp(0, 15)
    else:
        scale = w.abs().amax(2, keepdim=True).float() / 7
        zero = torch.full_like(scale, 8)
    code = (w / scale.half() + zero.half()).round_().clamp_(0, 15).to(torch.uint8).view(rows, -1)[:, :cols]
    code = torch.nn.functional.pad(code, (0, -cols % 32))
    return {"values": code[:, 0::2] | code[:, 1::2] << 4, "scales": (scale[:, :, 0].t() / math.sqrt(cols)).to(dtype).contiguous(),
            "zeros": zero[:, :, 0].t().to(torch.uint8).contiguous() if zeros else None}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    dtype = TYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        state["X"] = _normal(g, rows, cols, dtype)
        state["R"] = _normal(g, rows, cols, TYPES[case["residual"]], 3.0) if case["residual"] else None
        state["w"] = (1 + 0.2 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
    elif case["op"] == "int4":
        rows, cols, n = case["rows"], case["cols"], case["n"]
        state["W"] = _weights(g, rows, cols, case["group"], dtype, case["zeros"])
        X = _normal(g, n, cols, dtype)
        if case["x_group"] >= 0:
            X = _plain_e4m3(X.float(), case["x_group"])
        state["X"] = X
    else:
        T, H, I, E, top = case["tokens"], case["hidden"], case["inner"], case["experts"], case["top"]
        state["X"] = _normal(g, T, H, dtype)
        if case["group"]:
            state["gate_up"] = _weights(g, E * 2 * I, H, case["group"], dtype, True)
            state["down"] = _weights(g, E * H, I, case["group"], dtype, True)
        else:
            state["gate_up"] = torch.randn(E, 2 * I, H, generator=g, device="cuda").mul_(1 / math.sqrt(H)).to(dtype)
            state["down"] = torch.randn(E, H, I, generator=g, device="cuda").mul_(1 / math.sqrt(I)).to(dtype)
        state["router"] = (torch.randn(E, H, generator=g, device="cuda") / math.sqrt(H)).to(dtype)
        if case["routed"]:
            ids = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :top].int()
            ids[torch.rand(T, top, generator=g, device="cuda") < 0.1] = -1
            state["ids"] = ids
            state["shares"] = torch.rand(T, top, generator=g, device="cuda")
    return state


# ------------------------------------------------------------------ the plain form

def _plain_e4m3(y, group):
    """(values, scales [rows, groups]) of y; a scale of 0 stands for zeros."""
    rows, cols = y.shape
    size = group or cols
    y = torch.nn.functional.pad(y, (0, -cols % size)).view(rows, -1, size)
    scale = y.abs().amax(2) / TOP
    q = (y / torch.where(scale > 0, scale, 1.0)[:, :, None]).clamp(-TOP, TOP).to(TYPES["e4m3"])
    return q.view(rows, -1)[:, :cols].contiguous(), scale


def _plain_x(X, x_group):
    if x_group < 0:
        return X.float()
    q, scale = X
    return q.float() * scale.repeat_interleave(x_group or q.shape[1], 1)[:, :q.shape[1]]


def _plain_int4(w, cols, group, rows=slice(None)):
    """Those rows of the matrix, in 32 bits."""
    code = torch.stack([w["values"][rows] & 15, w["values"][rows] >> 4], -1).flatten(-2)[..., :cols].float()
    scale = w["scales"].t()[rows].float().repeat_interleave(group, -1)[..., :cols]
    zero = w["zeros"].t()[rows].float().repeat_interleave(group, -1)[..., :cols] if w["zeros"] is not None else 8.0
    return (code - zero) * scale


def _plain_moe(s):
    T, H, I, top = s["tokens"], s["hidden"], s["inner"], s["top"]
    X = s["X"].float()
    if s["routed"]:
        ids, shares = s["ids"], s["shares"]
    else:
        # in 64 bits, for which of two experts is the larger
        logits = s["X"].double() @ s["router"].double().t()
        ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :top]
        p = torch.exp(logits - logits.amax(1, keepdim=True)).gather(1, ids)
        shares = (p / p.sum(1, keepdim=True)).float()
        ids = ids.int()
    used = torch.unique(ids[ids >= 0]).long()
    if s["group"]:
        rows = lambda n: (used[:, None] * n + torch.arange(n, device=X.device)).view(-1)  # noqa: E731
        gate_up = _plain_int4(s["gate_up"], H, s["group"], rows(2 * I)).view(-1, 2 * I, H)
        down = _plain_int4(s["down"], I, s["group"], rows(H)).view(-1, H, I)
    else:
        gate_up, down = s["gate_up"][used].float(), s["down"][used].float()
    h = X @ gate_up.transpose(1, 2)  # [used, T, 2 I]
    gate, up = h[..., :I], h[..., I:]
    y = (gate / (1 + torch.exp(-gate)) * up) @ down.transpose(1, 2)
    share = ((ids[None] == used[:, None, None]) * shares).sum(2)  # [used, T]
    y = (y * share[:, :, None]).sum(0).to(s["X"].dtype)
    return y if s["routed"] else {"y": y, "ids": ids, "shares": shares}


def run(state):
    s = state
    if own:
        import hopper_spmm_b200 as hs
        if s["op"] == "norm":
            y = hs.rms_norm(s["X"], s["w"], EPS, residual=s["R"], dtype=TYPES[s["out"]], group=s["group"] or None)
            y, h = y if s["R"] is not None else (y, None)
            y = (y.values, y.scales) if s["out"] == "e4m3" else y
            return (y, h)
        if s["op"] == "int4":
            W = hs.Int4Matrix(s["rows"], s["cols"], s["group"], **s["W"])
            out = TYPES[s["out"]]
            X = hs.Fp8Matrix(*s["X"], group=s["x_group"] or None) if s["x_group"] >= 0 else s["X"]
            return W.linear(X, dtype=out)
        I, H, E = s["inner"], s["hidden"], s["experts"]
        gate_up, down = s["gate_up"], s["down"]
        if s["group"]:
            gate_up = hs.Int4Matrix(E * 2 * I, H, s["group"], **gate_up)
            down = hs.Int4Matrix(E * H, I, s["group"], **down)
        layer = hs.MoeLayer(s["router"], gate_up, down, top_k=s["top"])
        if s["routed"]:
            return layer.experts(s["X"], s["ids"], s["shares"])
        y, ids, shares = layer.forward(s["X"], return_routing=True)
        return {"y": y, "ids": ids, "shares": shares}
    if s["op"] == "norm":
        h = s["X"].float()
        if s["R"] is not None:
            h = h + s["R"].float()
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + EPS) * s["w"].float()
        y = _plain_e4m3(y, s["group"]) if s["out"] == "e4m3" else y.to(TYPES[s["out"]])
        return (y, h.to(s["R"].dtype) if s["R"] is not None else None)
    if s["op"] == "int4":
        return (_plain_x(s["X"], s["x_group"]) @ _plain_int4(s["W"], s["cols"], s["group"]).t()).to(TYPES[s["out"]])
    return _plain_moe(s)


def work(case):
    """Inputs once, outputs once; of the experts those that are chosen, as many as so many tokens choose on average."""
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        rows, cols, group = case["rows"], case["cols"], case["group"]
        res = 2 * TYPES[case["residual"]].itemsize if case["residual"] else 0
        scales = 4 * rows * (-(-cols // group) if group else 1) if case["out"] == "e4m3" else 0
        return {"bytes": rows * cols * (size + res + TYPES[case["out"]].itemsize) + cols * size + scales, "flops": 0}
    if case["op"] == "int4":
        rows, cols, n, group = case["rows"], case["cols"], case["n"], case["group"]
        x = n * cols * (size if case["x_group"] < 0 else 1)
        return {"bytes": rows * cols / 2 + rows * -(-cols // group) * (size + case["zeros"]) + x + rows * n * TYPES[case["out"]].itemsize, "flops": 2 * rows * cols * n}
    T, H, I, E, top, group = case["tokens"], case["hidden"], case["inner"], case["experts"], case["top"], case["group"]
    chosen = E * (1 - (1 - top / E) ** T)
    value = 0.5 + (size + 1) / group if group else size
    return {"bytes": chosen * 3 * H * I * value + E * H * size * (not case["routed"]) + 2 * T * H * size, "flops": 6 * T * top * H * I + 2 * T * E * H * (not case["routed"])}


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_matrix(w, cols, group, first, count):
    """Rows first .. first + count of the 4-bit matrix."""
    v = w["values"][first:first + count].long()
    code = torch.empty(count, v.shape[1] * 2, dtype=torch.float64, device=v.device)
    code[:, 0::2] = v % 16
    code[:, 1::2] = v // 16
    at = torch.arange(cols, device=v.device) // group
    zero = 8 if w["zeros"] is None else w["zeros"][:, first:first + count][at].t().double()
    return (code[:, :cols] - zero) * w["scales"][:, first:first + count][at].t().double()


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "norm":
        h = s["X"].double() + (s["R"].double() if s["R"] is not None else 0)
        y = h * (h.square().mean(1, keepdim=True) + EPS).rsqrt() * s["w"].double()
        if s["out"] == "e4m3":
            at = torch.arange(y.shape[1], device=y.device) // (s["group"] or y.shape[1])
            scale = torch.zeros(y.shape[0], int(at[-1]) + 1, dtype=torch.float64, device=y.device)
            scale = scale.index_reduce_(1, at, y.abs(), "amax") / TOP
            a = y / scale[:, at].clamp(min=1e-300)
            unit = torch.exp2(torch.frexp(a.abs())[1].clamp(min=-5).double() - 4)
            y = ((a / unit).round() * unit, scale)
        return (y, h if s["R"] is not None else None)
    if s["op"] == "int4":
        if s["x_group"] >= 0:
            q, scale = s["X"]
            X = q.double() * scale.double()[:, torch.arange(s["cols"], device=q.device) // (s["x_group"] or s["cols"])]
        else:
            X = s["X"].double()
        return X @ _exact_matrix(s["W"], s["cols"], s["group"], 0, s["rows"]).t()
    T, H, I, E = s["tokens"], s["hidden"], s["inner"], s["experts"]
    X = s["X"].double()
    if s["routed"]:
        ids, shares = s["ids"].cpu(), s["shares"].double().cpu()
    else:
        logits = (X @ s["router"].double().t()).cpu()
        ids = torch.argsort(-logits, dim=1, stable=True)[:, :s["top"]]
        shares = torch.softmax(logits.gather(1, ids), 1)
    y = torch.zeros_like(X)
    for e in range(E):
        t, j = torch.where(ids == e)
        if len(t) == 0:
            continue
        if s["group"]:
            gate_up, down = _exact_matrix(s["gate_up"], H, s["group"], e * 2 * I, 2 * I), _exact_matrix(s["down"], I, s["group"], e * H, H)
        else:
            gate_up, down = s["gate_up"][e].double(), s["down"][e].double()
        gate, up = (X[t.cuda()] @ gate_up.t()).split(I, 1)
        y.index_add_(0, t.cuda(), shares[t, j].cuda()[:, None] * ((gate * torch.sigmoid(gate) * up) @ down.t()))
    return y if s["routed"] else {"y": y, "ids": ids.int(), "shares": shares}
