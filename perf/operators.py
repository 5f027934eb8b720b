"""The 4-bit floating-point operators as measurable cases.

A matrix in 4 bits holds e2m1 values (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, and one scale per
block of a row: ``nvfp4`` has e4m3 scales for blocks of 16 and a power of two for the whole matrix, ``mxfp4`` powers of two
(e8m0) for blocks of 32.  ``op`` of a case:

* ``quantize``  X to 4 bits, blocks along its rows (``axis`` 1) or columns (``axis`` 0: the transpose), and back again
* ``linear``    Y = W Xᵀ with W kept in 4 bits and X, new at every call, brought to 4 bits first
* ``weight``    Y = W B with W kept in 4 bits and B in 16
* ``train``     one step of a linear layer in 4 bits: forward, gradient of the input, gradient of the weights; all three
                operands are quantised along whatever axis their product sums over

Sizes are those of the pruned layers that the library is benchmarked with (28672 x 8192, 14336 x 4096; 8, 64, 192 and 2048
columns) and ragged ones between.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def _case(name, op, fmt, rows, cols, n=0, dtype="bf16", out="bf16", axis=1, tokens_first=False):
    """`rows` x `cols`: W (or X, where it is quantised alone).  `n`: tokens.  `tokens_first`: the dense operand and the
    result are [n, ...] row by row, as activations usually lie, instead of [..., n]."""
    c = {"op": op, "format": fmt, "rows": rows, "cols": cols, "n": n, "dtype": dtype, "out": out, "axis": axis,
         "tokens_first": tokens_first}
    return dict(c, name=name) if name else c


def listed():
    return [
        # the activations of a batch of eight in decoding: nothing but latency
        _case("quantize_nv_8x8192", "quantize", "nvfp4", 8, 8192, dtype="f16", out="f16"),
        # a layer's weights when a model is loaded
        _case("quantize_nv_28672x8192", "quantize", "nvfp4", 28672, 8192, dtype="f16", out="f16"),
        # activations of ragged size from a full-precision part of a model, transposed for a gradient
        _case("quantize_mx_5001x4090_t", "quantize", "mxfp4", 5001, 4090, dtype="f32", out="f32", axis=0),
        # decoding of eight sequences, both operands in 4 bits
        _case("linear_nv_n8", "linear", "nvfp4", 28672, 8192, 8, dtype="f16", out="f16"),
        # a long prompt, both operands in 4 bits
        _case("linear_nv_n2048", "linear", "nvfp4", 28672, 8192, 2048, tokens_first=True),
        # a batch of short prompts through a layer of odd shape
        _case("linear_mx_ragged", "linear", "mxfp4", 14331, 4090, 333, out="f32"),
        # one token
        _case("weight_nv_n1", "weight", "nvfp4", 28672, 8192, 1, dtype="f16", out="f16", tokens_first=True),
        # a small layer of a speculative model, a few tokens
        _case("weight_mx_small_n5", "weight", "mxfp4", 2048, 1024, 5, tokens_first=True),
        # a batch of short prompts, activations kept in 16 bits (the library's own layout)
        _case("weight_nv_n192", "weight", "nvfp4", 28672, 8192, 192, dtype="f16", out="f16"),
        # a long prompt, activations kept in 16 bits
        _case("weight_mx_n2048", "weight", "mxfp4", 28672, 8192, 2048, tokens_first=True),
        # a training step of a square layer, two sequences of 2048
        _case("train_nv_4096", "train", "nvfp4", 4096, 4096, 4096),
        # ... of a narrow layer of odd shape
        _case("train_mx_ragged", "train", "mxfp4", 2050, 1111, 777, out="f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the same ranges; three in four have sizes of no particular form."""
    op = rng.choice(["quantize", "linear", "linear", "weight", "weight", "train"])
    fmt = rng.choice(["nvfp4", "mxfp4"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    out = rng.choice(["bf16", "f16", "f32"])
    step = rng.choice([1, 1, 2, 64])
    axis, tokens_first = 1, rng.random() < 0.5

    def size(lo, hi):
        return max(lo, _log_int(rng, lo, hi) // step * step)

    if op == "quantize":
        rows, cols, n, axis = size(1, 16384), size(32, 8192), 0, rng.choice([0, 1])
    elif op == "train":
        rows, cols, n = size(512, 4096), size(512, 4096), size(64, 4096)
    else:
        rows, cols, n = size(1024, 28672), size(512, 8192), _log_int(rng, 1, 2048)
        if n > 16 and rng.random() < 0.5:
            n = n // 16 * 16
    if op == "weight":  # scales that are powers of two over the whole range need bfloat16's range
        dtype = "bf16" if fmt == "mxfp4" or dtype == "f32" else dtype
    return _case(None, op, fmt, rows, cols, n, dtype, out, axis, tokens_first)


# ------------------------------------------------------------------ the plain form

def _ceil(a, b):
    return -(-a // b)


def _plain_quantize(x, fmt):
    """(codes 0..15 [R, K], scales [R, blocks] as 32-bit values, the matrix's scale) of x along its rows.

    All steps are exact or rounded as the definition says in 32 bits: factors 2^k change no digits, a quotient of 24 bits
    rounds to a border of the few-bit types only where it is one."""
    R, K = x.shape
    blk = BLOCK[fmt]
    x = torch.nn.functional.pad(x.float(), (0, _ceil(K, blk) * blk - K)).view(R, -1, blk)
    amax = x.abs().amax(2)
    if fmt == "mxfp4":
        e = torch.frexp(amax)[1] - 3
        e = torch.where(amax > 0, e, -127).clamp(-127, 127)
        scale, whole = torch.exp2(e.double()), torch.ones((), dtype=torch.float64, device=x.device)
        q = x.abs().double() / scale[:, :, None]
    else:
        m, k = torch.frexp(x.abs().amax().double() / 2688)
        k = torch.where(m == 0, 0, torch.where(m == 0.5, k - 1, k)).clamp(-126, 127)
        whole = torch.exp2(k.double())
        scale = (amax / 6 / whole.float()).clamp(max=448).to(torch.float8_e4m3fn).float()
        q = x.abs() / whole.float() / torch.where(scale > 0, scale, torch.inf)[:, :, None]
    code = ((q > 0.25).to(torch.uint8) + (q >= 0.75) + (q > 1.25) + (q >= 1.75) + (q > 2.5) + (q >= 3.5) + (q > 5)).to(torch.uint8)
    code += torch.signbit(x).to(torch.uint8) * 8
    return code.view(R, -1)[:, :K], scale, whole


def _lut(device, dtype):
    v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=dtype, device=device)
    return torch.cat([v, -v])


def _plain_values(code, scale, whole, fmt, dtype=torch.float32):
    """The matrix that (codes, scales) stand for."""
    K = code.shape[1]
    s = (scale * whole).to(dtype).repeat_interleave(BLOCK[fmt], 1)[:, :K]
    return _lut(code.device, dtype)[code.int()] * s


def _round_trip(x, fmt):
    return _plain_values(*_plain_quantize(x, fmt), fmt)


# ------------------------------------------------------------------ 4-bit matrices as they are stored

def _store(code, scale, whole, fmt):
    """values: two codes a byte, low half first, rows padded with zeros to a multiple of 16 bytes.  scales: blocks of 128 rows x
    4 scales, byte (r % 32) * 16 + (r / 32) * 4 + j of a block for its row r and scale j; blocks row-block by row-block, zeros
    where the matrix ends inside one.  scale: 32-bit, one number."""
    R, K = code.shape
    code = torch.nn.functional.pad(code, (0, _ceil(K, 32) * 32 - K))
    values = code[:, 0::2] | code[:, 1::2] << 4
    if fmt == "mxfp4":
        s = (torch.frexp(scale)[1] - 1 + 127).to(torch.uint8)
    else:
        s = scale.to(torch.float8_e4m3fn).view(torch.uint8)
    R4, G = _ceil(R, 128), _ceil(s.shape[1], 4)
    s = torch.nn.functional.pad(s, (0, G * 4 - s.shape[1], 0, R4 * 128 - R))
    s = s.view(R4, 4, 32, G, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)
    return {"values": values.contiguous(), "scales": s, "scale": whole.float().view(1)}


def _load(w, rows, cols, fmt, dtype):
    """The matrix that is stored, in `dtype`."""
    code = torch.stack([w["values"] & 15, w["values"] >> 4], 2).view(rows, -1)[:, :cols]
    blocks = _ceil(cols, BLOCK[fmt])
    s = w["scales"].view(_ceil(rows, 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(_ceil(rows, 128) * 128, -1)[:rows, :blocks]
    s = torch.exp2(s.double() - 127) if fmt == "mxfp4" else s.contiguous().view(torch.float8_e4m3fn).double()
    s = (s * w["scale"].double()).to(dtype).repeat_interleave(BLOCK[fmt], 1)[:, :cols]
    return _lut(code.device, dtype)[code.int()] * s


# ------------------------------------------------------------------ the cases

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, n, dtype = case["rows"], case["cols"], case["n"], TYPES[case["dtype"]]

    def normal(r, c, spread):
        """Normal values; every 64th column, at places of the seed, is 20 times as large: the outlier channels of activations."""
        x = torch.randn(r, c, generator=g, device="cuda")
        at = torch.randint(0, c, (max(1, c // 64),), generator=g, device="cuda")
        x[:, at] *= 20
        return (x * spread).to(dtype)

    state = dict(case)
    if case["op"] == "quantize":
        state["X"] = normal(rows, cols, 1.0)
    elif case["op"] == "train":
        state["W"] = (torch.randn(rows, cols, generator=g, device="cuda") / math.sqrt(cols)).to(dtype)
        state["X"] = normal(n, cols, 1.0)
        state["dY"] = normal(n, rows, 1e-3)
    else:
        w = torch.randn(rows, cols, generator=g, device="cuda") / math.sqrt(cols)
        state["W"] = _store(*_plain_quantize(w.half(), case["format"]), case["format"])
        x = normal(n, cols, 1.0)
        state["B"] = x if case["tokens_first"] or case["op"] == "linear" else x.t().contiguous()
    return state


def _weight(hs, s):
    w = s["W"]
    return hs.Fp4Matrix(s["rows"], s["cols"], s["format"], values=w["values"], scales=w["scales"], tensor_scale=w["scale"])


def run(state):
    s, fmt, out = state, state["format"], TYPES[state["out"]]
    if own:
        import hopper_spmm_b200 as hs
        if s["op"] == "quantize":
            return hs.fp4_quantize(s["X"], fmt, axis=s["axis"]).dequantize(dtype=out)
        if s["op"] == "train":
            W, Wt = hs.fp4_quantize_both(s["W"], fmt)
            X, Xt = hs.fp4_quantize_both(s["X"], fmt)
            dY, dYt = hs.fp4_quantize_both(s["dY"], fmt)
            return {"Y": X.matmul(W, dtype=out, sync=False), "dX": dY.matmul(Wt, dtype=out, sync=False),
                    "dW": dYt.matmul(Xt, dtype=out, sync=False)}
        W = _weight(hs, s)
        if s["op"] == "linear":
            X = hs.fp4_quantize(s["B"], fmt)
            return X.matmul(W, dtype=out, sync=False) if s["tokens_first"] else W.matmul(X, dtype=out, sync=False)
        if s["tokens_first"]:
            Y = torch.empty(s["n"], s["rows"], dtype=out, device=s["B"].device)
            W.matmul(s["B"].t(), Y.t(), dtype=out, sync=False)
            return Y
        return W.matmul(s["B"], dtype=out, sync=False)
    if s["op"] == "quantize":
        x = s["X"] if s["axis"] == 1 else s["X"].t()
        return _round_trip(x, fmt).to(out)
    if s["op"] == "train":
        W, X, dY = s["W"], s["X"], s["dY"]
        Y = _round_trip(X, fmt) @ _round_trip(W, fmt).t()
        dX = _round_trip(dY, fmt) @ _round_trip(W.t(), fmt).t()
        dW = _round_trip(dY.t(), fmt) @ _round_trip(X.t(), fmt).t()
        return {"Y": Y.to(out), "dX": dX.to(out), "dW": dW.to(out)}
    W = _load(s["W"], s["rows"], s["cols"], fmt, torch.float32)
    if s["op"] == "linear":
        X = _round_trip(s["B"], fmt)
        Y = X @ W.t() if s["tokens_first"] else W @ X.t()
    else:
        B = s["B"].float()
        Y = B @ W.t() if s["tokens_first"] else W @ B
    return Y.to(out)


def work(case):
    """Inputs once, outputs once, and what is kept in 4 bits at 4 bits and its scales."""
    rows, cols, n = case["rows"], case["cols"], case["n"]
    b_in, b_out = TYPES[case["dtype"]].itemsize, TYPES[case["out"]].itemsize
    b_4 = 0.5 + 1 / BLOCK[case["format"]]
    if case["op"] == "quantize":
        return {"bytes": rows * cols * (b_in + b_4 + b_out), "flops": 0}
    if case["op"] == "train":
        ins, outs = rows * cols + n * cols + n * rows, n * rows + n * cols + rows * cols
        return {"bytes": ins * b_in + outs * b_out, "flops": 6 * rows * cols * n}
    return {"bytes": rows * cols * b_4 + n * cols * b_in + rows * n * b_out, "flops": 2 * rows * cols * n}


# ------------------------------------------------------------------ the definition in 64 bits

_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest_e2m1(a):
    """The nearest of the eight values to a >= 0, at equal distance the one with an even code."""
    v = torch.tensor(_E2M1, dtype=torch.float64, device=a.device)
    up = torch.searchsorted(v, a).clamp(1, 7)  # v[up - 1] < a <= v[up], at the ends the nearest pair
    low, high = a - v[up - 1], v[up] - a
    return v[torch.where((low < high) | (low == high) & ((up - 1) % 2 == 0), up - 1, up)]


def _nearest_e4m3(a):
    """The nearest e4m3 value to a >= 0: multiples of 2^(e - 3) for a in [2^e, 2^(e+1)), e >= -6, at most 448."""
    e = (torch.frexp(a)[1] - 1).clamp(min=-6)
    unit = torch.exp2((e - 3).double())
    return (torch.round(a / unit) * unit).clamp(max=448.0)


def _exact_round_trip(x, fmt):
    x = x.double()
    R, K = x.shape
    blk = BLOCK[fmt]
    x = torch.cat([x, x.new_zeros(R, -K % blk)], 1).unflatten(1, (-1, blk))
    top = x.abs().max(2, keepdim=True).values
    if fmt == "mxfp4":
        s = torch.exp2((torch.frexp(top)[1] - 3).clamp(-127, 127).double())
        s[top == 0] = 2.0 ** -127
    else:
        most = float(top.max())
        whole = 1.0
        if most > 0:
            m, k = math.frexp(most / 2688)
            whole = 2.0 ** min(127, max(-126, k - 1 if m == 0.5 else k))
        s = _nearest_e4m3(top / 6 / whole) * whole
    y = torch.where(s > 0, _nearest_e2m1((x.abs() / torch.where(s > 0, s, 1.0)).clamp(max=6.0)), 0.0)
    return (torch.copysign(y, x) * s).flatten(1)[:, :K]


def exact(case, seed):
    s = prepare(case, seed)
    fmt = s["format"]
    if s["op"] == "quantize":
        return _exact_round_trip(s["X"] if s["axis"] == 1 else s["X"].t(), fmt)
    if s["op"] == "train":
        q = {k: (_exact_round_trip(s[k], fmt), _exact_round_trip(s[k].t(), fmt)) for k in ("W", "X", "dY")}
        return {"Y": q["X"][0] @ q["W"][0].t(), "dX": q["dY"][0] @ q["W"][1].t(), "dW": q["dY"][1] @ q["X"][1].t()}
    W = _load(s["W"], s["rows"], s["cols"], fmt, torch.float64)
    if s["op"] == "linear":
        X = _exact_round_trip(s["B"], fmt)
        return X @ W.t() if s["tokens_first"] else W @ X.t()
    B = s["B"].double()
    return B @ W.t() if s["tokens_first"] else W @ B
