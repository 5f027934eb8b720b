"""4-bit matrices in 64 bits, from their definition, for the tests: values, their stored bytes, and products."""
import torch

BLOCK = {"nvfp4": 16, "mxfp4": 32}
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def e4m3_values():
    """The 127 numbers of e4m3 from 0 to 448, by code."""
    out = []
    for code in range(127):
        e, m = code >> 3, code & 7
        out.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    return torch.tensor(out, dtype=torch.float64)


def nearest(a, table):
    """Index into the ascending table of the number nearest to a >= 0; of two as near, the even index."""
    up = torch.searchsorted(table, a.contiguous()).clamp(1, len(table) - 1)
    low, high = a - table[up - 1], table[up] - a
    return torch.where((low < high) | ((low == high) & ((up - 1) % 2 == 0)), up - 1, up)


def tensor_exponent(x):
    """k of the tensor's scale 2^k."""
    a = x.double().abs()
    most = float(a[torch.isfinite(a)].max()) if torch.isfinite(a).any() else 0.0
    if most == 0:
        return 0
    k = -126
    while most > 2688 * 2.0 ** k and k < 127:
        k += 1
    return k


def quantize(x, fmt, k=None):
    """(codes [R, K], scale bytes [R, blocks], k) of x along its rows; k: the tensor's exponent where it is given."""
    R, K = x.shape
    blk = BLOCK[fmt]
    k = (tensor_exponent(x) if k is None else k) if fmt == "nvfp4" else 0
    x = torch.cat([x.double(), torch.zeros(R, -K % blk, dtype=torch.float64, device=x.device)], 1).view(R, -1, blk)
    bad = ~torch.isfinite(x).all(2)
    clean = torch.where(bad[:, :, None], 0.0, x)
    top = clean.abs().amax(2)
    if fmt == "mxfp4":
        e = (torch.frexp(top)[1] - 3).clamp(-127, 127)
        e = torch.where(top > 0, e, -127)
        byte, s = e + 127, torch.exp2(e.double())
        byte = torch.where(bad, 255, byte)
    else:
        byte = nearest((top / 6 * 2.0 ** -k).clamp(max=448.0), e4m3_values().to(x.device))
        s = e4m3_values().to(x.device)[byte] * 2.0 ** k
        byte = torch.where(bad, 127, byte)
    safe = torch.where(s > 0, s, 1.0)[:, :, None]
    code = nearest((clean.abs() / safe).clamp(max=6.0), torch.tensor(E2M1, dtype=torch.float64, device=x.device))
    code = torch.where((s > 0)[:, :, None], code, 0)
    code = code + 8 * torch.signbit(clean).to(torch.int64)
    return code.view(R, -1)[:, :K].to(torch.uint8), byte.to(torch.uint8), k


def values(code, byte, k, fmt):
    """What codes and scale bytes stand for, in 64 bits."""
    v = torch.tensor(E2M1 + [-e for e in E2M1], dtype=torch.float64, device=code.device)[code.long()]
    if fmt == "mxfp4":
        s = torch.where(byte == 255, torch.nan, torch.exp2(byte.double() - 127))
    else:
        s = torch.cat([e4m3_values(), torch.tensor([torch.nan], dtype=torch.float64)]).to(code.device)[byte.long()]
    return v * s.repeat_interleave(BLOCK[fmt], 1)[:, :code.shape[1]] * 2.0 ** k


def scale_index(rows, n_scales):
    """Where scale j of row r is stored, [rows, n_scales]."""
    r, j = torch.arange(rows)[:, None], torch.arange(n_scales)[None, :]
    return ((r // 128) * ((n_scales + 3) // 4) + j // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + j % 4


def pack(code, byte, fmt):
    """The stored arrays (values [R, pitch], scales), zeros in every padding."""
    R, K = code.shape
    pitch = (K + 31) // 32 * 16
    full = torch.zeros(R, 2 * pitch, dtype=torch.uint8, device=code.device)
    full[:, :K] = code
    scales = torch.zeros((R + 127) // 128 * ((byte.shape[1] + 3) // 4) * 512, dtype=torch.uint8, device=code.device)
    scales[scale_index(R, byte.shape[1]).to(code.device)] = byte
    return full[:, 0::2] | full[:, 1::2] << 4, scales


def unpack(values_, scales, rows, cols, fmt):
    code = torch.stack([values_ & 15, values_ >> 4], 2).view(rows, -1)[:, :cols]
    n = (cols + BLOCK[fmt] - 1) // BLOCK[fmt]
    return code, scales[scale_index(rows, n).to(scales.device)]


def matrix_values(m):
    """What an Fp4Matrix stands for, in 64 bits."""
    code, byte = unpack(m.values, m.scales, m.rows, m.cols, m.format)
    return values(code, byte, 0, m.format) * (m.tensor_scale.double() if m.format == "nvfp4" else 1.0)


EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}  # half a subnormal step


def check_product(got, a, b, step):
    """got = a b up to the rounding of fp32 sums and of got's type.  Every product of two operands is exact in fp32; the sum takes
    ceil(K / step) additions to an accumulator, each off by at most 2^-22 of the sum of magnitudes (a truncated fp32 addition
    of a partial sum that is itself aligned and truncated to as many bits), and a few that join parts."""
    want, mag = a @ b, a.abs() @ b.abs()
    bound = mag * ((a.shape[1] + step - 1) // step + 12) * 2.0 ** -22
    bound = bound + (want.abs() + bound) * EPS[got.dtype] + TINY[got.dtype]
    err = (got.double() - want).abs()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), "NaN in other places"
    worst = float((err / bound)[~nan].max()) if (~nan).any() else 0.0
    assert worst <= 1, f"{worst:.2f} times the bound"
    return worst
