"""Matrices of 4-bit integers in 64 bits, from their definition, for the tests."""
import torch

import hopper_spmm_b200 as hs
from fp4_ref import EPS, TINY


def arrays(rows, cols, group, seed, dtype=torch.float16, zeros=True, device="cuda", spread=None):
    """Random codes, scales and zeros; anything in the padding of values."""
    g = torch.Generator(device=device).manual_seed(seed)
    groups = -(-cols // (group or cols)) if cols else (0 if group else 1)
    values = torch.randint(0, 256, (rows, (cols + 31) // 32 * 16), generator=g, device=device, dtype=torch.uint8)
    scales = (torch.rand(groups, rows, generator=g, device=device) + 0.1) * (spread or 0.05)
    z = torch.randint(0, 16, (groups, rows), generator=g, device=device, dtype=torch.uint8) if zeros else None
    return values, scales.to(dtype), z


def matrix(rows, cols, group, seed, dtype=torch.float16, zeros=True, spread=None):
    v, s, z = arrays(rows, cols, group, seed, dtype, zeros, spread=spread)
    return hs.Int4Matrix(rows, cols, group, values=v, scales=s, zeros=z)


def values_of(m, rows=slice(None)):
    """What these rows of an Int4Matrix stand for, in 64 bits."""
    v = m.values[rows]
    code = torch.stack([v & 15, v >> 4], 2).view(v.shape[0], -1)[:, :m.cols].double()
    at = torch.arange(m.cols, device=v.device) // (m.group or max(m.cols, 1))
    zero = 8 if m.zeros is None else m.zeros[:, rows][at].t().double()
    return (code - zero) * m.scales[:, rows][at].t().double()


def check_product(got, a, b, span):
    """got = a b up to the roundings of its sums and type.  Products are exact; `span` of them are added up 16 at a time, each addition off by at most 2^-22 of
    the sum of magnitudes (a truncated fp32 addition of a partial sum that is itself aligned and truncated); a product with the columns' scale, a fused
    addition for each span and one for each part of k (28 at most) are roundings of fp32."""
    want, mag = a @ b, a.abs() @ b.abs()
    bound = mag * (span / 16 * 2.0 ** -22 + (-(-a.shape[1] // span) + 28 + 3) * 2.0 ** -24)
    bound = bound + (want.abs() + bound) * EPS[got.dtype] + TINY[got.dtype]
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), "NaN in other places"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~nan].double(), want[~fine & ~nan])
    worst = float((err / bound)[fine].max()) if fine.any() else 0.0
    assert worst <= 1, f"{worst:.2f} times the bound"
