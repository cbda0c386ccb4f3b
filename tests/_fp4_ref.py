"""Float64 restatement of the 4-bit microscaled operators, from their formulas."""
from __future__ import annotations

import torch

BLOCK = {"nvfp4": 16, "mxfp4": 32}
LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def e4m3_values(device):
    """The 127 finite non-negative values, ascending (byte = index)."""
    b = torch.arange(127, dtype=torch.float64, device=device)
    e, m = torch.div(b, 8, rounding_mode="floor"), b % 8
    return torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2(e - 7))


def nearest(t, table):
    """Index of the nearest entry of an ascending table for t >= 0; ties to the even index, past the end the last."""
    mid = ((table[1:] + table[:-1]) / 2).contiguous()
    t = t.contiguous()
    lo = torch.searchsorted(mid, t, right=False)
    hi = torch.searchsorted(mid, t, right=True)
    return torch.where(lo % 2 == 0, lo, hi)


def quantize(x, kind, g=1.0):
    """x [rows, cols] (any float type) -> row-major bytes (codes [rows, nb*B/2], scales [rows, nb])."""
    x = x.double()
    rows, cols = x.shape
    b = BLOCK[kind]
    nb = -(-cols // b)
    v = torch.zeros(rows, nb * b, dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, nb, b)
    bad = ~torch.isfinite(v).all(-1)
    a = torch.where(bad[..., None], torch.zeros_like(v), v.abs()).amax(-1)
    g = torch.as_tensor(g, dtype=torch.float64, device=x.device).reshape(())
    if kind == "nvfp4":
        table = e4m3_values(x.device)
        byte = nearest(a / (6 * g), table)
        s = table[byte] * g
    else:
        _, e = torch.frexp(a)
        byte = torch.where(a > 0, (e - 3).clamp(-127, 127) + 127, torch.zeros_like(e))
        s = torch.exp2(byte.double() - 127)
    t = torch.where(s[..., None] > 0, v.abs() / s[..., None].clamp(min=1e-300), 0.0)
    code = nearest(torch.where(bad[..., None], torch.zeros_like(t), t), LEVELS.to(x.device))
    sign = torch.signbit(v) & ~bad[..., None]
    code = (code + 8 * sign).to(torch.uint8).view(rows, -1)
    byte = torch.where(bad, torch.full_like(byte, 127 if kind == "nvfp4" else 255), byte)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte.to(torch.uint8)


def values(codes, scales, kind, cols, g=1.0):
    """Row-major bytes [..., rows, *] -> float64 values [..., rows, cols]."""
    dev = codes.device
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    q = LEVELS.to(dev)[n & 7] * torch.where(n >= 8, -1.0, 1.0).double()
    if kind == "nvfp4":
        table = torch.cat((e4m3_values(dev), torch.full((1,), float("nan"), dtype=torch.float64, device=dev)))
        s = table[scales.long()]
    else:
        s = torch.where(scales == 255, float("nan"), torch.exp2(scales.double() - 127))
    g = torch.as_tensor(g, dtype=torch.float64, device=dev)
    return ((q.unflatten(-1, (-1, BLOCK[kind])) * s[..., None]).flatten(-2) * g)[..., :cols]


def silu_mul(gu):
    g, u = gu.double().chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def product_bound(x, w, dtype):
    """(y, bound) of y = x W^T for float64 values x [m, K], w [n, K] and an output of ``dtype``.

    Products of two 4-bit values and their scales are exact (2 * (2 + 4) bits).  A K = 64 step sums 64 of them and the
    accumulator: at worst each addend loses the bits below 2^-24 of the largest partial sum, which is at most
    S = sum |x||w|, so a step is off by at most 65 * 2^-24 S_step + 2^-24 S and all steps together by
    (65 + steps) * 2^-24 S.  The two global scales cost three roundings, the output half a step of its type.
    """
    y = x @ w.T
    S = x.abs() @ w.abs().T
    steps = -(-x.shape[-1] // 64)
    tol = (65 + steps + 3) * 2.0 ** -24 * S
    if dtype != torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (y.abs() + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return y, tol
