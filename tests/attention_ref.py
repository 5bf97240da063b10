"""Plain 64-bit forms of the rotary positions, the 4-bit cache and attention
over it, which the GPU tests compare with."""

import math

import torch

HALF = 2.0**-8  # half a step of bf16, relative


def codes(x):
    """(codes, step, minimum) of head vectors, in 64 bits; NaN minimum where a value is not finite."""
    x = x.double()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s, m = ((hi - lo) / 15).float().bfloat16().double(), lo.float().bfloat16().double()
    c = torch.where(s > 0, ((x - m) / s).round().clamp(0, 15), torch.zeros_like(x))
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    return torch.where(bad, 0.0, c), torch.where(bad, 0.0, s), torch.where(bad, math.nan, m)


def held(x):
    c, s, m = codes(x)
    return c * s + m


def rotate(x, pos, inv_freq, interleaved, factor=1.0):
    """x [tokens][heads][dim] turned by the tokens' positions; the table is held in 32 bits."""
    rot = 2 * len(inv_freq)
    z = pos.double()[:, None] * torch.as_tensor(inv_freq, dtype=torch.float64, device=x.device)
    cos, sin = ((f(z) * factor).float().double()[:, None] for f in (torch.cos, torch.sin))
    i = torch.arange(0, rot, 2, device=x.device) if interleaved else torch.arange(rot // 2, device=x.device)
    j = i + (1 if interleaved else rot // 2)
    y = x.double().clone()
    y[..., i] = x[..., i].double() * cos - x[..., j].double() * sin
    y[..., j] = x[..., j].double() * cos + x[..., i].double() * sin
    return y


def attend(q, k, v, first, window, scale):
    """One sequence: q [rows][heads][dim], row r is token first + r; k, v [tokens][kv_heads][dim] (values held).
    Returns the output and how far a kernel that rounds probabilities, keys and values to bf16 may be off:
    half a step of the output, of each value (sum p |v|), of each probability, and of each key, which moves
    a score by at most HALF * |scale| * sum |q| |k| and the output by twice that times sum p |v|.
    A probability may be rounded times its step s, on the code less 8: that errs on s |c - 8| =
    |v - (m + 8 s)| <= |v| + |mid| + s, mid the middle of the vector (codes reach 0 and at least 14, so mid is
    within s of m + 8 s, and s <= (max - min) / 14)."""
    rows, heads, _ = q.shape
    q = q.double()
    group = heads // k.shape[1]
    i = first + torch.arange(rows, device=q.device)[:, None]
    j = torch.arange(k.shape[0], device=q.device)
    seen = (j <= i) & ((j > i - window) if window else torch.ones_like(j, dtype=torch.bool))
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(heads):
        kk, vv = k[:, h // group], v[:, h // group]
        if kk.shape[0] == 0:
            continue
        x = (q[:, h] @ torch.nan_to_num(kk).T * scale)
        x = torch.where(torch.isnan(kk).any(-1)[None] | torch.isnan(vv).any(-1)[None], math.nan, x)
        x = x.masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = (x - torch.where(top == -math.inf, 0.0, top)).exp()
        p = torch.where(seen, p, 0.0)
        total = p.sum(-1, keepdim=True)
        p = torch.where(seen.any(-1, keepdim=True), p / total, 0.0)
        o = p @ torch.nan_to_num(vv)
        a = p @ torch.nan_to_num(vv).abs()
        lo, hi = torch.nan_to_num(vv).amin(-1), torch.nan_to_num(vv).amax(-1)
        b = a + (p @ ((lo + hi).abs() / 2 + (hi - lo) / 14))[:, None]
        sway = abs(scale) * (q[:, h].abs() @ torch.nan_to_num(kk).abs().T).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        out[:, h] = o
        tol[:, h] = HALF * (o.abs() + a + b + 2 * sway * a) + 1e-5 * a + 1e-30
    return out, tol
