"""How far the attention kernels may be off, counted for the roundings that they make.

Both hold sums, maxima and references in 32 bits and round to f16 (11 bits, half a step 2^-11 of the value), the
output to bf16 (half a step 2^-8):
  * a key's values (many rows; few rows multiply bare codes): a score moves by at most d_j = 2^-11 |scale| sum |q K_j|,
    the output by sum p_j d_j |V_j - o| <= sum p_j d_j |V_j| + |o| sum p_j d_j;
  * a value and its probability (many rows), 2^-11 of p |V| each; or a probability times its value's step (few rows),
    2^-11 of p s c = p (V - m), m the vector's smallest: together at most 2^-11 p (2 |V| + |m|);
  * f16's smallest steps, 2^-24, where the largest of 128 keys or values in turn is 2^13 or more and a vector's largest at
    most 2^12 below (many rows): half of one is 2^-26 of the vector's largest;
  * 32-bit sums of D products and of the keys, and the exponential's argument: 2^-20 and 1e-5.
That is the worst case.  Roundings are independent, so over many outputs from values around zero their root mean
square is far below it: 2^-7 / sqrt(12) = 0.00226 of the output for its bf16, a few 2^-10 / sqrt(12) = 0.0003 for the
others, that of the keys times the scores' own size (about 4 for these inputs): 0.0026 in all.  RMS allows 0.004."""

import math

import torch

BF16, F16 = 2.0**-8, 2.0**-11
RMS = 0.004


def attend(q, k, v, first, window, scale):
    """One sequence: q [rows][heads][dim], row r is token first + r; k, v [tokens][kv_heads][dim] (values held, finite).
    (output, worst case), in 64 bits."""
    rows, heads, _ = q.shape
    q = q.double()
    group = heads // k.shape[1]
    i = first + torch.arange(rows, device=q.device)[:, None]
    j = torch.arange(k.shape[0], device=q.device)
    seen = j <= i
    if window:
        seen = seen & (j > i - window)
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    if k.shape[0] == 0:
        return out, tol
    for h in range(heads):
        kk, vv = k[:, h // group], v[:, h // group]
        x = (q[:, h] @ kk.T * scale).masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = (x - torch.where(top == -math.inf, 0.0, top)).exp()
        p = torch.where(seen.any(-1, keepdim=True), p / p.sum(-1, keepdim=True), 0.0)
        o, a = p @ vv, p @ vv.abs()
        low = (p @ vv.amin(-1).abs())[:, None]
        fine = 2.0**-26 * (p @ vv.abs().amax(-1))[:, None]
        moved = p * (abs(scale) * 1.05 * ((F16 + 2.0**-20) * (q[:, h].abs() @ kk.abs().T)
                                          + 2.0**-26 * q[:, h].abs().sum(-1, keepdim=True) * kk.abs().amax(-1)))
        out[:, h] = o
        tol[:, h] = (BF16 * o.abs() + F16 * (2 * a + low) + fine + moved @ vv.abs() + o.abs() * moved.sum(-1, keepdim=True)
                     + 1.1e-5 * a + 1e-37)
    return out, tol


def check(out, q, k, v, q_len, kv_len, window=0, scale=None, rms=True):
    """Every sequence against its form in 64 bits; ``rms`` where the values are spread around zero."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    a = b = 0
    for ql, kl in zip(q_len, kv_len):
        want, tol = attend(q[a : a + ql], k[b : b + kl], v[b : b + kl], kl - ql, window, scale)
        got = out[a : a + ql].double()
        assert torch.isfinite(got).all(), (ql, kl)
        off = (got - want).abs()
        if ql:
            assert float((off / tol.clamp(min=1e-300)).max()) <= 1.0, (ql, kl, float((off / tol.clamp(min=1e-300)).max()))
        if rms and ql:
            size = float(want.square().mean().sqrt())
            assert float(off.square().mean().sqrt()) <= RMS * size, (ql, kl, float(off.square().mean().sqrt()) / max(size, 1e-300))
        a, b = a + ql, b + kl
