"""8-bit rows and projections against 64-bit forms.  Codes are whole numbers and
have to be equal: the kernel takes a quotient in 64 bits wherever 32 cannot
decide it.  Scales and outputs: a few roundings of 2^-24."""

import math

import pytest
import torch

from klearu_b200._lib import KlError
from klearu_b200.quant import Q8Linear, add_rms_norm_q8, quantize_rows_q8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0**-24


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def check_norm(r, h, weight, eps, norm):
    """h: what is quantized before the norm (f32)."""
    cols = h.shape[1]
    u = h.double() * weight.double()
    top = u.abs().amax(-1, keepdim=True)
    want = torch.where(top > 0, (u * 127 / top).round(), 0.0)
    assert torch.equal(r.codes.double(), want)
    rms = (h.double().square().mean(-1) + eps).sqrt() if norm else 1.0
    scale = top[:, 0] / rms / 127
    # the sum of squares: cols roundings at worst, halved by the root; product, root, quotients: one each
    assert ((r.scales.double() - scale).abs() <= (cols / 2 + 6) * U * scale).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (5, 17), (130, 1000), (2, 11008), (700, 64), (1, 49152),
                                       (2, 8190)])
def test_norm_codes(gpu_ctx, rows, cols, dtype):
    x, res = randn(rows, cols, seed=1, dtype=dtype), 4 * randn(rows, cols, seed=2)
    w = 1 + 0.2 * randn(cols, seed=3)
    r = add_rms_norm_q8(x, w, residual=res, eps=1e-5, ctx=gpu_ctx)
    h = x.float() + res
    assert torch.equal(r.hidden, h)
    check_norm(r, h, w, 1e-5, True)
    r = add_rms_norm_q8(x, w, eps=1e-3, one_plus_weight=True, ctx=gpu_ctx)
    assert r.hidden is None
    check_norm(r, x.float(), 1 + w, 1e-3, True)
    r = quantize_rows_q8(x, ctx=gpu_ctx)
    check_norm(r, x.float(), torch.ones(cols, device=DEV), 0, False)


def test_norm_at_borders(gpu_ctx):
    """Values that stand on the border of two codes, where rounding goes to the even one."""
    t = torch.arange(-127, 127, device=DEV).float() + 0.5
    x = torch.cat([t, torch.tensor([127.0, -127.0], device=DEV)]).repeat(4, 1)
    for mul in (1.0, 0.3, 1e-20, 1e15):
        y = x * mul
        check_norm(quantize_rows_q8(y, ctx=gpu_ctx), y, torch.ones(256, device=DEV), 0, False)
    w = 1 + 0.1 * randn(256, seed=5)
    y = x / w  # borders up to a rounding
    check_norm(add_rms_norm_q8(y, w, eps=0.0, ctx=gpu_ctx), y, w, 0.0, True)


def test_norm_in_place_views_and_special_rows(gpu_ctx):
    rows, cols = 6, 100
    base = randn(rows, 131, seed=1)
    res = base[:, 3:103]
    keep = base.clone()
    x = randn(rows, 3, cols, seed=2, dtype=torch.bfloat16)[:, 1]
    want = x.float() + res
    r = add_rms_norm_q8(x, torch.ones(cols, device=DEV), residual=res, hidden=res, ctx=gpu_ctx)
    assert r.hidden is res and torch.equal(res, want)
    assert torch.equal(base[:, :3], keep[:, :3]) and torch.equal(base[:, 103:], keep[:, 103:])
    check_norm(r, want, torch.ones(cols, device=DEV), 1e-5, True)
    y = randn(5, cols, seed=4)
    y[0], y[1, 7], y[2, 3], y[3, 9] = 0.0, math.nan, math.inf, 3e38
    r = add_rms_norm_q8(y, torch.ones(cols, device=DEV), ctx=gpu_ctx)
    assert r.scales[0] == 0 and (r.codes[0] == 0).all()
    assert torch.isnan(r.scales[1:4]).all() and (r.codes[1:4] == 0).all()
    check_norm(add_rms_norm_q8(y[4:], torch.ones(cols, device=DEV), ctx=gpu_ctx), y[4:], torch.ones(cols, device=DEV), 1e-5, True)
    assert torch.isfinite(r.scales[4])
    z = y[4:].clone()
    q = add_rms_norm_q8(z, torch.ones(cols, device=DEV), hidden=z, ctx=gpu_ctx)  # h = x, in place
    assert torch.equal(q.codes, r.codes[4:])


def codes(rows, cols, seed, pad=True):
    ld = -(-cols // 16) * 16 if pad else cols
    return torch.randint(-127, 128, (rows, ld), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV,
                         dtype=torch.int8)[:, :cols]


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 127, 130, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (17, 16), (64, 100), (130, 128), (257, 1000), (1000, 4096), (96, 11008)])
def test_product(gpu_ctx, m, n, k):
    a, w = codes(m, k, 1), codes(n, k, 2, pad=False)
    sa, sw = 0.1 + randn(m, seed=3).abs(), 0.01 + randn(n, seed=4).abs()
    bias = randn(n, seed=5)
    exact = (a.double() @ w.double().T)
    want = exact * sa.double()[:, None] * sw.double()
    lin = Q8Linear(w, sw, ctx=gpu_ctx)
    got = lin.forward(a, sa)
    assert got.dtype == torch.float32
    assert ((got.double() - want).abs() <= 4 * U * want.abs()).all()
    got = lin.forward(a, sa, out_dtype=torch.bfloat16)
    assert ((got.double() - want).abs() <= (2.0**-8 + 4 * U) * want.abs()).all()
    lin = Q8Linear(w, sw, bias=bias, ctx=gpu_ctx)
    start = randn(m, n, seed=6)
    out = start.clone()
    assert lin.forward(a, sa, out=out, accumulate=True) is out
    full = want + bias.double() + start.double()
    size = want.abs() + bias.double().abs() + start.double().abs()
    assert ((out.double() - full).abs() <= 6 * U * size).all()


@pytest.mark.parametrize("m,n,k", [(257, 9700, 40), (700, 8001, 200), (1025, 4096, 272), (2560, 2000, 1000)])
def test_product_of_many_tiles(gpu_ctx, m, n, k):
    """More tiles of 256 x 128 than the device has processors, so that each takes several, ragged at both edges."""
    a, w = codes(m, k, 1), codes(n, k, 2, pad=False)
    sa, sw, bias = 0.1 + randn(m, seed=3).abs(), 0.01 + randn(n, seed=4).abs(), randn(n, seed=5)
    want = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    lin = Q8Linear(w, sw, bias=bias, ctx=gpu_ctx)
    got = lin.forward(a, sa)
    assert ((got.double() - want - bias.double()).abs() <= 5 * U * (want.abs() + bias.double().abs())).all()
    wide = torch.full((m, n + 9), 7.0, dtype=torch.bfloat16, device=DEV)
    lin.forward(a, sa, out=wide[:, 1 : n + 1])
    tol = 2.0**-8 * (want + bias.double()).abs() + 5 * U * (want.abs() + bias.double().abs())
    assert ((wide[:, 1 : n + 1].double() - want - bias.double()).abs() <= tol).all()
    assert (wide[:, :1] == 7).all() and (wide[:, n + 1 :] == 7).all()
    start = randn(m, n + 3, seed=6)
    out = start.clone()[:, 2 : n + 2]
    lin.forward(a, sa, out=out, accumulate=True)
    full = want + bias.double() + start[:, 2 : n + 2].double()
    size = want.abs() + bias.double().abs() + start[:, 2 : n + 2].double().abs()
    assert ((out.double() - full).abs() <= 6 * U * size).all()


def test_offsets_beyond_32_bits(gpu_ctx):
    """Rows so far apart that byte offsets pass 2^32."""
    far = 20_000_000  # 300 rows: 6e9 bytes of codes
    wide = torch.empty(300, far, dtype=torch.int8, device=DEV)
    out = torch.empty(300, far // 4, dtype=torch.float32, device=DEV)
    n, k = 40, 96
    w, sw = codes(n, k, 2, pad=False), 0.01 + randn(n, seed=4).abs()
    lin = Q8Linear(w, sw, ctx=gpu_ctx)
    x = randn(300, k, seed=1)
    rows = quantize_rows_q8(x, ctx=gpu_ctx)
    for m in (300, 64, 2):
        a = wide[300 - m :, far - 128 : far - 128 + k]
        a.copy_(rows.codes[300 - m :])
        o = out[300 - m :, far // 4 - 45 : far // 4 - 5]
        lin.forward(a, rows.scales[300 - m :], out=o)
        want = (a.double() @ w.double().T) * rows.scales[300 - m :, None].double() * sw.double()
        assert ((o.double() - want).abs() <= 4 * U * want.abs()).all()
    y = out[:, :k]
    y.copy_(x)
    assert torch.equal(quantize_rows_q8(y, ctx=gpu_ctx).codes, rows.codes)


def test_product_extremes(gpu_ctx):
    """-128 and the largest sums that 32 bits have to hold; NaN scales stay in their rows and channels."""
    k = 131071
    a = torch.full((3, k + 1), -128, dtype=torch.int8, device=DEV)[:, :k]
    w = torch.full((5, k), -128, dtype=torch.int8, device=DEV)
    w[1] = 127
    sa, sw = torch.ones(3, device=DEV), torch.ones(5, device=DEV)
    got = Q8Linear(w, sw, ctx=gpu_ctx).forward(a, sa)
    assert torch.equal(got[0].double(), (a[:1].double() @ w.double().T)[0].float().double())
    sa[1], sw[2] = math.nan, math.nan
    got = Q8Linear(w, sw, ctx=gpu_ctx).forward(a, sa)
    bad = torch.isnan(got)
    assert bad[1].all() and bad[:, 2].all() and bad.sum() == 7


@pytest.mark.parametrize("m", [3, 40, 200])
def test_product_views(gpu_ctx, m):
    """Rows of codes inside a wider matrix, an output with gaps that are left alone."""
    k, n = 72, 50
    wide = codes(m, 512, 1)
    a, w = wide[:, 16:88], codes(n, 100, 2, pad=False)[:, 5:77]
    sa, sw = 0.1 + randn(m, seed=3).abs(), 0.01 + randn(n, seed=4).abs()
    want = (a.double() @ w.double().T) * sa.double()[:, None] * sw.double()
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((m, n + 3), 9.0, dtype=dtype, device=DEV)
        Q8Linear(w, sw, ctx=gpu_ctx).forward(a, sa, out=out[:, 1 : n + 1])
        assert ((out[:, 1 : n + 1].double() - want).abs() <= ((2.0**-8 if dtype == torch.bfloat16 else 0) + 4 * U) * want.abs()).all()
        assert (out[:, 0] == 9).all() and (out[:, n + 1 :] == 9).all()


def test_from_weights(gpu_ctx):
    w = randn(40, 64, seed=1)
    w[3] = 0
    x = randn(5, 64, seed=2)
    r = quantize_rows_q8(x, ctx=gpu_ctx)
    got = Q8Linear.from_weights(w.cpu().numpy(), ctx=gpu_ctx).forward(r.codes, r.scales)
    top = w.double().abs().amax(-1, keepdim=True)
    held = torch.where(top > 0, (w.double() * 127 / top).round() * top / 127, 0.0)
    want = (r.codes.double() * r.scales.double()[:, None]) @ held.T
    assert ((got.double() - want).abs() <= 1e-5 * (x.double().abs() @ w.double().abs().T)).all()
    assert (got[:, 3] == 0).all()


def test_refusals(gpu_ctx):
    x = randn(4, 32)
    w = torch.ones(32, device=DEV)
    for bad in (x.half(), x.cpu(), x.T, x[0], x[:, :0], x.clone().requires_grad_()):
        with pytest.raises(ValueError):
            add_rms_norm_q8(bad, w, ctx=gpu_ctx)
    with pytest.raises(ValueError):
        add_rms_norm_q8(x, w[:31], ctx=gpu_ctx)
    with pytest.raises(ValueError):
        add_rms_norm_q8(x, w, residual=x[:3], ctx=gpu_ctx)
    with pytest.raises(ValueError):
        add_rms_norm_q8(x, w, residual=x.bfloat16(), ctx=gpu_ctx)
    with pytest.raises(KlError):
        add_rms_norm_q8(x, w, eps=-1.0, ctx=gpu_ctx)
    with pytest.raises(KlError):
        quantize_rows_q8(torch.zeros(1, 49153, device=DEV), ctx=gpu_ctx)
    c, s = codes(4, 32, 1), torch.ones(4, device=DEV)
    with pytest.raises(ValueError):
        Q8Linear(c.float(), s, ctx=gpu_ctx)
    with pytest.raises(ValueError):
        Q8Linear(c, s[:3], ctx=gpu_ctx)
    with pytest.raises(KlError):
        Q8Linear(torch.zeros(1, 131072, dtype=torch.int8, device=DEV), s[:1], ctx=gpu_ctx)
    lin = Q8Linear(c, s, ctx=gpu_ctx)
    for a, sc in ((c[:, :16], s), (c.int(), s), (c, s[:3]), (codes(4, 48, 1)[:, 3:35], s), (codes(4, 40, 1, pad=False)[:, :32], s)):
        with pytest.raises(ValueError):
            lin.forward(a, sc)
    with pytest.raises(ValueError):
        lin.forward(c, s, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        lin.forward(c, s, accumulate=True)
    with pytest.raises(ValueError):
        lin.forward(c, s, out=torch.zeros(4, 4, dtype=torch.bfloat16, device=DEV), accumulate=True)
    with pytest.raises(ValueError):
        lin.forward(c, s, out=torch.zeros(4, 5, device=DEV))
    assert lin.forward(c[:0], s[:0]).shape == (0, 4)
    assert quantize_rows_q8(x[:0], ctx=gpu_ctx).codes.shape == (0, 32)
    gpu_ctx.sync()
