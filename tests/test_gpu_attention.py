"""Rotary positions, the paged 4-bit cache and attention over it, against plain
64-bit forms (attention_ref.py).

Inputs are bf16, so without a rotation a code is decided exactly: x - m and the
quotient's distance from a border need fewer bits than f32 has, unless a value
2^16 times smaller than m stands where 0 would be on the border.  With one, a
32-bit rotated value may fall on the other side of a border than the 64-bit one
(off by 3 roundings of 2^-24 against steps of at least 2^-9 of the minimum and
range): then a cached value is one step off, and a step or minimum one step of
bf16.  Attention is compared on the values that the cache holds."""

import math

import pytest
import torch

import attention_ref as R
from klearu_b200._lib import KL_EBOUNDS, KlError
from klearu_b200.attention import Kv4Cache, RopeTable, SeqBatch
from klearu_b200.core import Context

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def make_batch(q_len, kv_len, page, seed=0, extra_pages=0, max_q=None, max_kv=None):
    """Pages in an order of chance; returns the batch and the number of pages."""
    need = [-(-max(n, 0) // page) for n in kv_len]
    order = torch.randperm(sum(need) + extra_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.zeros(len(kv_len), max(need + [1]), dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
    cu = [0]
    for n in q_len:
        cu.append(cu[-1] + n)
    batch = SeqBatch(i32(cu), i32(kv_len), table.to(DEV), max_q=max(q_len + [0]) if max_q is None else max_q,
                     max_kv=max(kv_len + [0]) if max_kv is None else max_kv)
    return batch, max(1, sum(need) + extra_pages)


def randn(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def filled(ctx, kv_len, page, kv_heads, dim, seed=0, q_len=None, k=None, v=None, **kw):
    """A cache that holds random keys and values for kv_len tokens, a batch of q_len new ones, and the held values."""
    q_len = kv_len if q_len is None else q_len
    n = sum(kv_len)
    k = randn(n, kv_heads, dim, seed=seed + 1) * 1.5 + randn(kv_heads, dim, seed=seed + 2) if k is None else k
    v = randn(n, kv_heads, dim, seed=seed + 3) if v is None else v
    every, pages = make_batch(kv_len, kv_len, page, seed)
    cache = Kv4Cache(pages, page, kv_heads, dim, ctx=ctx)
    cache.append(k, v, every)
    cu = [0]
    for x in q_len:
        cu.append(cu[-1] + x)
    batch = SeqBatch(i32(cu), every.kv_len, every.page_table, max_q=kw.get("max_q", max(q_len)),
                     max_kv=kw.get("max_kv", max(kv_len)))
    return cache, batch, R.held(k), R.held(v)


def check_attend(out, q, batch, hk, hv, q_len, kv_len, window=0, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    a = b = 0
    for ql, kl in zip(q_len, kv_len):
        want, tol = R.attend(q[a : a + ql], hk[b : b + kl], hv[b : b + kl], kl - ql, window, scale)
        got = out[a : a + ql].double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        worst = float((torch.nan_to_num(got - want).abs() / torch.nan_to_num(tol, nan=1.0)).max()) if ql else 0.0
        assert worst <= 1.0, (ql, kl)
        a, b = a + ql, b + kl


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim,heads,kv_heads,page,q_len,kv_len", [
    (128, 4, 4, 16, [1], [1]), (128, 8, 2, 16, [5, 1, 33], [5, 40, 47]), (64, 3, 1, 48, [17, 2], [100, 2]),
    (64, 15, 5, 64, [1] * 70, list(range(1, 71))), (128, 7, 7, 32, [300, 0, 1], [300, 9, 513])])
def test_append_holds_the_codes(gpu_ctx, dim, heads, kv_heads, page, q_len, kv_len):
    t = sum(q_len)
    batch, pages = make_batch(q_len, kv_len, page)
    cache = Kv4Cache(pages, page, kv_heads, dim, ctx=gpu_ctx)
    q, k, v = randn(t, heads, dim, seed=1), randn(t, kv_heads, dim, seed=2) + 3, randn(t, kv_heads, dim, seed=3)
    k[0, 0] = 2.5  # a constant vector: step 0
    v[t // 2, -1, 3] = 1e4  # one channel far out
    assert torch.equal(cache.append(k, v, batch, q=q), q)
    got_k, got_v = cache.read(batch, t)
    assert torch.equal(got_k, R.held(k).float().bfloat16())
    assert torch.equal(got_v, R.held(v).float().bfloat16())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (128, 34), (128, 2), (64, 64), (64, 18), (64, 48)])
def test_rotation(gpu_ctx, dim, rot, interleaved):
    q_len, kv_len, heads, kv_heads = [9, 1, 4], [70000, 1, 131000], 3, 2
    t = sum(q_len)
    batch, pages = make_batch(q_len, kv_len, 1024)
    cache = Kv4Cache(pages, 1024, kv_heads, dim, ctx=gpu_ctx)
    rope = RopeTable(rot, 131072, interleaved=interleaved, scaling="by_parts", factor=16.0, original_positions=8192,
                     attention_factor=1.2, ctx=gpu_ctx)
    q, k, v = (randn(t, h, dim, seed=h) for h in (heads, kv_heads, kv_heads))
    got_q = cache.append(k, v, batch, q=q, rope=rope)
    got_k, got_v = cache.read(batch, t)
    pos = torch.cat([torch.arange(b - a, b, device=DEV) for a, b in zip(q_len, kv_len)])
    want = R.rotate(q, pos, rope.inv_freq, interleaved, 1.2)
    # half a bf16 step, and 3 roundings of the terms in 32 bits
    tol = R.HALF * want.abs() + 3 * 2.0**-24 * 1.2 * (q.double().abs() + q.double().abs().amax(-1, keepdim=True))
    assert ((got_q.double() - want).abs() <= tol).all()
    turned = R.rotate(k, pos, rope.inv_freq, interleaved, 1.2)
    c, s, m = R.codes(turned)
    # a code may be one step off at a border, and the bf16 step and minimum one of theirs; few are
    off = (got_k.double() - (c * s + m)).abs()
    assert (off <= 1.01 * s + 2 * R.HALF * (15 * s + m.abs())).all()
    assert (off > R.HALF * (15 * s + m.abs())).double().mean() < 1e-3
    assert torch.equal(got_v, R.held(v).float().bfloat16())


def test_rope_scaling_formulas(gpu_ctx):
    plain = RopeTable(64, 16, ctx=gpu_ctx).inv_freq
    assert (RopeTable(64, 16, scaling="linear", factor=4.0, ctx=gpu_ctx).inv_freq == plain / 4).all()
    parts = RopeTable(64, 16, scaling="by_parts", factor=4.0, original_positions=2048, ctx=gpu_ctx).inv_freq
    for f, g in zip(plain, parts):
        turns = 2048 * f / (2 * math.pi)
        want = f if turns >= 4 else f / 4 if turns <= 1 else f * ((turns - 1) / 3 + (1 - (turns - 1) / 3) / 4)
        assert abs(g - want) <= 1e-15 * f


def test_append_views_positions_and_in_place(gpu_ctx):
    """Queries, keys and values as views of one projection, odd strides, explicit positions, q_out = q."""
    dim, heads, kv_heads, t = 64, 5, 2, 11
    for pad in (0, 3):  # 3: rows that do not start on 16 bytes
        flat = randn(t, (heads + 2 * kv_heads) * dim + pad, seed=pad)
        q, k, v = (x.unflatten(1, (-1, dim)) for x in flat[:, pad:].split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
        batch, pages = make_batch([t], [t], 16)
        cache = Kv4Cache(pages, 16, kv_heads, dim, ctx=gpu_ctx)
        rope = RopeTable(dim, 1000, ctx=gpu_ctx)
        pos = torch.arange(t, dtype=torch.int32, device=DEV) * 7 + 5
        want = R.rotate(q, pos, rope.inv_freq, False)
        keep = flat.clone()
        got = cache.append(k, v, batch, q=q, rope=rope, positions=pos, q_out=q)
        assert got is q
        tol = R.HALF * want.abs() + 1e-5
        assert ((q.double() - want).abs() <= tol).all()
        assert torch.equal(flat[:, pad + heads * dim :], keep[:, pad + heads * dim :])
        gk, gv = cache.read(batch, t)
        assert torch.equal(gv, R.held(v).float().bfloat16())
        c, s, m = R.codes(R.rotate(k, pos, rope.inv_freq, False))
        assert ((gk.double() - (c * s + m)).abs() <= 1.01 * s + 2 * R.HALF * (15 * s + m.abs())).all()


def test_append_leaves_other_rows_and_tokens(gpu_ctx):
    """Padding in front, rows behind the last sequence, and the cache's other tokens."""
    dim, heads, kv_heads, page = 128, 2, 2, 16
    first = [20, 7]
    batch, pages = make_batch(first, first, page, max_q=20, max_kv=32)
    cache = Kv4Cache(pages + 1, page, kv_heads, dim, ctx=gpu_ctx)
    k, v = randn(27, kv_heads, dim, seed=1), randn(27, kv_heads, dim, seed=2)
    cache.append(k, v, batch)
    # sequence 0: one more token; sequence 1: 9 rows for a length of 7, two of them padding; 4 rows behind
    again = SeqBatch(i32([0, 1, 10]), i32([21, 7]), batch.page_table, max_q=9)
    k2, v2, q2 = randn(14, kv_heads, dim, seed=3), randn(14, kv_heads, dim, seed=4), randn(14, heads, dim, seed=5)
    q_out = torch.full_like(q2, 7.0)
    cache.append(k2, v2, again, q=q2, q_out=q_out)
    assert torch.equal(q_out[:1], q2[:1]) and torch.equal(q_out[3:10], q2[3:10])
    assert (q_out[1:3] == 0).all() and (q_out[10:] == 7).all()
    every = SeqBatch(i32([0, 21, 28]), i32([21, 7]), batch.page_table, max_q=21)
    gk, _ = cache.read(every, 28)
    want = torch.cat([k[:20], k2[:1], k2[3:10]])
    assert torch.equal(gk, R.held(want).float().bfloat16())
    gk, gv = cache.read(again, 14, k_out=torch.full((14, kv_heads, dim), 7.0, dtype=torch.bfloat16, device=DEV))
    assert (gk[1:3] == 0).all() and (gv[1:3] == 0).all() and (gk[10:] == 7).all()
    gpu_ctx.sync()


@pytest.mark.parametrize("interleaved,rot", [(None, 0), (True, 128), (False, 128), (False, 48), (True, 64)])
@pytest.mark.parametrize("dim", [64, 128])
def test_append_of_many_tokens(gpu_ctx, dim, interleaved, rot):
    """Prompts so long that a block takes several tokens; ragged, with padding and rows behind the last sequence."""
    heads, kv_heads, page = 16, 8, 48
    q_len, kv_len = [3001, 0, 5, 1800, 1], [3001, 4, 2, 1999, 700]  # the third: three rows of padding
    t = sum(q_len) + 3
    rot = min(rot, dim)
    batch, pages = make_batch(q_len, kv_len, page)
    cache = Kv4Cache(pages, page, kv_heads, dim, ctx=gpu_ctx)
    rope = RopeTable(rot, 4096, interleaved=interleaved, ctx=gpu_ctx) if rot else None
    q, k, v = (randn(t, h, dim, seed=s) for h, s in ((heads, 1), (kv_heads, 2), (kv_heads, 3)))
    q_out = torch.full_like(q, 7.0)
    cache.append(k, v, batch, q=q, rope=rope, q_out=q_out)
    gk, gv = cache.read(batch, t)
    pos = torch.cat([torch.arange(b - a, b, device=DEV) for a, b in zip(q_len, kv_len)])
    live = pos >= 0
    pos = pos.clamp(min=0)
    turned_q, turned_k = (R.rotate(x[:-3], pos, rope.inv_freq, interleaved) if rope else x[:-3].double() for x in (q, k))
    tol = R.HALF * turned_q.abs() + 3 * 2.0**-24 * (q[:-3].double().abs() + q.double().abs().amax())
    off = (q_out[:-3].double() - turned_q).abs()
    assert (off[live] <= tol[live]).all()
    assert (q_out[:-3][~live] == 0).all() and (q_out[-3:] == 7).all()
    assert torch.equal(gv[:-3][live], R.held(v[:-3]).float().bfloat16()[live])
    c, s, m = R.codes(turned_k)
    off, step = (gk[:-3].double() - (c * s + m)).abs()[live], (15 * s + m.abs())[live]
    assert (off <= 1.01 * s[live] + 2 * R.HALF * step).all()
    assert (off > R.HALF * step).double().mean() < 1e-3


@pytest.mark.parametrize("t", [4 * 65535 + 77, 32 * 65535 + 77])
def test_more_tokens_than_a_grid_is_high(gpu_ctx, t):
    batch, pages = make_batch([t], [t], 1024)
    cache = Kv4Cache(pages, 1024, 1, 64, ctx=gpu_ctx)
    k, v = randn(t, 1, 64, seed=1), randn(t, 1, 64, seed=2)
    cache.append(k, v, batch)
    gk, gv = cache.read(batch, t)
    assert torch.equal(gk, R.held(k).float().bfloat16()) and torch.equal(gv, R.held(v).float().bfloat16())


@pytest.mark.parametrize("max_q", [1, 60])
def test_more_sequences_than_a_grid_is_high(gpu_ctx, max_q):
    """70000 sequences of one token, every fifth without any; a token that sees only itself gives its value."""
    n = 70000
    kv = [0 if i % 5 == 0 else 1 for i in range(n)]
    table = torch.randperm(n, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(n, 1).to(DEV)
    batch = SeqBatch(torch.arange(n + 1, dtype=torch.int32, device=DEV), i32(kv), table, max_q=max_q, max_kv=1)
    cache = Kv4Cache(n, 16, 1, 64, ctx=gpu_ctx)
    q, k, v = randn(n, 2, 64, seed=1), randn(n, 1, 64, seed=2), randn(n, 1, 64, seed=3)
    cache.append(k, v, batch)
    out = cache.attend(q, batch)
    want = torch.where(torch.tensor(kv, device=DEV)[:, None, None] > 0, R.held(v), 0.0)
    # a value and the output are rounded once each
    assert ((out.double() - want).abs() <= 2 * R.HALF * 1.01 * (want.abs() + (v.double().abs().amax(-1, keepdim=True) / 7))).all()


@pytest.mark.parametrize("q_len", [[1, 3], [300, 70]])
def test_offsets_beyond_32_bits(gpu_ctx, q_len):
    """Pages behind the first 4 GB of a cache, rows of queries and outputs behind 4 GB of theirs."""
    kv_heads, dim, page, kv_len = 8, 128, 1024, [1500, 700]
    pages = 4100
    cache = Kv4Cache(pages, page, kv_heads, dim, ctx=gpu_ctx)
    table = i32([[4099, 3], [4098, 0]])
    n = sum(kv_len)
    k, v = randn(n, kv_heads, dim, seed=1), randn(n, kv_heads, dim, seed=2)
    cache.append(k, v, SeqBatch(i32([0, 1500, 2200]), i32(kv_len), table, max_q=1500))
    batch = SeqBatch(i32([0, q_len[0], sum(q_len)]), i32(kv_len), table, max_q=max(q_len))
    gk, _ = cache.read(batch, sum(q_len))
    want = R.held(torch.cat([k[1500 - q_len[0] : 1500], k[2200 - q_len[1] :]]))
    assert torch.equal(gk, want.float().bfloat16())
    t, far = sum(q_len), 4_400_000_000 // (2 * sum(q_len)) // 8 * 8
    q = torch.empty(t, far, dtype=torch.bfloat16, device=DEV)[:, far - 16 * dim :].unflatten(1, (16, dim))
    q.copy_(randn(t, 16, dim, seed=4))
    out = torch.empty(t, far, dtype=torch.bfloat16, device=DEV)[:, far - 16 * dim :].unflatten(1, (16, dim))
    cache.attend(q, batch, out=out)
    check_attend(out, q, batch, R.held(k), R.held(v), q_len, kv_len)


def test_not_finite_values_read_back_as_nan(gpu_ctx):
    batch, pages = make_batch([5], [5], 16)
    cache = Kv4Cache(pages, 16, 2, 64, ctx=gpu_ctx)
    k, v = randn(5, 2, 64, seed=1), randn(5, 2, 64, seed=2)
    k[1, 0, 5], k[2, 1, 0], v[3, 1, 63] = math.nan, math.inf, -math.inf
    k[4, 0, 0], k[4, 0, 1] = 3.3e38, -3.3e38  # the range passes f32
    cache.append(k, v, batch)
    gk, gv = cache.read(batch, 5)
    bad_k, bad_v = torch.zeros(5, 2, dtype=torch.bool, device=DEV), torch.zeros(5, 2, dtype=torch.bool, device=DEV)
    bad_k[1, 0] = bad_k[2, 1] = bad_k[4, 0] = bad_v[3, 1] = True
    assert torch.equal(torch.isnan(gk).all(-1), bad_k) and torch.equal(torch.isnan(gk).any(-1), bad_k)
    assert torch.equal(torch.isnan(gv).all(-1), bad_v) and torch.equal(torch.isnan(gv).any(-1), bad_v)


# ---------------------------------------------------------------------------
# attend
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (6, 2), (8, 1), (20, 1), (32, 8)])
@pytest.mark.parametrize("window", [0, 20])
def test_one_token_each(gpu_ctx, dim, heads, kv_heads, window):
    kv_len = [1, 2, 15, 16, 17, 31, 33, 100, 255, 1000, 64]
    q_len = [1] * len(kv_len)
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 48, kv_heads, dim, q_len=q_len)
    q = randn(len(kv_len), heads, dim, seed=9) * 2
    check_attend(cache.attend(q, batch, window=window), q, batch, hk, hv, q_len, kv_len, window)


@pytest.mark.parametrize("kv_len", [[9001], [20000, 3], [4097, 130, 70000]])
def test_long_contexts(gpu_ctx, kv_len):
    q_len = [1] * len(kv_len)
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 64, 2, 128, q_len=q_len)
    q = randn(len(kv_len), 8, 128, seed=9) * 2
    check_attend(cache.attend(q, batch), q, batch, hk, hv, q_len, kv_len)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,page,window", [(4, 4, 16, 0), (6, 2, 48, 0), (14, 2, 112, 300), (8, 1, 64, 1),
                                                        (32, 8, 32, 33)])
@pytest.mark.parametrize("q_len,kv_len", [([2, 3, 1, 7], [2, 500, 1, 64]), ([16, 17, 40], [16, 300, 41]),
                                          ([130, 1, 0, 257], [130, 77, 12, 700]), ([513], [1100])])
def test_several_tokens(gpu_ctx, dim, heads, kv_heads, page, window, q_len, kv_len):
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, page, kv_heads, dim, q_len=q_len)
    q = randn(sum(q_len), heads, dim, seed=9) * 2
    check_attend(cache.attend(q, batch, window=window), q, batch, hk, hv, q_len, kv_len, window)


@pytest.mark.parametrize("q_len,max_q", [([1, 1, 1], 400), ([300, 2], 1), ([40, 70], 1), ([300, 2], 0)])
def test_hints_do_not_change_the_result(gpu_ctx, q_len, max_q):
    kv_len = [n + 90 for n in q_len]
    for max_kv in (1, 100000):
        cache, batch, hk, hv = filled(gpu_ctx, kv_len, 16, 2, 128, q_len=q_len, max_q=max_q, max_kv=max_kv)
        q = randn(sum(q_len), 8, 128, seed=9)
        check_attend(cache.attend(q, batch), q, batch, hk, hv, q_len, kv_len)


@pytest.mark.parametrize("q_len,kv_len", [([3, 1, 0, 9], [0, 0, 0, 4]), ([200, 5], [30, 0])])
def test_rows_that_see_nothing(gpu_ctx, q_len, kv_len):
    """Rows in front of a sequence's first token, sequences without tokens, rows behind the last sequence."""
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 16, 2, 64, q_len=q_len)
    t = sum(q_len)
    q = randn(t + 3, 6, 64, seed=9)
    out = torch.full_like(q, 5.0)
    cache.attend(q, batch, out=out)
    assert (out[t:] == 5).all()
    a = b = 0
    for ql, kl in zip(q_len, kv_len):
        want, tol = R.attend(q[a : a + ql], hk[b : b + kl], hv[b : b + kl], kl - ql, 0, 64**-0.5)
        assert ((out[a : a + ql].double() - want).abs() <= tol).all()
        assert (out[a : a + max(0, ql - kl)] == 0).all()
        a, b = a + ql, b + kl


@pytest.mark.parametrize("q_len", [[1, 1], [3, 2], [70, 90]])
@pytest.mark.parametrize("dim", [64, 128])
def test_nan_in_unseen_tokens(gpu_ctx, q_len, dim):
    """A key or value that is NaN reaches the rows that see it, and no other: later tokens, tokens before the window."""
    kv_len = [q_len[0] + 60, q_len[1] + 25]
    n = sum(kv_len)
    k, v = randn(n, 2, dim, seed=1), randn(n, 2, dim, seed=2)
    k[2, 0, 1] = math.nan  # in front of the window of all rows but the first few
    v[kv_len[0] - 1, 1, 3] = math.inf  # the last token: only the last row sees it
    k[kv_len[0] + 30 if q_len[1] > 5 else n - 1, 0, 0] = math.nan
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 16, 2, dim, q_len=q_len, k=k, v=v)
    q = randn(sum(q_len), 4, dim, seed=9)
    for window in (0, 40):
        check_attend(cache.attend(q, batch, window=window), q, batch, hk, hv, q_len, kv_len, window)


def test_garbage_behind_the_sequence(gpu_ctx):
    """A page's tokens behind a sequence's end (another use of the page left NaN there) have no effect."""
    dim, page = 128, 64
    full, pages = make_batch([page], [page], page)
    cache = Kv4Cache(pages, page, 2, dim, ctx=gpu_ctx)
    k = randn(page, 2, dim, seed=1)
    v = randn(page, 2, dim, seed=2)
    k[10:] = math.nan
    v[10:] = math.inf
    cache.append(k, v, full)
    for n, ql in ((10, 1), (9, 4), (10, 10)):
        batch = SeqBatch(i32([0, ql]), i32([n]), full.page_table, max_q=ql)
        q = randn(ql, 16, dim, seed=3)
        check_attend(cache.attend(q, batch), q, batch, R.held(k[:n]), R.held(v[:n]), [ql], [n])


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e18])
def test_value_sizes(gpu_ctx, size):
    """Values of any size, constant vectors among them, and a score scale that makes one key win."""
    kv_len, q_len = [200, 40], [1, 20]
    n = sum(kv_len)
    v = (randn(n, 2, 64, seed=2).float() * size).bfloat16()
    v[7] = size
    k = randn(n, 2, 64, seed=1)
    k[5] = 0.25
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 16, 2, 64, q_len=q_len, k=k, v=v)
    q = randn(sum(q_len), 4, 64, seed=9)
    for scale in (0.125, 4.0, 0.0, -0.2):
        check_attend(cache.attend(q, batch, scale=scale), q, batch, hk, hv, q_len, kv_len, scale=scale)


@pytest.mark.parametrize("size", [1e-20, 1e-3, 300.0, 1e15])
def test_query_and_key_sizes(gpu_ctx, size):
    """Queries of one size and keys of its inverse: ordinary scores from extreme factors."""
    kv_len, q_len = [150], [2]
    k = (randn(150, 2, 128, seed=1).float() / size).bfloat16()
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 16, 2, 128, q_len=q_len, k=k)
    q = (randn(2, 8, 128, seed=9).float() * size).bfloat16()
    check_attend(cache.attend(q, batch), q, batch, hk, hv, q_len, kv_len)
    q_len = [140]
    batch = SeqBatch(i32([0, 140]), batch.kv_len, batch.page_table, max_q=140)
    q = (randn(140, 8, 128, seed=9).float() * size).bfloat16()
    check_attend(cache.attend(q, batch), q, batch, hk, hv, q_len, kv_len)


def test_nan_queries(gpu_ctx):
    cache, batch, hk, hv = filled(gpu_ctx, [50, 50], 16, 1, 64, q_len=[1, 30])
    q = randn(31, 4, 64, seed=9)
    q[0, 1, 3], q[9, 2, 0] = math.nan, math.inf
    out = cache.attend(q, batch)
    bad = torch.zeros(31, 4, dtype=torch.bool, device=DEV)
    bad[0, 1] = bad[9, 2] = True
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()


@pytest.mark.parametrize("q_len", [[2, 1], [150, 40]])
def test_strided_queries_and_outputs(gpu_ctx, q_len):
    kv_len = [300, 41]
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 16, 2, 64, q_len=q_len)
    t = sum(q_len)
    for pad in (8, 1):  # 1: rows that do not start on 16 bytes
        q = randn(6, t, 64 + pad, seed=9)[..., pad:].transpose(0, 1)
        out = torch.full((t, 6, 64 + pad), 3.0, dtype=torch.bfloat16, device=DEV)
        cache.attend(q, batch, out=out[..., pad:])
        check_attend(out[..., pad:], q, batch, hk, hv, q_len, kv_len)
        assert (out[..., :pad] == 3).all()


def test_shared_prefix_pages(gpu_ctx):
    """Two sequences whose tables name the same pages."""
    cache, batch, hk, hv = filled(gpu_ctx, [64], 16, 2, 128, q_len=[1])
    table = batch.page_table.expand(2, -1).contiguous()
    two = SeqBatch(i32([0, 1, 3]), i32([64, 50]), table, max_q=2)
    q = randn(3, 4, 128, seed=9)
    out = cache.attend(q, two)
    check_attend(out, q, two, torch.cat([hk, hk[:50]]), torch.cat([hv, hv[:50]]), [1, 2], [64, 50])


@pytest.mark.parametrize("q_len", [[1, 1, 1], [40, 3, 70]])
def test_same_bits_every_time(gpu_ctx, q_len):
    cache, batch, _, _ = filled(gpu_ctx, [5000, 300, 90], 32, 2, 128, q_len=q_len)
    q = randn(sum(q_len), 8, 128, seed=9)
    first = cache.attend(q, batch)
    for _ in range(5):
        assert torch.equal(cache.attend(q, batch), first)


# ---------------------------------------------------------------------------
# refusals and reports
# ---------------------------------------------------------------------------
def test_bad_pages_and_lengths_are_reported(gpu_ctx):
    ctx = Context(0)
    k, v, q = randn(40, 2, 64, seed=1), randn(40, 2, 64, seed=2), randn(40, 4, 64, seed=3)
    cache = Kv4Cache(3, 16, 2, 64, ctx=ctx)
    good = SeqBatch(i32([0, 40]), i32([40]), i32([[0, 1, 2]]), max_q=40)
    cache.append(k, v, good)
    ctx.sync()
    one = torch.zeros(1, 4, 64, dtype=torch.bfloat16, device=DEV)
    for cu, kv, table, rows in ((  # a page behind the cache, a negative one, a length beyond the table, rows beyond the tensor
            [0, 40], [40], [[0, 3, 2]], 40), ([0, 40], [40], [[0, -1, 2]], 40), ([0, 40], [49], [[0, 1, 2]], 40),
            ([0, 41], [40], [[0, 1, 2]], 40)):
        bad = SeqBatch(i32(cu), i32(kv), i32(table), max_q=41)
        for call in (lambda: cache.append(k, v, bad, q=q), lambda: cache.read(bad, rows), lambda: cache.attend(q, bad),
                     lambda: cache.attend(q, SeqBatch(i32(cu), i32(kv), i32(table), max_q=1))):
            call()
            with pytest.raises(KlError) as e:
                ctx.sync()
            assert e.value.status == KL_EBOUNDS
    # a token that no row sees may be anywhere
    cache.attend(q[:1], SeqBatch(i32([0, 1]), i32([16]), i32([[0, 99, -5]]), max_q=1))
    ctx.sync()
    rope = RopeTable(64, 30, ctx=ctx)
    out = cache.append(k, v, good, q=q, rope=rope)
    assert (out[30:] == 0).all()
    with pytest.raises(KlError):
        ctx.sync()
    assert one.shape == (1, 4, 64)


def test_refusals(gpu_ctx):
    for args in ((0, 16, 1, 64), (1, 24, 1, 64), (1, 0, 1, 64), (1, 16, 0, 64), (1, 16, 1, 96), (-1, 16, 1, 64)):
        with pytest.raises(KlError):
            Kv4Cache(*args, ctx=gpu_ctx)
    with pytest.raises(KlError):
        RopeTable(64, 0, ctx=gpu_ctx)
    cache = Kv4Cache(4, 16, 2, 64, ctx=gpu_ctx)
    batch = SeqBatch(i32([0, 4]), i32([4]), i32([[0]]), max_q=4)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    bad = [x.float(), x[:, :1], x[..., :32], x.cpu(), x.transpose(1, 2), x[0], x.clone().requires_grad_()]
    for y in bad:
        with pytest.raises(ValueError):
            cache.append(y, x, batch)
        with pytest.raises(ValueError):
            cache.append(x, y, batch)
    with pytest.raises(ValueError):
        cache.append(x, x[:3], batch)
    with pytest.raises(ValueError):
        cache.append(x, x, batch, q=x, positions=torch.zeros(4, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):
        cache.append(x, x, batch, q_out=x)
    with pytest.raises(KlError):
        cache.append(x, x, batch, rope=RopeTable(128, 16, ctx=gpu_ctx))
    with pytest.raises(ValueError):
        cache.append(x, x, batch, rope=RopeTable(64, 16, ctx=Context(0)))
    for y in (x.float(), x[..., :32], x.cpu(), x.clone().requires_grad_()):
        with pytest.raises(ValueError):
            cache.attend(y, batch)
        with pytest.raises(ValueError):
            cache.attend(x, batch, out=y)
    with pytest.raises(KlError):
        cache.attend(torch.zeros(4, 3, 64, dtype=torch.bfloat16, device=DEV), batch)  # 3 heads on 2
    with pytest.raises(KlError):
        cache.attend(x, batch, window=-1)
    with pytest.raises(KlError):
        cache.attend(x, batch, scale=math.nan)
    with pytest.raises(ValueError):
        cache.read(batch, -1)
    with torch.no_grad():
        cache.attend(x.clone().requires_grad_(), batch)
    empty = SeqBatch(i32([0]), i32([]), torch.zeros(0, 1, dtype=torch.int32, device=DEV), max_q=0)
    assert cache.attend(x, empty, out=x.clone()).shape == x.shape
    assert cache.attend(x[:0], batch).shape == (0, 2, 64)
    assert cache.append(x[:0], x[:0], batch, q=x[:0]).shape == (0, 2, 64)
    gpu_ctx.sync()


def test_handles_outlive_their_context():
    """A garbage collector may take the context before what was made with it."""
    ctx = Context(0)
    cache, rope = Kv4Cache(2, 16, 1, 64, ctx=ctx), RopeTable(64, 8, ctx=ctx)
    lib = ctx.lib
    ctx.close()
    assert lib.kl_kv4_destroy(cache.h) == 0 and lib.kl_rope_destroy(rope.h) == 0
    cache.h = rope.h = None


@pytest.mark.parametrize("heads,kv_heads,tokens", [(1, 1, 700), (3, 1, 5000), (60, 20, 300), (60, 20, 2), (128, 128, 40)])
def test_append_head_counts(gpu_ctx, heads, kv_heads, tokens):
    """Few and many heads on few and many tokens: every way of dealing them to the machine."""
    for dim in (64, 128):
        batch, pages = make_batch([tokens], [tokens], 16)
        cache = Kv4Cache(pages, 16, kv_heads, dim, ctx=gpu_ctx)
        q, k, v = (randn(tokens, h, dim, seed=s) for h, s in ((heads, 1), (kv_heads, 2), (kv_heads, 3)))
        assert torch.equal(cache.append(k, v, batch, q=q), q)
        got_k, got_v = cache.read(batch, tokens)
        assert torch.equal(got_k, R.held(k).float().bfloat16())
        assert torch.equal(got_v, R.held(v).float().bfloat16())


def test_rows_in_front_of_the_first_sequence(gpu_ctx):
    """cu_q that starts at 3: the rows before it belong to nobody, and nothing of theirs is written."""
    batch, pages = make_batch([6], [6], 16)
    cache = Kv4Cache(pages, 16, 2, 64, ctx=gpu_ctx)
    k, v = randn(6, 2, 64, seed=1), randn(6, 2, 64, seed=2)
    cache.append(k, v, batch)
    late = SeqBatch(i32([3, 5]), i32([8]), batch.page_table, max_q=2)
    k2, v2, q2 = randn(6, 2, 64, seed=3), randn(6, 2, 64, seed=4), randn(6, 4, 64, seed=5)
    q_out = torch.full_like(q2, 7.0)
    cache.append(k2, v2, late, q=q2, q_out=q_out)
    assert (q_out[:3] == 7).all() and (q_out[5] == 7).all() and torch.equal(q_out[3:5], q2[3:5])
    every = SeqBatch(i32([0, 8]), i32([8]), batch.page_table, max_q=8)
    got, _ = cache.read(every, 8)
    assert torch.equal(got, R.held(torch.cat([k, k2[3:5]])).float().bfloat16())
    out = cache.attend(q2, late, out=torch.full_like(q2, 7.0))
    assert (out[:3] == 7).all() and (out[5] == 7).all()


def test_many_empty_sequences_between(gpu_ctx):
    """Tokens whose sequences lie far apart in the batch, with thousands of empty ones between."""
    n = 9000
    q_len = [0] * n
    for b, x in ((0, 2), (1, 1), (4500, 5), (4504, 1), (8999, 3)):
        q_len[b] = x
    kv_len = [x if x else 0 for x in q_len]
    batch, pages = make_batch(q_len, kv_len, 16)
    t = sum(q_len)
    cache = Kv4Cache(pages, 16, 8, 64, ctx=gpu_ctx)
    k, v = randn(t, 8, 64, seed=1), randn(t, 8, 64, seed=2)
    cache.append(k, v, batch)
    got_k, got_v = cache.read(batch, t)
    assert torch.equal(got_k, R.held(k).float().bfloat16()) and torch.equal(got_v, R.held(v).float().bfloat16())
