"""Attention within the roundings that its kernels make (attention_bound.py): ordinary inputs, single keys counted,
values whose size changes along a sequence, tokens that a row does not see.  ``few`` and ``many`` are the kernels for few
and for many rows, chosen by the hints; ``many`` takes the keys in chunks of a step, ``whole`` all of a row's in one."""

import math

import pytest
import torch

import attention_bound as B
import attention_ref as R
from klearu_b200.attention import Kv4Cache, SeqBatch
from test_gpu_attention import DEV, i32, make_batch, randn

pytestmark = pytest.mark.gpu
KERNELS = ["few", "many", "whole"]


def batch_for(kernel, q_len, kv_len, page):
    """A batch whose hints choose the kernel, and its number of pages."""
    batch, pages = make_batch(q_len, kv_len, page)
    if kernel == "few":
        return SeqBatch(batch.cu_q, batch.kv_len, batch.page_table, max_q=1, max_kv=max(kv_len)), pages
    if kernel == "whole":
        return SeqBatch(batch.cu_q, batch.kv_len, batch.page_table, max_q=2**30, max_kv=max(kv_len)), pages
    n, cols = batch.page_table.shape
    table = torch.full((n, max(cols, 65536 // page)), -7, dtype=torch.int32, device=DEV)
    table[:, :cols] = batch.page_table
    return SeqBatch(batch.cu_q, batch.kv_len, table, max_q=max(200, sum(q_len)), max_kv=65536), pages


def attend(kernel, cache, q, batch, **kw):
    """``whole``: behind so many rows of no sequence that chunks of the keys would need more workspace than a call takes."""
    if kernel != "whole":
        return cache.attend(q, batch, **kw)
    t, heads, dim = q.shape
    rows = torch.zeros(t + 2**28 // (4 * heads * (dim + 2)), heads, dim, dtype=q.dtype, device=DEV)
    rows[:t] = q
    out = cache.attend(rows, batch, out=torch.full_like(rows, 7.0), **kw)
    assert (out[t:] == 7).all()
    return out[:t].clone()


def run(ctx, kernel, q, k, v, q_len, kv_len, page=16, window=0, scale=None, **kw):
    """Outputs for a cache that holds k and v, and the values that it holds."""
    batch, pages = batch_for(kernel, q_len, kv_len, page)
    cache = Kv4Cache(pages, page, k.shape[1], k.shape[2], ctx=ctx)
    every = SeqBatch(i32([sum(kv_len[:b]) for b in range(len(kv_len) + 1)]), batch.kv_len, batch.page_table, max_q=max(kv_len))
    cache.append(k, v, every)
    out = attend(kernel, cache, q, batch, window=window, scale=scale)
    hk, hv = R.held(k), R.held(v)
    B.check(out, q, hk, hv, q_len, kv_len, window, scale, **kw)
    return out


def inputs(q_len, kv_len, heads, kv_heads, dim, seed=0):
    n = sum(kv_len)
    k = randn(n, kv_heads, dim, seed=seed + 1) * 1.5 + randn(kv_heads, dim, seed=seed + 2)
    return randn(sum(q_len), heads, dim, seed=seed + 4) * 2, k, randn(n, kv_heads, dim, seed=seed + 3)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,page,window", [(4, 4, 16, 0), (6, 2, 48, 0), (14, 2, 112, 300), (8, 1, 64, 33)])
@pytest.mark.parametrize("q_len,kv_len", [([1], [1]), ([1, 1, 3], [9001, 17, 500]), ([41], [1000]), ([70, 130], [300, 5000])])
def test_ordinary_inputs(gpu_ctx, kernel, dim, heads, kv_heads, page, window, q_len, kv_len):
    q, k, v = inputs(q_len, kv_len, heads, kv_heads, dim)
    run(gpu_ctx, kernel, q, k, v, q_len, kv_len, page, window)


def test_whole_rows(gpu_ctx):
    """Blocks that take several tiles of rows, one after another."""
    q_len, kv_len = [1300, 900], [1300, 1005]
    for window in (0, 200):
        q, k, v = inputs(q_len, kv_len, 16, 8, 128)
        run(gpu_ctx, "many", q, k, v, q_len, kv_len, 48, window)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("n,rows,window", [(131071, 1, 0), (131071, 65, 0), (131071, 3, 100000), (5000, 70, 0), (9001, 1, 1234), (1000, 41, 130)])
def test_every_key_counts_once(gpu_ctx, kernel, n, rows, window):
    """Scores of zero, so that each key that a row sees counts alike, and values at the borders of what the rows see,
    each alone in its dimension: held exactly, seen or not, with nothing that could hide a missing or an extra key."""
    heads, dim, one = 2, 64, 15 * 256.0
    first = n - rows
    at = sorted({j for r in (0, rows // 2, rows - 1) for p in (first + r,) for j in
                 (0, 1, p, p + 1, *((p - window, p - window + 1) if window else ())) if 0 <= j < n})
    assert len(at) <= dim - 1
    v = torch.zeros(n, 1, dim, dtype=torch.bfloat16, device=DEV)
    for d, j in enumerate(at):
        v[j, 0, d] = one
    k, q = randn(n, 1, dim, seed=1), randn(rows, heads, dim, seed=2)
    batch, pages = batch_for(kernel, [rows], [n], 1024)
    cache = Kv4Cache(pages, 1024, 1, dim, ctx=gpu_ctx)
    cache.append(k, v, SeqBatch(i32([0, n]), batch.kv_len, batch.page_table, max_q=n))
    out = attend(kernel, cache, q, batch, window=window, scale=0.0).double()
    for r in range(rows):
        p = first + r
        low = max(0, p - window + 1) if window else 0
        for d, j in enumerate(at):
            want = one / (p + 1 - low) if low <= j <= p else 0.0
            # the count is exact, the probability a power of two: the output's rounding, and a sum's and quotient's
            assert ((out[r, :, d] - want).abs() <= want * (B.BF16 + 1e-5)).all(), (r, j)


# ---------------------------------------------------------------------------
# values whose size changes along the sequence
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("size", [1e-1, 1e-2, 1e-3, 1e-4, 1e-9, 1e4])
@pytest.mark.parametrize("zeros,n,rows", [(128, 600, 70), (500, 1500, 80), (300, 700, 3)])
def test_zero_values_first(gpu_ctx, kernel, size, zeros, n, rows):
    """Tokens whose value is zero in front (a cache is zeros before it is written), then values of any size."""
    q, k, v = inputs([rows], [n], 8, 2, 128)
    v = (v.float() * size).bfloat16()
    v[:zeros] = 0
    run(gpu_ctx, kernel, q, k, v, [rows], [n])


def test_zero_values_first_whole_rows(gpu_ctx):
    """Blocks that take several tiles of rows: a scale must not come from the tile before."""
    q_len, kv_len = [1300, 900, 40], [1300, 1005, 300]
    for size in (1e-3, 1e3):
        q, k, v = inputs(q_len, kv_len, 16, 8, 64)
        v[1300:] = (v[1300:].float() * size).bfloat16()
        v[:256] = v[1300:1556] = v[2305:2433] = 0
        run(gpu_ctx, "many", q, k, v, q_len, kv_len, rms=False)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("big,size", [(1e6, 1.0), (1e6, 1e-3), (1e10, 1.0), (1e2, 1e-4)])
@pytest.mark.parametrize("keys", [1, 16, 128, 300])
def test_large_values_that_hardly_count(gpu_ctx, kernel, big, size, keys):
    """The first keys' scores are 60 and more below the others', and their values far larger."""
    n, rows = 900, 70
    q, k, v = inputs([rows], [n], 8, 2, 64)
    v = (v.float() * size).bfloat16()
    q[..., 0] = 32.0
    k[:, :, 0] = 0.0
    k[:keys] *= 0.01
    k[:keys, :, 0] = -24.0
    v[:keys] = (v[:keys].float() * (big / size)).bfloat16()
    run(gpu_ctx, kernel, q, k, v, [rows], [n])


@pytest.mark.parametrize("kernel", KERNELS)
def test_sizes_that_come_and_go(gpu_ctx, kernel):
    """Values that grow and shrink by powers of ten from stretch to stretch of the sequence, zeros between."""
    n, rows = 2000, 90
    q, k, v = inputs([rows], [n], 4, 2, 64)
    size = torch.tensor([1e-6, 1e3, 0.0, 1e-12, 1.0, 1e9, 0.0, 1e-3, 30.0, 1e-9], device=DEV).repeat_interleave(200)
    v = (v.float() * size[:, None, None]).bfloat16()
    run(gpu_ctx, kernel, q, k, v, [rows], [n])
    # rows that see only the first of them
    for kl in (150, 390, 780, 950):
        run(gpu_ctx, kernel, q, k[:kl], v[:kl], [rows], [kl], rms=False)


@pytest.mark.parametrize("kernel", KERNELS)
def test_a_long_flat_tail(gpu_ctx, kernel):
    """One key that wins by 2^25.3 and 131070 whose share of the result is still 0.3%: none of it may be lost."""
    n, rows, dim = 131071, 40, 64
    q = torch.zeros(rows, 2, dim, dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 1.0
    k = torch.zeros(n, 1, dim, dtype=torch.bfloat16, device=DEV)
    k[0, 0, 0] = 25.3 * 0.6931471805599453
    v = torch.zeros(n, 1, dim, dtype=torch.bfloat16, device=DEV)
    v[1:, 0, 1] = 15.0
    v[0, 0, 2] = 15.0
    batch, pages = batch_for(kernel, [rows], [n], 1024)
    cache = Kv4Cache(pages, 1024, 1, dim, ctx=gpu_ctx)
    cache.append(k, v, SeqBatch(i32([0, n]), batch.kv_len, batch.page_table, max_q=n))
    out = attend(kernel, cache, q, batch, scale=1.0).double()
    top = float(torch.exp(R.held(k)[0, 0, 0]))
    # all of the tail's probabilities are rounded alike: f16 has steps of 2^-24 from 0 on, and the largest probability
    # stands at 2^6 or above, so half a step is 2^-31 of it
    tail = 2.0**-31 * top
    for r in range(rows):
        others = n - rows + r
        total = top + others
        assert ((out[r, :, 1] / (15 * others / total) - 1).abs() <= B.BF16 + tail + 1e-3).all(), r
        assert ((out[r, :, 2] / (15 * top / total) - 1).abs() <= B.BF16 + B.F16 + 1e-3).all(), r


# ---------------------------------------------------------------------------
# tokens that a row does not see
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("garbage", [1e6, 1e10, 1e30])
def test_stale_tokens_behind_the_sequence(gpu_ctx, kernel, garbage):
    """Another use of the page left large finite keys and values behind the sequence's end."""
    dim, page, rows = 128, 128, 70
    table = torch.full((1, 512 if kernel == "many" else 2), -7, dtype=torch.int32, device=DEV)
    table[0, 0], table[0, 1] = 1, 0
    for n in (90, 129, 250):
        k, v = randn(256, 2, dim, seed=1), randn(256, 2, dim, seed=2)
        k[n:] = (k[n:].float() * garbage).bfloat16()
        v[n:] = (v[n:].float() * garbage).bfloat16()
        cache = Kv4Cache(2, page, 2, dim, ctx=gpu_ctx)
        cache.append(k, v, SeqBatch(i32([0, 256]), i32([256]), table, max_q=256))
        now = SeqBatch(i32([0, rows]), i32([n]), table, max_q={"few": 1, "many": 200, "whole": 2**30}[kernel], max_kv=65536)
        q = randn(rows, 8, dim, seed=3)
        B.check(attend(kernel, cache, q, now), q, R.held(k[:n]), R.held(v[:n]), [rows], [n], rms=False)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("large", [1e5, 1e8, 1e30])
@pytest.mark.parametrize("window", [0, 150])
def test_large_tokens_that_some_rows_do_not_see(gpu_ctx, kernel, large, window):
    """Later tokens for the rows before them, and tokens in front of a window: large values there change nothing."""
    n, rows = 500, 140
    q, k, v = inputs([rows], [n], 4, 2, 64)
    at = [3, 230, 419, n - 20, n - 1]
    for j in at:
        v[j] = (v[j].float() * large).bfloat16()
    out = run(gpu_ctx, kernel, q, k, v, [rows], [n], window=window, rms=False)
    if not window:
        return
    # rows 20 to 55 (tokens 380 to 415) see tokens from 231 on and none of the large ones: small errors of their own
    want, _ = B.attend(q[20:56], R.held(k)[:416], R.held(v)[:416], 380, window, 64**-0.5)
    off = out[20:56].double() - want
    assert float(off.square().mean().sqrt()) <= B.RMS * float(want.square().mean().sqrt())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("large", [1e5, 1e8, 1e20])
def test_large_keys_that_some_rows_do_not_see(gpu_ctx, kernel, large):
    n, rows = 500, 140
    q, k, v = inputs([rows], [n], 4, 2, 64)
    for j in (3, 430, n - 1):
        k[j] = (k[j].float() * large).bfloat16()
    # tokens 380 to 429: none of the large keys but the first, which a window of 300 leaves out
    run_rows, first = 50, 380
    batch, pages = batch_for(kernel, [rows], [n], 16)
    cache = Kv4Cache(pages, 16, 2, 64, ctx=gpu_ctx)
    cache.append(k, v, SeqBatch(i32([0, n]), batch.kv_len, batch.page_table, max_q=n))
    out = attend(kernel, cache, q, batch, window=300)
    i = first - (n - rows)
    want, tol = B.attend(q[i : i + run_rows], R.held(k)[:430], R.held(v)[:430], first, 300, 64**-0.5)
    off = (out[i : i + run_rows].double() - want).abs()
    assert float((off / tol).max()) <= 1.0
    assert float(off.square().mean().sqrt()) <= B.RMS * float(want.square().mean().sqrt())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("window", [2**40, 2**31 - 1, 2**31 - 2, 10**6])
@pytest.mark.parametrize("q_len,kv_len", [([9], [4]), ([300], [30]), ([70, 9], [3, 900])])
def test_padding_and_a_window_that_reaches_all(gpu_ctx, kernel, window, q_len, kv_len):
    """Rows in front of the first token beside rows that see keys, and a window as large as a number gets."""
    q, k, v = inputs(q_len, kv_len, 4, 2, 64)
    out = run(gpu_ctx, kernel, q, k, v, q_len, kv_len, window=window, rms=False)
    assert torch.equal(out, run(gpu_ctx, kernel, q, k, v, q_len, kv_len, rms=False))


@pytest.mark.parametrize("size", [2.0**114, 2.0**117, 2.0**125])
def test_largest_queries(gpu_ctx, size):
    """Queries up to the type's end and keys so small that the scores are ordinary."""
    for kernel, rows in (("few", 3), ("many", 70), ("whole", 70)):
        q, k, v = inputs([rows], [300], 4, 2, 64)
        q = (q.clamp(-3, 3).double() * size).bfloat16()
        k = (k.double() / size).bfloat16()
        run(gpu_ctx, kernel, q, k, v, [rows], [300])


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("size,spread", [(1e5, 1.0), (1e7, 1.0), (3e8, 1.0), (1e12, 1.0), (1e8, 1e8)])
def test_large_scores(gpu_ctx, kernel, size, spread):
    """Scores far beyond the range of the exponential: the key that wins by far gives the output, and nothing passes f16."""
    rows, n = 90, 400
    q, k, v = inputs([rows], [n], 4, 2, 64)
    k = (k.float() * size * spread ** torch.linspace(-1, 0, n, device=DEV)[torch.randperm(n, device=DEV)][:, None, None]).bfloat16()
    batch, pages = batch_for(kernel, [rows], [n], 16)
    cache = Kv4Cache(pages, 16, 2, 64, ctx=gpu_ctx)
    cache.append(k, v, SeqBatch(i32([0, n]), batch.kv_len, batch.page_table, max_q=n))
    out = attend(kernel, cache, q, batch).double()
    assert torch.isfinite(out).all()
    hk, hv = R.held(k), R.held(v)
    for h in range(4):
        x = q[:, h].double() @ hk[:, h // 2].T / 8
        at = torch.arange(n, device=DEV)[None] > torch.arange(n - rows, n, device=DEV)[:, None]
        two = x.masked_fill(at, -float("inf")).topk(2, -1)
        # a score is within 64 (2^-11 + 2^-20) |q| |K| / 8 of its own; where the second is further off it counts for nothing
        clear = two.values[:, 0] - two.values[:, 1] > 30 + 2 * (B.F16 + 2.0**-20) / 8 * (q[:, h].double().abs() @ hk[:, h // 2].abs().T).amax(-1)
        want = hv[two.indices[:, 0], h // 2]
        tol = (B.BF16 + 2 * B.F16) * want.abs() + 3 * B.F16 * hv[two.indices[:, 0], h // 2].abs().amax(-1, keepdim=True)
        assert clear.sum() > rows // 3 and ((out[:, h] - want).abs() <= tol)[clear].all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("first,last", [(256, 384), (300, 428), (0, 128)])
@pytest.mark.parametrize("big", [1e7, 1e10])
def test_large_values_count_by_their_probabilities(gpu_ctx, kernel, first, last, big):
    """A stretch of keys whose probabilities are about 1 / big of the others' and whose values are big times theirs: both
    halves of the result count."""
    n, rows = 900, 70
    q, k, v = inputs([rows], [n], 4, 2, 64)
    q *= 0.25
    q[..., 0] = 32.0
    k[:, :, 0] = 0.0
    k[first:last, :, 0] = -math.log(big) / (32.0 * 64**-0.5)
    v[first:last] = (v[first:last].float() * big).bfloat16()
    run(gpu_ctx, kernel, q, k, v, [rows], [n])
