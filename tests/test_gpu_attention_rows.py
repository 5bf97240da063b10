"""Attention for many rows: the cases of test_gpu_attention.py once more, with
hints and tables so wide that the calls take the tensor-core kernel with the
keys in chunks, and cases whose blocks are many enough for whole rows."""

import pytest
import torch

import attention_ref as R
import test_gpu_attention as base
from klearu_b200.attention import Kv4Cache, SeqBatch
from test_gpu_attention import DEV, check_attend, filled, i32, randn

pytestmark = pytest.mark.gpu


def wide(cu_q, kv_len, page_table, max_q=None, max_kv=None):
    """The batch with a page table for 65536 tokens and hints to match; what lies behind the sequences is never read."""
    n, cols = page_table.shape
    table = torch.full((n, max(cols, 4096)), -7, dtype=torch.int32, device=DEV)
    table[:, :cols] = page_table
    return SeqBatch(cu_q, kv_len, table, max_q=max(1, int(cu_q[-1])), max_kv=65536)


@pytest.fixture
def many(monkeypatch):
    monkeypatch.setattr(base, "SeqBatch", wide)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,page,window", [(4, 4, 16, 0), (6, 2, 48, 0), (14, 2, 112, 300), (8, 1, 64, 1),
                                                        (16, 2, 32, 129)])
@pytest.mark.parametrize("q_len,kv_len", [([60, 37, 41], [60, 500, 1000]), ([300, 1, 0, 129], [700, 1, 5, 129]), ([130, 129], [9000, 130])])
def test_rows_and_chunks(gpu_ctx, many, dim, heads, kv_heads, page, window, q_len, kv_len):
    base.test_several_tokens(gpu_ctx, dim, heads, kv_heads, page, window, q_len, kv_len)


@pytest.mark.parametrize("q_len,kv_len", [([70, 1, 0, 9], [0, 0, 0, 4]), ([200, 5], [30, 0])])
def test_rows_that_see_nothing(gpu_ctx, many, q_len, kv_len):
    base.test_rows_that_see_nothing(gpu_ctx, q_len, kv_len)


@pytest.mark.parametrize("dim", [64, 128])
def test_nan_in_unseen_tokens(gpu_ctx, many, dim):
    base.test_nan_in_unseen_tokens(gpu_ctx, [70, 90], dim)


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e18])
def test_value_sizes(gpu_ctx, many, size):
    """Values of any size, constant vectors among them, and a score scale that makes one key win."""
    kv_len, q_len = [1000, 140], [70, 120]
    n = sum(kv_len)
    v = (randn(n, 2, 64, seed=2).float() * size).bfloat16()
    v[7] = size
    v[300:500] = 0  # steps of 128 keys without a value, and one with values of another size
    v[640:700] = v[640:700] * 1e-3
    k = randn(n, 2, 64, seed=1)
    k[5] = 0.25
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 16, 2, 64, q_len=q_len, k=k, v=v)
    q = randn(sum(q_len), 4, 64, seed=9)
    for scale in (0.125, 4.0, 0.0, -0.2):
        check_attend(cache.attend(q, batch, scale=scale), q, batch, hk, hv, q_len, kv_len, scale=scale)


@pytest.mark.parametrize("size", [1e-20, 1e-3, 300.0, 1e15])
def test_query_and_key_sizes(gpu_ctx, many, size):
    """Queries of one size and keys of its inverse: ordinary scores from extreme factors."""
    kv_len, q_len = [700], [66]
    k = (randn(700, 2, 128, seed=1).float() / size).bfloat16()
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 16, 2, 128, q_len=q_len, k=k)
    q = (randn(66, 8, 128, seed=9).float() * size).bfloat16()
    check_attend(cache.attend(q, batch), q, batch, hk, hv, q_len, kv_len)


def test_nan_queries(gpu_ctx, many):
    cache, batch, hk, hv = filled(gpu_ctx, [900], 16, 2, 64, q_len=[80])
    q = randn(80, 4, 64, seed=9)
    q[3, 1, 5], q[60, 2, 0] = float("nan"), float("inf")
    out = cache.attend(q, batch)
    assert torch.isnan(out[3, 1]).all() and torch.isnan(out[60, 2]).all()
    bad = torch.isnan(out).any(-1)
    assert bad.sum() == 2
    q[3, 1], q[60, 2] = 0, 0
    want = cache.attend(q, batch)
    assert torch.equal(out[~bad], want[~bad])
    check_attend(want, q, batch, hk, hv, [80], [900])


def test_more_sequences_than_a_grid_is_high(gpu_ctx):
    """70000 sequences of one token, every fifth without any; a token that sees only itself gives its value."""
    n = 70000
    kv = [0 if i % 5 == 0 else 1 for i in range(n)]
    table = torch.randperm(n, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(n, 1).to(DEV)
    batch = SeqBatch(torch.arange(n + 1, dtype=torch.int32, device=DEV), i32(kv), table, max_q=60, max_kv=128)
    cache = Kv4Cache(n, 128, 1, 64, ctx=gpu_ctx)
    q, k, v = randn(n, 2, 64, seed=1), randn(n, 1, 64, seed=2), randn(n, 1, 64, seed=3)
    cache.append(k, v, batch)
    out = cache.attend(q, batch)
    want = torch.where(torch.tensor(kv, device=DEV)[:, None, None] > 0, R.held(v), 0.0)
    # a value and the output are rounded once each
    assert ((out.double() - want).abs() <= 2 * R.HALF * 1.01 * (want.abs() + (v.double().abs().amax(-1, keepdim=True) / 7))).all()


def test_strided_queries_and_outputs(gpu_ctx, many):
    base.test_strided_queries_and_outputs(gpu_ctx, [150, 40])


def test_same_bits_every_time(gpu_ctx, many):
    base.test_same_bits_every_time(gpu_ctx, [40, 3, 70])


def test_offsets_beyond_32_bits(gpu_ctx, many):
    base.test_offsets_beyond_32_bits(gpu_ctx, [300, 70])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads,window,q_len,kv_len", [
    (32, 8, 0, [150, 300, 201, 1], [500, 300, 201, 450]), (16, 8, 0, [1300, 900], [1300, 1005]), (16, 8, 200, [1300, 900], [1300, 1005]),
    (8, 8, 1, [600] * 5, [600] * 5), (40, 4, 0, [700, 500], [100, 1400])])
def test_whole_rows(gpu_ctx, dim, heads, kv_heads, window, q_len, kv_len):
    """So many rows that no keys are shared out; the last: 600 rows that see nothing, as padding in front."""
    cache, batch, hk, hv = filled(gpu_ctx, kv_len, 48, kv_heads, dim, q_len=q_len)
    q = randn(sum(q_len), heads, dim, seed=9)
    out = cache.attend(q, batch, window=window)
    check_attend(out, q, batch, hk, hv, q_len, kv_len, window)
    assert torch.equal(out, cache.attend(q, batch, window=window))
    # rows strided and behind the last sequence, an output left alone there
    pad = torch.full((sum(q_len) + 3, heads + 1, dim + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    qs, o = pad.clone()[:, 1:, 8:], pad[:, :heads, :dim]
    qs[: sum(q_len)] = q
    cache.attend(qs, batch, window=window, out=o)
    assert torch.equal(o[: sum(q_len)], out)
    assert (pad[-3:] == 7).all() and (pad[:, heads:] == 7).all() and (pad[..., dim:] == 7).all()


def test_values_that_are_not_finite(gpu_ctx):
    """Whole rows: a token whose vectors are not finite makes NaN of the rows that see it, and of no others."""
    n, heads, kv_heads, dim = 1200, 16, 8, 128
    k, v = randn(n, kv_heads, dim, seed=1), randn(n, kv_heads, dim, seed=2)
    k[700, 3, 5], v[900, 5, 9] = float("nan"), float("inf")
    cache, batch, _, _ = filled(gpu_ctx, [n], 16, kv_heads, dim, k=k, v=v)
    q = randn(n, heads, dim, seed=3)
    out = cache.attend(q, batch)
    bad = torch.isnan(out).any(-1)
    want = torch.zeros_like(bad)
    want[700:, 6:8] = True
    want[900:, 10:12] = True
    assert torch.equal(bad, want)
    assert torch.isnan(out[want]).all()
