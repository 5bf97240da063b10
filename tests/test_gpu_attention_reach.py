"""What the calls of the attention half do at the edges of their arguments: lengths beyond the table, streams other than
the context's, tiny rows, tangents."""

import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import attention_bound as B
import attention_ref as R
from klearu_b200._lib import KL_EBOUNDS, KlError
from klearu_b200.attention import Kv4Cache, RopeTable, SeqBatch
from klearu_b200.core import Context
from klearu_b200.dejavu import FfnStack, SparseMlp, SparsityPredictor
from klearu_b200.quant import Q8Linear, add_rms_norm_q8, quantize_rows_q8
from test_gpu_attention import DEV, i32, randn
from test_gpu_decoder_layer import Layer
from test_gpu_q8 import check_norm

pytestmark = pytest.mark.gpu


def reported(ctx):
    with pytest.raises(KlError) as e:
        ctx.sync()
    return e.value.status == KL_EBOUNDS


# ---------------------------------------------------------------------------
# lengths and rows beyond what the call's arrays hold
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("q_len", [1, 5, 60])
def test_tokens_beyond_the_table(q_len):
    """A sequence longer than its row of the table: its tokens keep their numbers, those that have a page are written and
    attended to, the others are not, and nothing of the tokens before them changes.  60: the kernel for many rows."""
    ctx = Context(0)
    page, heads, kv_heads, dim, held = 1024, 32, 8, 64, 8192
    n = held + 10  # ten tokens more than the table has room for
    table = i32([[5, 2, 7, 0, 1, 6, 3, 4]])
    cache = Kv4Cache(8, page, kv_heads, dim, ctx=ctx)
    k, v = randn(n, kv_heads, dim, seed=1), randn(n, kv_heads, dim, seed=2)
    old = SeqBatch(i32([0, held]), i32([held]), table, max_q=held)
    cache.append(k[:held], v[:held], old)
    ctx.sync()
    first = n - q_len
    new = SeqBatch(i32([0, q_len]), i32([n]), table, max_q=q_len)
    k2, v2, q = randn(q_len, kv_heads, dim, seed=3), randn(q_len, kv_heads, dim, seed=4), randn(q_len, heads, dim, seed=5)
    rope = RopeTable(dim, 16384, ctx=ctx)
    turned = cache.append(k2, v2, new, q=q, rope=rope)
    assert reported(ctx)
    pos = torch.arange(first, n, device=DEV)
    want = R.rotate(q, pos, rope.inv_freq, False)
    assert ((turned.double() - want).abs() <= R.HALF * want.abs() + 1e-5).all()
    fit = max(0, held - first)  # of the new tokens
    hk, hv = R.held(k[:held]), R.held(v[:held])
    gk, gv = cache.read(old, held)
    assert torch.equal(gk[: held - fit], hk[: held - fit].float().bfloat16())
    assert torch.equal(gv[: held - fit], hv[: held - fit].float().bfloat16())
    assert torch.equal(gv[held - fit :], R.held(v2[:fit]).float().bfloat16())
    rk, rv = cache.read(new, q_len)
    assert reported(ctx)
    assert torch.equal(rv[:fit], gv[held - fit :]) and torch.equal(rk[:fit], gk[held - fit :])
    assert (rk[fit:] == 0).all() and (rv[fit:] == 0).all()
    # every row sees the tokens up to its own that there are; with a window the last of its own numbers
    for window in (0, 25, 8):
        out = cache.attend(q, new, window=window)
        assert reported(ctx)
        for r in range(q_len):
            p = first + r
            low, high = max(0, p - window + 1) if window else 0, min(p + 1, held)
            if low >= high:
                assert (out[r] == 0).all()
                continue
            want, _ = B.attend(q[r : r + 1], gk[low:high].double(), gv[low:high].double(), high - low - 1, 0, dim**-0.5)
            # read() rounds the held keys and values to bf16: 2^-7 / sqrt(12) of each, and a score's error from its keys
            # (scale sqrt(sum q^2 K^2) of that, about 2.5) moves the output as much again
            size = float(want.square().mean().sqrt())
            assert float((out[r].double() - want[0]).square().mean().sqrt()) <= 0.01 * size + 1e-4, (window, r)


@pytest.mark.parametrize("rows", [5, 60])
def test_rows_beyond_the_tensor(rows):
    """A batch with more rows than the call's tensors: the rows that there are keep their tokens' numbers."""
    ctx = Context(0)
    page, heads, kv_heads, dim, n, lost = 1024, 32, 8, 64, 8000, 7
    table = i32([list(range(8))])
    cache = Kv4Cache(8, page, kv_heads, dim, ctx=ctx)
    k, v = randn(n, kv_heads, dim, seed=1), randn(n, kv_heads, dim, seed=2)
    cache.append(k, v, SeqBatch(i32([0, n]), i32([n]), table, max_q=n))
    ctx.sync()
    first = n - rows - lost  # the call says rows + 7 new tokens and has only so many rows
    batch = SeqBatch(i32([0, rows + lost]), i32([n]), table, max_q=rows + lost)
    k2, v2, q = randn(rows, kv_heads, dim, seed=3), randn(rows, kv_heads, dim, seed=4), randn(rows, heads, dim, seed=5)
    cache.append(k2, v2, batch)
    assert reported(ctx)
    k[first : first + rows], v[first : first + rows] = k2, v2
    every = SeqBatch(i32([0, n]), i32([n]), table, max_q=n)
    gk, gv = cache.read(every, n)
    assert torch.equal(gk, R.held(k).float().bfloat16()) and torch.equal(gv, R.held(v).float().bfloat16())
    out = cache.attend(q, batch)
    assert reported(ctx)
    want, tol = B.attend(q, R.held(k), R.held(v), first, 0, dim**-0.5)
    assert ((out.double() - want).abs() <= tol).all()


def test_sequences_without_a_row_in_the_tensor():
    """A batch of which a whole sequence lies behind the call's tensors: reported by every call, the others served."""
    ctx = Context(0)
    cache = Kv4Cache(8, 16, 2, 64, ctx=ctx)
    table = i32([[0, 1], [2, 3], [4, 5]])
    k, v, q = randn(5, 2, 64, seed=1), randn(5, 2, 64, seed=2), randn(5, 4, 64, seed=3)
    batch = SeqBatch(i32([0, 2, 5, 9]), i32([2, 3, 4]), table, max_q=4)
    assert torch.equal(cache.append(k, v, batch, q=q), q)
    assert reported(ctx)
    gk, _ = cache.read(batch, 5)
    assert reported(ctx) and torch.equal(gk, R.held(k).float().bfloat16())
    cache.attend(q, batch)
    assert reported(ctx)
    ctx.sync()


# ---------------------------------------------------------------------------
# streams
# ---------------------------------------------------------------------------
def test_errors_of_another_stream_are_reported():
    """A call that runs on a stream which is not the context's: the next sync waits for it and reports what it saw."""
    ctx = Context(0)
    cache = Kv4Cache(3, 16, 2, 64, ctx=ctx)
    bad = SeqBatch(i32([0, 40]), i32([40]), i32([[0, 3, 2]]), max_q=40)
    cache.read(SeqBatch(i32([0, 40]), i32([40]), i32([[0, 1, 2]]), max_q=40), 40)
    ctx.sync()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # about 50 ms of a busy stream in front
        cache.read(bad, 40)
    assert reported(ctx)
    ctx.sync()  # and once only
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.read(bad, 40)
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        graph.replay()
    assert reported(ctx)


def ffn(ctx, h=192, layers=1):
    rng = np.random.default_rng(3)
    w = lambda *s: (rng.standard_normal(s) * 0.05).astype(np.float32)  # noqa: E731
    pred = [SparsityPredictor(w(40, h), w(40), w(256, 40), w(256), ctx=ctx) for _ in range(layers)]
    mlp = [SparseMlp(w(256, h), w(256, h), w(h, 256), ctx=ctx) for _ in range(layers)]
    return FfnStack(pred, mlp, np.ones((layers, h), np.float32), ctx=ctx)


def test_both_halves_of_a_layer_on_another_stream(gpu_ctx):
    """Norm, projection and the MLP stack on torch's current stream, in order, whichever stream the context has."""
    stack = ffn(gpu_ctx)
    w = randn(192, 192, seed=2, dtype=torch.float32) / 14
    back = Q8Linear.from_weights(w, ctx=gpu_ctx)
    norm = torch.ones(192, device=DEV)

    def layer(hidden):
        rows = add_rms_norm_q8(hidden, norm, ctx=gpu_ctx)
        back.forward(rows.codes, rows.scales, out=hidden, accumulate=True)
        stack.decode(hidden, 0.25)
        rows = add_rms_norm_q8(hidden, norm, ctx=gpu_ctx)
        back.forward(rows.codes, rows.scales, out=hidden, accumulate=True)

    start = randn(3, 192, seed=1, dtype=torch.float32)
    want = start.clone()
    for _ in range(3):
        layer(want)
    torch.cuda.synchronize()
    hidden = start.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)  # what is not ordered behind this runs too early
        for _ in range(3):
            layer(hidden)
        got = hidden.clone()
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("tokens", [3, 40])
def test_the_mlp_half_in_a_captured_graph(gpu_ctx, tokens):
    """Captured on another buffer than the one it ran on, replayed before and after larger calls replaced its scratch."""
    stack = ffn(gpu_ctx, layers=2)
    start = randn(tokens, 192, seed=1, dtype=torch.float32)
    want = start.clone()
    for _ in range(3):
        stack.decode(want, 0.25)
    hidden = start.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stack.decode(hidden, 0.25)
    assert torch.equal(hidden, start)  # captured, not run
    graph.replay()
    graph.replay()
    for big in (20, 300):
        stack.decode(randn(big, 192, seed=2, dtype=torch.float32), 0.75)
    junk = [torch.full((1 << 18,), float("nan"), device=DEV) for _ in range(8)]  # what was freed is somebody else's now
    graph.replay()
    assert torch.equal(hidden, want) and len(junk) == 8
    gpu_ctx.sync()


def test_the_stack_beside_larger_calls_of_its_mlp(gpu_ctx):
    """The stack's own graph goes on when a call of one of its MLPs needs more scratch than the graph's."""
    stack, twin = ffn(gpu_ctx, layers=2), ffn(gpu_ctx, layers=2)
    hidden = randn(3, 192, seed=1, dtype=torch.float32)
    want = hidden.clone()
    for step in range(5):
        if step == 3:
            mlp = stack._keep[1][0]
            mlp.forward_sparse(randn(20, 192, seed=2, dtype=torch.float32), torch.arange(256, device=DEV).repeat(20, 1))
            junk = [torch.full((1 << 18,), float("nan"), device=DEV) for _ in range(8)]
        stack.decode(hidden, 0.25)
        twin.decode(want, 0.25)
        assert torch.equal(hidden, want), step
    assert len(junk) == 8


def test_a_whole_layer_in_a_captured_graph(gpu_ctx):
    """Both halves of two layers in one graph, replayed token after token, against calls one by one; hints of the cache's
    whole capacity; a prompt through the same layers between the tokens."""
    def model():
        return [(Layer(gpu_ctx, 2, 640), ffn(gpu_ctx)) for _ in range(2)]

    def step(layers, hidden, batch_of):
        for half, stack in layers:
            half(hidden, batch_of(half))
            stack.decode(hidden, 0.25)

    def prompt(layers, q_len, length, seed):
        hidden = 2 * randn(sum(q_len), Layer.hidden, seed=seed, dtype=torch.float32)
        cu = i32([0, q_len[0], sum(q_len)])
        step(layers, hidden, lambda half: SeqBatch(cu, i32(length), half.table, max_q=max(q_len)))

    mine, twin = model(), model()
    for x in (mine, twin):
        prompt(x, [30, 200], [30, 200], 5)
        first = 2 * randn(2, Layer.hidden, seed=6, dtype=torch.float32)
        step(x, first, lambda half: SeqBatch(i32([0, 1, 2]), i32([31, 201]), half.table, max_q=1))
    kv, cu = i32([32, 202]), i32([0, 1, 2])
    hidden = torch.zeros(2, Layer.hidden, device=DEV)
    graph = torch.cuda.CUDAGraph()
    batches = {half: SeqBatch(cu, kv, half.table, max_q=1) for half, _ in mine}
    with torch.cuda.graph(graph):
        step(mine, hidden, batches.__getitem__)
    for n in range(4):
        start = 2 * randn(2, Layer.hidden, seed=10 + n, dtype=torch.float32)
        hidden.copy_(start)
        graph.replay()
        plain = start.clone()
        step(twin, plain, lambda half: SeqBatch(cu, kv.clone(), half.table, max_q=1))
        assert torch.equal(hidden, plain), n
        kv += 1
        if n == 1:  # 40 and 90 more prompt tokens, whose scratch is larger than the graph's
            for x in (mine, twin):
                prompt(x, [40, 90], [73, 293], 20)
            kv += torch.tensor([40, 90], dtype=torch.int32, device=DEV)
    gpu_ctx.sync()


def test_reading_into_one_given_output(gpu_ctx):
    cache = Kv4Cache(2, 16, 2, 64, ctx=gpu_ctx)
    batch = SeqBatch(i32([0, 9]), i32([9]), i32([[1]]), max_q=9)
    k, v = randn(9, 2, 64, seed=1), randn(9, 2, 64, seed=2)
    cache.append(k, v, batch)
    wide = torch.full((9, 2, 72), 7.0, dtype=torch.bfloat16, device=DEV)
    for name, other in (("k_out", 1), ("v_out", 0)):
        got = cache.read(batch, 9, **{name: wide[..., :64]})
        assert got[1 - other].data_ptr() == wide.data_ptr() and (wide[..., 64:] == 7).all()
        assert torch.equal(got[0], R.held(k).float().bfloat16()) and torch.equal(got[1], R.held(v).float().bfloat16())


def test_a_capture_of_the_mlp_half_that_has_not_run(gpu_ctx):
    """Refused with an error that leaves the capture as it is."""
    stack = ffn(gpu_ctx, layers=2)
    hidden, x = randn(3, 192, seed=1, dtype=torch.float32), torch.zeros(4, device=DEV)
    before = hidden.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        for _ in range(2):
            with pytest.raises(KlError):
                stack.decode(hidden, 0.25)
        x.add_(1)
    graph.replay()
    assert torch.equal(hidden, before) and (x == 2).all()
    stack.decode(hidden, 0.25)
    gpu_ctx.sync()
    assert not torch.equal(hidden, before)


def test_a_context_with_a_stream_of_its_own():
    """What the context's own stream holds and what torch's current stream holds both come before and after the stack."""
    own = torch.cuda.Stream()
    ctx = Context(0, stream=own)
    stack, twin = ffn(ctx), ffn(Context(0))
    start = randn(3, 192, seed=1, dtype=torch.float32)
    want, hidden = start.clone(), torch.zeros_like(start)
    for _ in range(3):
        twin.decode(want, 0.25)
    torch.cuda.synchronize()
    with torch.cuda.stream(own):
        torch.cuda._sleep(50_000_000)
        hidden.copy_(start)
    for _ in range(3):
        stack.decode(hidden, 0.25)  # behind what the context's stream holds
    ctx.sync()
    assert torch.equal(hidden, want)
    with torch.cuda.stream(own):
        torch.cuda._sleep(50_000_000)
        hidden.copy_(start)
    for _ in range(3):
        stack.decode(hidden, 0.25)
    got = hidden.clone()  # on the current stream
    torch.cuda.synchronize()
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# rows of extreme sizes
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cols", [256, 77])
@pytest.mark.parametrize("size", [3e-37, 1e-37, 1e-38, 1e-40, 3e-44])
def test_codes_of_tiny_rows(gpu_ctx, cols, size):
    """Rows so small that 127 over their largest value is no 32-bit number."""
    x = (randn(5, cols, seed=1, dtype=torch.float32).double() * size).float()
    x[1] = 0
    x[2, 3] = size * 40
    x[3, ::2] = 0
    ones = torch.ones(cols, device=DEV)
    r = quantize_rows_q8(x, ctx=gpu_ctx)
    u = x.double()
    top = u.abs().amax(-1, keepdim=True)
    assert torch.equal(r.codes.double(), torch.where(top > 0, (u * 127 / top).round(), 0.0))
    # a scale below the normal numbers has steps of 2^-149
    assert ((r.scales.double() - top[:, 0] / 127).abs() <= 2.0**-149 + 4 * 2.0**-24 * top[:, 0] / 127).all()
    r = add_rms_norm_q8(x, ones, eps=1e-5, ctx=gpu_ctx)
    assert torch.equal(r.codes.double(), torch.where(top > 0, (u * 127 / top).round(), 0.0))
    want = top[:, 0] / (u.square().mean(-1) + 1e-5).sqrt() / 127
    assert ((r.scales.double() - want).abs() <= 2.0**-149 + 8 * 2.0**-24 * want).all()


@pytest.mark.parametrize("cols", [256, 77])
@pytest.mark.parametrize("size", [1e-15, 1e-19, 1e-22, 1e-25, 1e-33])
def test_norm_of_small_rows_without_eps(gpu_ctx, cols, size):
    """The squares of these rows are below the normal 32-bit numbers, their root mean square is not."""
    x = (randn(5, cols, seed=1, dtype=torch.float32).double() * size).float()
    w = 1 + 0.2 * randn(cols, seed=3, dtype=torch.float32)
    check_norm(add_rms_norm_q8(x, w, eps=0.0, ctx=gpu_ctx), x, w, 0.0, True)


@pytest.mark.parametrize("cols", [256, 77])
@pytest.mark.parametrize("x_size,w_size", [(1e-30, 1e-20), (1e-38, 1e-9), (1e-42, 1.0)])
def test_products_below_32_bits(gpu_ctx, cols, x_size, w_size):
    """Values times weights that are all zero in 32 bits: their codes and scale are those of the definition."""
    x = (randn(4, cols, seed=1, dtype=torch.float32).double() * x_size).float()
    x[1] = 0
    w = (1 + 0.2 * randn(cols, seed=3, dtype=torch.float32)) * w_size
    r = add_rms_norm_q8(x, w, eps=0.0, ctx=gpu_ctx)
    u = x.double() * w.double()
    top = u.abs().amax(-1, keepdim=True)
    assert torch.equal(r.codes.double(), torch.where(top > 0, (u * 127 / top).round(), 0.0))
    want = top[:, 0] / x.double().square().mean(-1).sqrt() / 127
    live = [0, 2, 3]
    assert ((r.scales.double() - want).abs() <= (cols / 2 + 6) * 2.0**-24 * want)[live].all()


@pytest.mark.parametrize("cols", [256, 77])
def test_codes_of_large_rows(gpu_ctx, cols):
    """Without a norm the sum of squares is nobody's business: rows whose squares pass 32 bits have codes."""
    x = randn(4, cols, seed=1, dtype=torch.float32) * 1e25
    x[1] *= 1e12
    check_norm(quantize_rows_q8(x, ctx=gpu_ctx), x, torch.ones(cols, device=DEV), 0, False)
    r = add_rms_norm_q8(x, torch.ones(cols, device=DEV), ctx=gpu_ctx)
    assert torch.isnan(r.scales).all() and (r.codes == 0).all()


# ---------------------------------------------------------------------------
# the table of angles, tangents
# ---------------------------------------------------------------------------
def test_attention_factor_has_64_bits(gpu_ctx):
    """A factor that is no 32-bit number: cosines times it are rounded once, and a turned query of ones shows them."""
    factor, rot, t = 1 + 2.0**-24 * 0.99, 64, 65536
    rope = RopeTable(rot, t, attention_factor=factor, ctx=gpu_ctx)
    cache = Kv4Cache(t // 1024, 1024, 1, 64, ctx=gpu_ctx)
    batch = SeqBatch(i32([0, t]), i32([t]), torch.arange(t // 1024, dtype=torch.int32, device=DEV).view(1, -1), max_q=t)
    kv = torch.zeros(t, 1, 64, dtype=torch.bfloat16, device=DEV)
    # a pair (1, 0) turns into the table's (cos, sin), shown in bf16; of four million numbers about forty lie so close to
    # a border of bf16 that a factor rounded to 32 bits (here to 1) puts them on the other side
    q = torch.zeros(t, 1, 64, dtype=torch.bfloat16, device=DEV)
    q[..., : rot // 2] = 1.0
    got = cache.append(kv, kv, batch, q=q, rope=rope)[:, 0]
    z = torch.arange(t, dtype=torch.float64)[:, None] * torch.as_tensor(rope.inv_freq)
    want = torch.cat([(z.cos() * factor).float(), (z.sin() * factor).float()], 1).bfloat16()
    assert torch.equal(got.cpu(), want)


def test_tangents_are_refused(gpu_ctx):
    cache = Kv4Cache(4, 16, 2, 64, ctx=gpu_ctx)
    batch = SeqBatch(i32([0, 4]), i32([4]), i32([[0]]), max_q=4)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError):
            cache.attend(dual, batch)
        with pytest.raises(ValueError):
            cache.append(dual, x, batch)
        h = torch.ones(2, 64, device=DEV)
        with pytest.raises(ValueError):
            quantize_rows_q8(forward_ad.make_dual(h, h), ctx=gpu_ctx)
        cache.attend(x, batch)  # a tensor without a tangent is welcome


def test_hints_of_the_whole_capacity(gpu_ctx):
    """Hints of the cache's whole capacity, as a captured loop has them, beside exact ones: the same results within the
    roundings, and no row lost."""
    for kv_len in ([777], [8000], [3000, 1, 8000, 450]):
        q_len = [1] * len(kv_len)
        n = sum(kv_len)
        cols = 1024
        table = torch.zeros(len(kv_len), cols, dtype=torch.int32, device=DEV)
        at = 0
        for b, x in enumerate(kv_len):
            need = -(-x // 128)
            table[b, :need] = torch.arange(at, at + need, device=DEV)
            at += need
        cache = Kv4Cache(at, 128, 8, 128, ctx=gpu_ctx)
        k, v = randn(n, 8, 128, seed=1), randn(n, 8, 128, seed=2)
        cu = [0]
        for x in kv_len:
            cu.append(cu[-1] + x)
        cache.append(k, v, SeqBatch(i32(cu), i32(kv_len), table, max_q=max(kv_len)))
        q = randn(len(kv_len), 32, 128, seed=3)
        for max_kv in (max(kv_len), 131072, None, 1):
            batch = SeqBatch(i32(list(range(len(kv_len) + 1))), i32(kv_len), table, max_q=1, max_kv=max_kv)
            B.check(cache.attend(q, batch), q, R.held(k), R.held(v), q_len, kv_len)


def test_hints_of_the_whole_capacity_share_the_keys_out(gpu_ctx):
    """Eight ragged sequences of up to 30000 tokens: chunks follow their lengths, not a hint of 131072 (2.7 times the time)."""
    kv_len = [30000, 4000, 17000, 9000, 25000, 700, 12000, 21000]
    n, page = sum(kv_len), 128
    table, at = torch.zeros(8, 1024, dtype=torch.int32), 0
    for b, x in enumerate(kv_len):
        table[b, : -(-x // page)] = torch.arange(at, at - (-x // page))
        at -= -x // page
    table = table.to(DEV)
    cache = Kv4Cache(at, page, 8, 128, ctx=gpu_ctx)
    cu = [sum(kv_len[:b]) for b in range(9)]
    cache.append(randn(n, 8, 128, seed=1), randn(n, 8, 128, seed=2), SeqBatch(i32(cu), i32(kv_len), table, max_q=max(kv_len)))
    q, times = randn(8, 32, 128, seed=3), []
    for max_kv in (30000, 131072):
        batch = SeqBatch(i32(list(range(9))), i32(kv_len), table, max_q=1, max_kv=max_kv)
        cache.attend(q, batch)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                cache.attend(q, batch)
        best = math.inf
        for _ in range(8):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
    assert times[1] <= 2 * times[0], times


def test_numbers_past_31_bits(gpu_ctx):
    """What a C int would take for another number is refused."""
    for size in (2**32 + 16, -(2**32) + 16):
        with pytest.raises((ValueError, KlError)):
            Kv4Cache(4, size, 2, 64, ctx=gpu_ctx)
        with pytest.raises((ValueError, KlError)):
            Kv4Cache(4, 16, size, 64, ctx=gpu_ctx)
        with pytest.raises((ValueError, KlError)):
            RopeTable(size, 64, ctx=gpu_ctx)
    cache = Kv4Cache(4, 16, 2, 64, ctx=gpu_ctx)
    batch = SeqBatch(i32([0, 4]), i32([4]), i32([[0]]), max_q=4)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    for window in (-(2**32), -(2**33), -(2**32) + 3):
        with pytest.raises(KlError):
            cache.attend(x, batch, window=window)
    with pytest.raises(ValueError):
        cache.read(batch, 2**32)
    gpu_ctx.sync()


def test_calls_after_their_context_is_closed():
    ctx = Context(0)
    cache = Kv4Cache(4, 16, 2, 64, ctx=ctx)
    lin = Q8Linear.from_weights(torch.ones(4, 16), ctx=ctx)
    batch = SeqBatch(i32([0, 4]), i32([4]), i32([[0]]), max_q=4)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    codes, scales = torch.zeros(4, 16, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    ctx.close()
    for call in (lambda: cache.append(x, x, batch), lambda: cache.read(batch, 4), lambda: cache.attend(x, batch),
                 lambda: lin.forward(codes, scales), lambda: quantize_rows_q8(x.flatten(1), ctx=ctx), lambda: RopeTable(64, 4, ctx=ctx)):
        with pytest.raises(RuntimeError):
            call()
