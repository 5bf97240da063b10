"""A decoder layer put together from its parts, as a serving loop runs it: norm
to 8-bit rows, the projections, rotary positions and append, attention, the
output projection into the residual stream, then the sparse MLP stack on the
same stream; prompts, single tokens, captured graphs and streams.

Each part is compared with its plain 64-bit form on the inputs that it got."""

import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import attention_ref as R
from klearu_b200 import _lib
from klearu_b200._lib import KL_EINVAL, HeadRowsC, KlError, SeqBatchC, check
from klearu_b200.attention import Kv4Cache, RopeTable, SeqBatch
from klearu_b200.core import Context
from klearu_b200.dejavu import FfnStack, SparseMlp, SparsityPredictor
from klearu_b200.quant import Q8Linear, add_rms_norm_q8, quantize_rows_q8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0**-24


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Layer:
    """The attention half of a layer: hidden 192, 6 query heads on 2 of 64."""

    hidden, heads, kv_heads, dim, page = 192, 6, 2, 64, 16

    def __init__(self, ctx, seqs, longest):
        h, n = self.hidden, (self.heads + 2 * self.kv_heads) * self.dim
        self.norm = 1 + 0.1 * randn(h, seed=1)
        self.wqkv, self.wo = randn(n, h, seed=2) / h**0.5, randn(h, self.heads * self.dim, seed=3) / (self.heads * self.dim) ** 0.5
        self.qkv = Q8Linear.from_weights(self.wqkv, ctx=ctx)
        self.out = Q8Linear.from_weights(self.wo, ctx=ctx)
        self.rope = RopeTable(self.dim, longest, ctx=ctx)
        cols = -(-longest // self.page)
        self.cache = Kv4Cache(seqs * cols, self.page, self.kv_heads, self.dim, ctx=ctx)
        self.table = torch.randperm(seqs * cols, generator=torch.Generator().manual_seed(5)).to(torch.int32).to(DEV).view(seqs, cols)
        self.ctx = ctx

    def __call__(self, hidden, batch):
        """Adds the attention half to hidden in place; returns what its parts saw and gave."""
        hq, hk, d = self.heads, self.kv_heads, self.dim
        rows = add_rms_norm_q8(hidden, self.norm, ctx=self.ctx)
        qkv = self.qkv.forward(rows.codes, rows.scales, out_dtype=torch.bfloat16)
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hk * d, hk * d], 1))
        turned = self.cache.append(k, v, batch, q=q, rope=self.rope)
        o = self.cache.attend(turned, batch)
        orows = quantize_rows_q8(o.flatten(1), ctx=self.ctx)
        self.out.forward(orows.codes, orows.scales, out=hidden, accumulate=True)
        return {"rows": rows, "qkv": qkv, "q": q, "turned": turned, "o": o, "orows": orows}


def check_parts(layer, before, hidden, parts, batch, q_len, kv_len):
    def q8(w):
        top = w.double().abs().amax(-1, keepdim=True)
        return (w.double() * 127 / top).round() * top / 127

    rows = parts["rows"]
    x = rows.codes.double() * rows.scales.double()[:, None]
    want = before.double() / (before.double().square().mean(-1, keepdim=True) + 1e-5).sqrt() * layer.norm.double()
    # half a step of 1 / 127 of the row's largest, and the scale's own roundings
    assert ((x - want).abs() <= want.abs().amax(-1, keepdim=True) / 254 * 1.001).all()
    want = x @ q8(layer.wqkv).T
    assert ((parts["qkv"].double() - want).abs() <= R.HALF * want.abs() + 1e-5 * (x.abs() @ q8(layer.wqkv).abs().T)).all()
    pos = torch.cat([torch.arange(b - a, b, device=DEV) for a, b in zip(q_len, kv_len)])
    want = R.rotate(parts["q"], pos, layer.rope.inv_freq, False)
    assert ((parts["turned"].double() - want).abs() <= R.HALF * want.abs() + 1e-5).all()
    # attention over what the cache holds for each sequence
    a = 0
    for b, (ql, kl) in enumerate(zip(q_len, kv_len)):
        one = SeqBatch(i32([0, kl]), batch.kv_len[b : b + 1], batch.page_table[b : b + 1], max_q=kl)
        k, v = layer.cache.read(one, kl)
        # read() rounds the held values to bf16: half a step more for keys and values
        want, tol = R.attend(parts["turned"][a : a + ql], k.double(), v.double(), kl - ql, 0, layer.dim**-0.5)
        assert ((parts["o"][a : a + ql].double() - want).abs() <= 2 * tol).all()
        a += ql
    o = parts["orows"].codes.double() * parts["orows"].scales.double()[:, None]
    want = before.double() + o @ q8(layer.wo).T
    assert ((hidden.double() - want).abs() <= 1e-5 * (before.double().abs() + o.abs() @ q8(layer.wo).abs().T)).all()


def test_prompts_then_tokens(gpu_ctx):
    """Two ragged prompts, one of them in two chunks, then tokens one by one, with the MLP stack after the attention half."""
    layer = Layer(gpu_ctx, 2, 300)
    h = layer.hidden
    rng = np.random.default_rng(3)
    w = lambda *s: (rng.standard_normal(s) * 0.05).astype(np.float32)  # noqa: E731
    pred = SparsityPredictor(w(40, h), w(40), w(256, 40), w(256), ctx=gpu_ctx)
    mlp = SparseMlp(w(256, h), w(256, h), w(h, 256), ctx=gpu_ctx)
    stack = FfnStack([pred], [mlp], np.ones((1, h), np.float32), ctx=gpu_ctx)
    length = [0, 0]
    for q_len in ([130, 7], [61, 100], [1, 1], [1, 1], [3, 1]):
        length = [a + b for a, b in zip(length, q_len)]
        cu = i32(np.cumsum([0] + q_len).tolist())
        batch = SeqBatch(cu, i32(length), layer.table, max_q=max(q_len), max_kv=max(length))
        hidden = 2 * randn(sum(q_len), h, seed=sum(length))
        before = hidden.clone()
        parts = layer(hidden, batch)
        check_parts(layer, before, hidden, parts, batch, q_len, length)
        copy = hidden.clone()
        stack.decode(hidden, 0.25)
        assert torch.equal(hidden, stack.decode(copy, 0.25)) and not torch.equal(hidden, before)
    gpu_ctx.sync()


def test_captured_decode_loop(gpu_ctx):
    """One graph, captured once, decodes token after token with the lengths updated in place."""
    layer, twin = Layer(gpu_ctx, 3, 200), Layer(gpu_ctx, 3, 200)
    start = [40, 1, 95]
    for x in (layer, twin):
        first = SeqBatch(i32(np.cumsum([0] + start).tolist()), i32(start), x.table, max_q=max(start))
        x(randn(sum(start), x.hidden, seed=9), first)
    kv = i32([s + 1 for s in start])
    batch = SeqBatch(i32([0, 1, 2, 3]), kv, layer.table, max_q=1, max_kv=200)
    hidden = randn(3, layer.hidden, seed=10)
    keep = hidden.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(hidden.clone(), batch)  # any first-call set-up outside the graph
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(hidden, batch)
    for step in range(4):
        hidden.copy_(keep + step)
        graph.replay()
        plain = keep + step
        twin(plain, SeqBatch(i32([0, 1, 2, 3]), kv.clone(), twin.table, max_q=1, max_kv=200))
        assert torch.equal(hidden, plain), step
        kv += 1
    gpu_ctx.sync()


def test_streams_and_graphs_at_once(gpu_ctx):
    """Calls follow torch's current stream; two graphs of one cache replayed at the same time have workspaces of their own."""
    kv_len = [6000, 900, 3000]
    n = sum(kv_len)
    cache = Kv4Cache(n // 16 + 4, 16, 2, 128, ctx=gpu_ctx)
    cols = [-(-k // 16) for k in kv_len]
    table = torch.zeros(3, max(cols), dtype=torch.int32)
    at = 0
    for b, c in enumerate(cols):
        table[b, :c] = torch.arange(at, at + c)
        at += c
    table = table.to(DEV)
    every = SeqBatch(i32(np.cumsum([0] + kv_len).tolist()), i32(kv_len), table, max_q=max(kv_len))
    cache.append(randn(n, 2, 128, seed=1, dtype=torch.bfloat16), randn(n, 2, 128, seed=2, dtype=torch.bfloat16), every)
    batch = SeqBatch(i32([0, 1, 2, 3]), i32(kv_len), table, max_q=1, max_kv=6000)
    qs = [randn(3, 8, 128, seed=s, dtype=torch.bfloat16) for s in (3, 4)]
    want = [cache.attend(q, batch) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    graphs, outs = [], []
    for q, s in zip(qs, streams):
        with torch.cuda.stream(s):
            assert torch.equal(cache.attend(q, batch), want[len(graphs)])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cache.attend(q, batch))
        graphs.append(g)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_kernels_that_begin_early(gpu_ctx):
    """Calls one behind the other, where a kernel may begin while the one before ends, give what they give with a
    wait after each; buffers are written again by the next call as soon as the last has read them."""
    layer, twin = Layer(gpu_ctx, 4, 700), Layer(gpu_ctx, 4, 700)
    wide = Q8Linear.from_weights(randn(700, layer.hidden, seed=20), ctx=gpu_ctx)
    back = Q8Linear.from_weights(randn(layer.hidden, 700, seed=21) / 700, ctx=gpu_ctx)

    def run(x, wait):
        length, got = 0, []
        hidden = None
        for step in range(60):
            n = 37 if step % 20 == 0 else 1
            length += n
            batch = SeqBatch(i32([0, n, 2 * n, 3 * n, 4 * n]), i32([length] * 4), x.table, max_q=n)
            if hidden is None or hidden.shape[0] != 4 * n:
                hidden = randn(4 * n, x.hidden, seed=step)
            for _ in range(3):
                rows = add_rms_norm_q8(hidden, x.norm, ctx=gpu_ctx)
                wait()
                up = wide.forward(rows.codes, rows.scales)
                wait()
                rows = quantize_rows_q8(up, ctx=gpu_ctx)
                wait()
                back.forward(rows.codes, rows.scales, out=hidden, accumulate=True)
                wait()
            x(hidden, batch)
            wait()
            hidden /= hidden.abs().amax()
            got.append(hidden.clone())
        return got

    slow = run(twin, torch.cuda.synchronize)
    for _ in range(3):
        fast = run(layer, lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(fast, slow))


def test_calls_allocate_nothing(gpu_ctx):
    """Apart from torch's own tensors: a second call of every kind adds no allocation of the library's."""
    layer = Layer(gpu_ctx, 1, 400)
    n = C.c_uint64()

    def count():
        check(gpu_ctx.lib.kl_alloc_count(C.byref(n)))
        return n.value

    def both():
        layer(randn(300, layer.hidden), SeqBatch(i32([0, 300]), i32([300]), layer.table, max_q=300))
        layer(randn(1, layer.hidden), SeqBatch(i32([0, 1]), i32([301]), layer.table, max_q=1))

    both()
    before = count()
    both()
    assert count() == before


def test_context_of_its_own(gpu_ctx):
    """A layer on a context whose stream is not the current one: calls still run on torch's current stream."""
    own = Context(0, stream=torch.cuda.Stream())
    layer, twin = Layer(own, 1, 64), Layer(gpu_ctx, 1, 64)
    a, b = randn(20, layer.hidden, seed=4), randn(20, layer.hidden, seed=4)
    layer(a, SeqBatch(i32([0, 20]), i32([20]), layer.table, max_q=20))
    twin(b, SeqBatch(i32([0, 20]), i32([20]), twin.table, max_q=20))
    assert torch.equal(a, b)
    own.sync()


def test_c_entry_points_refuse(gpu_ctx):
    """What the C calls check themselves: workspaces, strides, null pointers, types."""
    lib = gpu_ctx.lib
    cache = Kv4Cache(64, 16, 2, 64, ctx=gpu_ctx)
    table, kv, cu = i32([list(range(64))]), i32([1000]), i32([0, 1])
    s = SeqBatchC(cu.data_ptr(), kv.data_ptr(), table.data_ptr(), 64, 64, 1, 1, 1, 1000)
    q = randn(1, 2, 64, dtype=torch.bfloat16)
    rows = HeadRowsC(q.data_ptr(), 128, 64)
    need = C.c_size_t()
    assert lib.kl_kv4_attend_workspace(cache.h, C.byref(s), 2, 0, C.byref(need)) == 0 and need.value > 0
    space = torch.empty(need.value + 16, dtype=torch.uint8, device=DEV)

    def attend(seqs=s, heads=2, q=rows, out=rows, scale=1.0, window=0, ws=space.data_ptr(), size=None):
        size = need.value if size is None else size
        ref = lambda x: None if x is None else C.byref(x)  # noqa: E731
        return lib.kl_kv4_attend(cache.h, ref(seqs), heads, ref(q), ref(out), scale, window, ws, size)

    assert attend() == 0
    bad = SeqBatchC(cu.data_ptr(), kv.data_ptr(), table.data_ptr(), 63, 64, 1, 1, 1, 1000)
    none = SeqBatchC(None, kv.data_ptr(), table.data_ptr(), 64, 64, 1, 1, 1, 1000)
    for kw in ({"size": need.value - 1}, {"ws": None}, {"ws": space.data_ptr() + 4}, {"seqs": None}, {"seqs": bad}, {"seqs": none},
               {"heads": 3}, {"heads": 0}, {"q": None}, {"out": HeadRowsC(None, 128, 64)}, {"q": HeadRowsC(q.data_ptr() + 1, 128, 64)},
               {"q": HeadRowsC(q.data_ptr(), -128, 64)}, {"scale": float("inf")}, {"window": -1}):
        assert attend(**kw) == KL_EINVAL, kw
    lin = Q8Linear.from_weights(randn(8, 32), ctx=gpu_ctx)
    a = torch.zeros(4, 32, dtype=torch.int8, device=DEV)
    sc, out = torch.ones(4, device=DEV), torch.zeros(4, 8, device=DEV)
    ok = [a.data_ptr(), 32, sc.data_ptr(), 4, out.data_ptr(), _lib.DTYPE_F32, 8, 0]
    assert lib.kl_q8_linear_forward(lin.h, *ok) == 0
    for i, v in ((0, a.data_ptr() + 1), (0, None), (1, 24), (1, 31), (2, None), (3, -1), (4, None), (5, 7), (6, 7)):
        assert lib.kl_q8_linear_forward(lin.h, *[v if i == j else x for j, x in enumerate(ok)]) == KL_EINVAL, (i, v)
    assert lib.kl_q8_linear_forward(lin.h, *ok[:5], _lib.DTYPE_BF16, 8, 1) == KL_EINVAL
    x = randn(2, 32)
    codes = torch.zeros(2, 32, dtype=torch.int8, device=DEV)
    ok = [gpu_ctx.h, x.data_ptr(), _lib.DTYPE_F32, 32, None, 0, None, 2, 32, 0.0, 0, 0, None, 0, codes.data_ptr(), 32, sc.data_ptr()]
    assert lib.kl_norm_q8(*ok) == 0
    for i, v in ((1, None), (2, 9), (3, 31), (7, -1), (8, 0), (9, -1.0), (14, None), (15, 31), (16, None)):
        assert lib.kl_norm_q8(*[v if i == j else y for j, y in enumerate(ok)]) == KL_EINVAL, (i, v)
    with pytest.raises(KlError):
        check(lib.kl_kv4_append(cache.h, None, C.byref(s), None, 0, None, None, C.byref(rows), None), gpu_ctx.h)
    gpu_ctx.sync()


FIRST = """
import torch
from klearu_b200.attention import Kv4Cache, RopeTable, SeqBatch
from klearu_b200.quant import Q8Linear, add_rms_norm_q8
dev = "cuda:0"
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
x, w = torch.randn(600, 256, device=dev), torch.ones(256, device=dev)
wide = Q8Linear(torch.ones(9000, 256, dtype=torch.int8, device=dev), torch.ones(9000, device=dev))
cache, rope = Kv4Cache(64, 64, 8, 64), RopeTable(64, 4096)
qkv = torch.randn(600, 24, 64, device=dev, dtype=torch.bfloat16)
table = torch.arange(64, dtype=torch.int32, device=dev).view(1, 64)
prompt = SeqBatch(i32([0, 600]), i32([600]), table, max_q=600, max_kv=600)
token = SeqBatch(i32([0, 1]), i32([600]), table, max_q=1, max_kv=4096)

def run():
    r = add_rms_norm_q8(x, w)
    y = [wide.forward(r.codes[:n], r.scales[:n]) for n in (1, 40, 600)]
    q = cache.append(qkv[:, 8:16], qkv[:, 16:], prompt, q=qkv[:, :8], rope=rope)
    k, v = cache.read(prompt, 600)
    o = [cache.attend(q, prompt), cache.attend(q[:1], token), cache.attend(torch.cat([q] * 4, 1), prompt)]
    return [r.codes, r.scales, *y, q, k, v, *o]

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = run()
g.replay()
want = run()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("captured first")
"""


def test_first_calls_can_be_captured(gpu_ctx):
    """In a process of its own: no call needs to have run before it is captured."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=root)
    done = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=240, env=env)
    assert done.returncode == 0 and "captured first" in done.stdout, done.stderr[-2000:]


def test_outputs_that_overlap_and_in_place(gpu_ctx):
    cache = Kv4Cache(64, 16, 2, 64, ctx=gpu_ctx)
    table = i32([list(range(64))])
    every = SeqBatch(i32([0, 1000]), i32([1000]), table, max_q=1000)
    k, v = randn(1000, 2, 64, seed=1, dtype=torch.bfloat16), randn(1000, 2, 64, seed=2, dtype=torch.bfloat16)
    cache.append(k, v, every)
    for n in (1, 5, 200):
        batch = SeqBatch(i32([0, n]), i32([1000]), table, max_q=n)
        q = randn(n, 4, 64, seed=3, dtype=torch.bfloat16)
        want = cache.attend(q, batch)
        assert torch.equal(cache.attend(q, batch, window=2**40), want)
        assert cache.attend(q, batch, out=q) is q and torch.equal(q, want)
    q = randn(8, 4, 64, dtype=torch.bfloat16)
    batch = SeqBatch(i32([0, 8]), i32([1000]), table, max_q=8)
    flat = torch.zeros(8 * 4 * 64, dtype=torch.bfloat16, device=DEV)
    for bad in (flat[:256].view(1, 4, 64).expand(8, 4, 64), flat[:512].view(8, 1, 64).expand(8, 4, 64),
                flat.as_strided((8, 4, 64), (128, 64, 1)), flat.as_strided((8, 4, 64), (64, 64, 1))):
        with pytest.raises(ValueError):
            cache.attend(q, batch, out=bad)
        with pytest.raises(ValueError):
            cache.append(k[:8], v[:8], batch, q=q, q_out=bad)
    fine = flat.as_strided((8, 4, 64), (64, 512, 1))  # heads outside, tokens inside
    assert torch.equal(cache.attend(q, batch, out=fine), cache.attend(q, batch))
    with pytest.raises(ValueError):
        cache.append("k", v, batch)
