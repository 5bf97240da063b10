"""The attention half of a decoder layer: rotary positions, a paged cache of
4-bit keys and values, and attention over it.

``dejavu.FfnStack`` runs the MLP half of klearu-llm's decode step on the
residual stream; these calls are what comes before it in each layer (the
reference keeps f32 keys and values, crates/klearu-llm/src/model/kv_cache.rs).
``quant`` has the 8-bit projections around them.

Every call launches on torch's current stream, like a torch operator, and can
be captured in a CUDA graph; tensors have to be on the context's device.  As for
all handles of the library, one host thread at a time calls a context and what
was made with it.
Nothing here has a backward pass: an input that requires a gradient is refused
while gradients are recorded, and so is one with a forward-mode tangent.
"""

from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch
from torch.autograd import forward_ad

from ._lib import HeadRowsC, SeqBatchC, check
from .core import Context, default_context


_BF16 = torch.bfloat16
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def launch(ctx: Context, what: str, *args) -> None:
    """One C call on torch's current stream of the context's device."""
    if not ctx.h:
        raise RuntimeError("the context is closed")
    s = _raw_stream(ctx.device)
    lib, own = ctx.lib, ctx.stream.cuda_stream
    with ctx.launch_lock:
        if s == own:
            status = getattr(lib, what)(*args)
        else:
            lib.kl_ctx_set_stream(ctx.h, s)
            try:
                status = getattr(lib, what)(*args)
            finally:
                lib.kl_ctx_set_stream(ctx.h, own)
        if status:
            check(status, ctx.h, what)


def want(ctx: Context, t: torch.Tensor, what: str, dtype) -> None:
    """What every tensor argument has to be."""
    if not isinstance(t, torch.Tensor) or t.get_device() != ctx.device:
        raise ValueError(f"{what} must be a tensor on cuda:{ctx.device}")
    if t.dtype is not dtype and not (isinstance(dtype, tuple) and t.dtype in dtype):
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires a gradient, and this call has no backward pass")
    if forward_ad._current_level >= 0 and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what} has a tangent, which this call would drop; unpack it first")


class RopeTable:
    """Rotary positions: pair i of a head turns by p * base^(-2i / rot_dim) at
    position p < max_positions.  The pairs are dims (2i, 2i + 1) with
    ``interleaved``, else (i, i + rot_dim / 2); dims from rot_dim on stay.

    ``scaling`` stretches the frequencies f for contexts longer than the trained
    one: ``"linear"``: f / factor; ``"by_parts"``: with r = original_positions *
    f / (2 pi) turns over the trained context and k = clamp((r - low_turns) /
    (high_turns - low_turns), 0, 1), f * (k + (1 - k) / factor).
    ``attention_factor`` multiplies cosines and sines.  Angles are computed in
    64 bits."""

    def __init__(self, rot_dim: int, max_positions: int, base: float = 10000.0, interleaved: bool = False,
                 scaling: str | None = None, factor: float = 1.0, original_positions: int | None = None,
                 low_turns: float = 1.0, high_turns: float = 4.0, attention_factor: float = 1.0,
                 ctx: Context | None = None):
        if rot_dim < 2 or rot_dim % 2 or rot_dim >= 2**31:
            raise ValueError("rot_dim must be even and >= 2")
        if not (base > 0 and factor > 0 and math.isfinite(attention_factor)):
            raise ValueError("base and factor must be > 0, attention_factor finite")
        f = float(base) ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
        if scaling == "linear":
            f = f / factor
        elif scaling == "by_parts":
            if original_positions is None or not high_turns > low_turns:
                raise ValueError("by_parts needs original_positions and high_turns > low_turns")
            turns = original_positions * f / (2 * math.pi)
            keep = np.clip((turns - low_turns) / (high_turns - low_turns), 0.0, 1.0)
            f = f * (keep + (1 - keep) / factor)
        elif scaling is not None:
            raise ValueError('scaling must be None, "linear" or "by_parts"')
        self.ctx = ctx or default_context()
        self.lib = self.ctx.lib
        self.rot_dim, self.max_positions, self.interleaved = rot_dim, max_positions, interleaved
        self.inv_freq = np.ascontiguousarray(f)
        h = C.c_void_p()
        launch(self.ctx, "kl_rope_create_f64", self.ctx.h, rot_dim, max_positions, self.inv_freq.ctypes.data,
               attention_factor, int(interleaved), C.byref(h))
        self.h = h

    def __del__(self):
        if getattr(self, "h", None):
            self.lib.kl_rope_destroy(self.h)


class SeqBatch:
    """The sequences of a call (int32 tensors on the GPU): rows ``cu_q[b]`` to
    ``cu_q[b + 1]`` of the call's token tensors are sequence b's new tokens, the
    last of its ``kv_len[b]`` tokens; its token j is in page
    ``page_table[b, j // page_size]``.

    ``max_q`` and ``max_kv`` are the largest numbers of new and of all tokens;
    they choose the launch (too small or too large is slower, not wrong; a
    ``max_kv`` of the whole table costs a few us), so one object, its tensors
    updated in place, serves a captured decode loop.  Tokens beyond the table or
    the call's tensors are reported by ``Context.sync``, not written and not
    attended to."""

    def __init__(self, cu_q: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor, max_q: int,
                 max_kv: int | None = None):
        for t, name, dim in ((cu_q, "cu_q", 1), (kv_len, "kv_len", 1), (page_table, "page_table", 2)):
            if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.int32 or t.dim() != dim:
                raise ValueError(f"{name} must be a {dim}-D int32 CUDA tensor")
            if t.device != cu_q.device:
                raise ValueError("cu_q, kv_len and page_table must be on one device")
            if t.numel() and t.stride(-1) != 1:
                raise ValueError(f"{name} must be contiguous in its last dimension")
        n = kv_len.shape[0]
        if cu_q.shape[0] != n + 1 or page_table.shape[0] != n:
            raise ValueError("cu_q must have one entry more than kv_len, page_table one row each")
        if max_q < 0 or (max_kv is not None and max_kv < 0):
            raise ValueError("max_q and max_kv must be >= 0")
        self._tensors = (cu_q, kv_len, page_table)
        self.num_seqs, self.max_q = n, int(max_q)
        self.max_kv = 2**31 - 1 if max_kv is None else min(int(max_kv), 2**31 - 1)
        self.device = cu_q.device.index
        self.sizes = (n, self.max_q, self.max_kv, page_table.shape[1])
        self._c: dict[int, object] = {}  # the C struct by num_tokens

    cu_q = property(lambda self: self._tensors[0])
    kv_len = property(lambda self: self._tensors[1])
    page_table = property(lambda self: self._tensors[2])

    def c(self, num_tokens: int):
        """A reference to the C struct for a call with so many rows."""
        got = self._c.get(num_tokens)
        if got is None:
            if len(self._c) >= 64:
                self._c.clear()
            cu_q, kv_len, table = self._tensors
            wide = table.shape[1]
            got = self._c[num_tokens] = C.byref(SeqBatchC(
                cu_q.data_ptr(), kv_len.data_ptr(), table.data_ptr(), table.stride(0) if self.num_seqs > 1 else wide, wide,
                self.num_seqs, num_tokens, min(self.max_q, 2**31 - 1), self.max_kv))
        return got


class Kv4Cache:
    """A paged cache of keys and values in 4 bits: ``num_pages`` pages of
    ``page_size`` tokens (a multiple of 16) for ``kv_heads`` heads of ``head_dim``
    64 or 128.  A head vector x is held as x ~ s * c + m with m = bf16(min x),
    s = bf16((max x - min x) / 15) and codes c in 0..15: ``head_dim + 8`` bytes
    for a token's key and value in one head."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, ctx: Context | None = None):
        if max(page_size, kv_heads, head_dim) >= 2**31 or min(page_size, kv_heads, head_dim) < 0:
            raise ValueError("page_size, kv_heads and head_dim must be whole numbers of 31 bits")
        self.ctx = ctx or default_context()
        self.lib = self.ctx.lib
        self.num_pages, self.page_size, self.kv_heads, self.head_dim = num_pages, page_size, kv_heads, head_dim
        h = C.c_void_p()
        launch(self.ctx, "kl_kv4_create", self.ctx.h, num_pages, page_size, kv_heads, head_dim, C.byref(h))
        self.h = h
        self._workspace: dict[tuple, int] = {}  # bytes by the sizes that decide them

    def __del__(self):
        if getattr(self, "h", None):
            self.lib.kl_kv4_destroy(self.h)

    def _rows(self, t: torch.Tensor, what: str, tokens: int | None = None, heads: int | None = None):
        want(self.ctx, t, what, _BF16)
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or shape[2] != self.head_dim or stride[2] != 1:
            raise ValueError(f"{what} must be [tokens][heads][{self.head_dim}], contiguous in the last dimension")
        if (tokens is not None and shape[0] != tokens) or (heads is not None and shape[1] != heads):
            raise ValueError(f"{what} has shape {tuple(shape)}, expected {tokens} tokens and {heads} heads")
        return C.byref(HeadRowsC(t.data_ptr(), stride[0], stride[1]))

    def _out(self, t: torch.Tensor, what: str, tokens: int, heads: int):
        """``_rows`` of a tensor to be written, whose rows must lie apart."""
        r = self._rows(t, what, tokens, heads)
        reach = self.head_dim  # of the rows so far, from the closest together to the farthest apart
        for step, n in sorted((s, n) for s, n in zip(t.stride(), t.shape[:2]) if n > 1):
            if step < reach:
                raise ValueError(f"{what}'s rows overlap")
            reach += step * (n - 1)
        return r

    def _new(self, like: torch.Tensor, tokens: int, heads: int):
        """A new [tokens][heads][head_dim] tensor and its C rows."""
        d = self.head_dim
        t = torch.empty_like(like) if like.is_contiguous() else like.new_empty((tokens, heads, d))
        return t, C.byref(HeadRowsC(t.data_ptr(), heads * d, d))

    def _batch(self, batch: SeqBatch, tokens: int):
        if batch.device != self.ctx.device:
            raise ValueError(f"the batch must be on cuda:{self.ctx.device}")
        return batch.c(tokens)

    def append(self, k: torch.Tensor, v: torch.Tensor, batch: SeqBatch, q: torch.Tensor | None = None,
               rope: RopeTable | None = None, positions: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Turns q and k by their positions (their tokens' numbers, or ``positions``
        [tokens] int32) and writes k and v [tokens][kv_heads][head_dim] (bf16) to
        the cache; returns the turned q [tokens][q_heads][head_dim] (``q_out`` if
        given, which may be q).  Rows of no sequence are left as they are.  Two
        rows must not name the same token of the same page."""
        rk = self._rows(k, "k", heads=self.kv_heads)
        t = k.shape[0]
        rv = self._rows(v, "v", t, self.kv_heads)
        heads, rq, ro = 0, None, None
        if q is not None:
            rq = self._rows(q, "q", t)
            heads = q.shape[1]
            if q_out is None:
                q_out, ro = self._new(q, t, heads)
            else:
                ro = self._out(q_out, "q_out", t, heads)
        elif q_out is not None:
            raise ValueError("q_out without q")
        if positions is not None:
            want(self.ctx, positions, "positions", torch.int32)
            if positions.shape != (t,) or not positions.is_contiguous():
                raise ValueError("positions must be contiguous, one for each token")
        if rope is not None and rope.ctx is not self.ctx:
            raise ValueError("the rope must share the cache's context")
        c = self._batch(batch, t)
        if t:
            launch(self.ctx, "kl_kv4_append", self.h, rope.h if rope is not None else None, c,
                   None if positions is None else positions.data_ptr(), heads, rq, rk, rv, ro)
        return q_out

    def read(self, batch: SeqBatch, num_tokens: int, k_out: torch.Tensor | None = None,
             v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The values that the cached keys and values of the batch's new tokens
        stand for, [num_tokens][kv_heads][head_dim] (bf16), num_tokens the rows of
        the call (cu_q's last entry, or more).  Rows of no sequence are left as
        they are."""
        if not 0 <= num_tokens < 2**31:
            raise ValueError("num_tokens must be in [0, 2^31)")
        c = self._batch(batch, num_tokens)
        heads = self.kv_heads
        if k_out is None and v_out is None:
            both = batch.kv_len.new_empty((2, num_tokens, heads, self.head_dim), dtype=_BF16)
            k_out, v_out = both.unbind()
            at, d = both.data_ptr(), heads * self.head_dim
            rk = C.byref(HeadRowsC(at, d, self.head_dim))
            rv = C.byref(HeadRowsC(at + 2 * num_tokens * d, d, self.head_dim))
        else:
            if k_out is None:
                k_out = torch.empty_like(v_out)
            elif v_out is None:
                v_out = torch.empty_like(k_out)
            rk, rv = self._out(k_out, "k_out", num_tokens, heads), self._out(v_out, "v_out", num_tokens, heads)
        if num_tokens:
            launch(self.ctx, "kl_kv4_read", self.h, c, rk, rv)
        return k_out, v_out

    def attend(self, q: torch.Tensor, batch: SeqBatch, scale: float | None = None, window: int = 0,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """softmax(scale * q . K^T) . V for q [tokens][q_heads][head_dim] (bf16,
        q_heads a multiple of kv_heads, query head h on key head
        h // (q_heads / kv_heads)).  A token sees the tokens up to its own number
        in its sequence, and with ``window`` only the last ``window`` of those;
        one that sees nothing gets zeros.  ``scale`` defaults to
        head_dim ** -0.5.  Returns ``out`` (allocated if None; it may be q), rows
        of no sequence left as they are."""
        rq = self._rows(q, "q")
        t, heads = q.shape[0], q.shape[1]
        if out is None:
            out, ro = self._new(q, t, heads)
        else:
            ro = self._out(out, "out", t, heads)
        c = self._batch(batch, t)
        if t == 0 or heads == 0:
            return out
        window = max(-1, min(window, 2**31 - 1))  # a C int would take a number past 31 bits for another
        key = (batch.sizes, t, heads, window)
        need = self._workspace.get(key)
        if need is None:
            n = C.c_size_t()
            launch(self.ctx, "kl_kv4_attend_workspace", self.h, c, heads, window, C.byref(n))
            if len(self._workspace) >= 4096:
                self._workspace.clear()
            need = self._workspace[key] = n.value
        # from torch's allocator in stream order: a captured graph keeps one of its own
        space = q.new_empty((need + 1) // 2) if need else None
        launch(self.ctx, "kl_kv4_attend", self.h, c, heads, rq, ro, self.head_dim**-0.5 if scale is None else scale, window,
               space.data_ptr() if need else None, need)
        return out
