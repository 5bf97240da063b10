"""8-bit rows and projections: codes with one f32 scale for each row (token)
and each output channel, products summed in 32-bit integers.

``add_rms_norm_q8`` is the residual addition and norm that a decoder layer
begins with (``dejavu.FfnStack`` applies the same norm in f32), with its output
as the codes that ``Q8Linear`` takes.  Calls launch on torch's current stream
and can be captured in a CUDA graph; nothing here has a backward pass.
"""

from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from . import _lib
from .attention import launch, want
from .core import Context, default_context


class Q8Rows(NamedTuple):
    """x ~ codes * scales[:, None]; hidden: what was quantized before the norm (f32), if asked for."""

    codes: torch.Tensor   # [rows][cols] int8, rows start on 16 bytes
    scales: torch.Tensor  # [rows] f32
    hidden: torch.Tensor | None


def _two(t: torch.Tensor, what: str) -> int:
    """The row stride of a 2-D tensor that is contiguous in its last dimension."""
    stride, shape = t.stride(), t.shape
    if len(shape) != 2 or (stride[1] != 1 and t.numel()):
        raise ValueError(f"{what} must be 2-D, contiguous in its last dimension")
    return stride[0] if shape[0] > 1 else max(shape[1], stride[0])


def _rows_q8(x, weight, residual, eps, norm, one_plus, hidden, ctx) -> Q8Rows:
    if ctx is None:  # the tensor's device says which context
        if not isinstance(x, torch.Tensor) or not x.is_cuda:
            raise ValueError("x must be a CUDA tensor")
        ctx = default_context(x.get_device())
    want(ctx, x, "x", (torch.float32, torch.bfloat16))
    ldx = _two(x, "x")
    rows, cols = x.shape
    if cols == 0:
        raise ValueError("x has no columns")
    if weight is not None:
        want(ctx, weight, "weight", torch.float32)
        if weight.shape != (cols,) or not weight.is_contiguous():
            raise ValueError("weight must be contiguous, one for each column")
    ldr = ldh = 0
    if residual is not None:
        want(ctx, residual, "residual", torch.float32)
        ldr = _two(residual, "residual")
    if hidden is not None:
        want(ctx, hidden, "hidden", torch.float32)
        ldh = _two(hidden, "hidden")
    if (ldr and residual.shape != x.shape) or (ldh and hidden.shape != x.shape):
        raise ValueError("residual and hidden must have x's shape")
    ld = -(-cols // 16) * 16
    if ld == cols and x.is_contiguous():
        codes = torch.empty_like(x, dtype=torch.int8)
    else:
        codes = x.new_empty((rows, ld), dtype=torch.int8)[:, :cols]
    scales = x.new_empty(rows, dtype=torch.float32)
    if rows:
        launch(ctx, "kl_norm_q8", ctx.h, x.data_ptr(),
               _lib.DTYPE_BF16 if x.dtype == torch.bfloat16 else _lib.DTYPE_F32, ldx,
               None if residual is None else residual.data_ptr(), ldr,
               None if weight is None else weight.data_ptr(), rows, cols, eps, norm, int(one_plus),
               None if hidden is None else hidden.data_ptr(), ldh,
               codes.data_ptr(), ld, scales.data_ptr())
    return Q8Rows(codes, scales, hidden)


def add_rms_norm_q8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-5,
                    one_plus_weight: bool = False, hidden: torch.Tensor | None = None,
                    ctx: Context | None = None) -> Q8Rows:
    """h = x + residual (x f32 or bf16 [rows][cols], residual f32), then the codes
    and scales of h / sqrt(mean(h^2) + eps) * weight (1 + weight with
    ``one_plus_weight``).  ``hidden`` receives h; pass ``residual`` itself to
    update the residual stream in place; by default, with a residual, a new
    tensor.  A row that is not finite gets scale NaN."""
    if hidden is None and isinstance(residual, torch.Tensor):
        hidden = torch.empty_like(residual) if residual.is_contiguous() else residual.new_empty(residual.shape)
    return _rows_q8(x, weight, residual, eps, 1, one_plus_weight, hidden, ctx)


def quantize_rows_q8(x: torch.Tensor, ctx: Context | None = None) -> Q8Rows:
    """The codes and scales of x's rows as they are (an attention output before
    its projection, a weight matrix): scale = max|x| / 127."""
    return _rows_q8(x, None, None, 0.0, 0, False, None, ctx)


class Q8Linear:
    """A projection with weights in 8 bits: ``codes`` [out][in] int8 and
    ``scales`` [out] f32, optional ``bias`` [out] f32 (CUDA tensors, copied)."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None,
                 ctx: Context | None = None):
        self.ctx = ctx or default_context()
        self.lib = self.ctx.lib
        want(self.ctx, codes, "codes", torch.int8)
        ld = _two(codes, "codes")
        self.out_features, self.in_features = codes.shape
        for t, name in ((scales, "scales"), (bias, "bias")):
            if t is not None:
                want(self.ctx, t, name, torch.float32)
                if t.shape != (self.out_features,) or not t.is_contiguous():
                    raise ValueError(f"{name} must be contiguous, one for each output")
        h = C.c_void_p()
        launch(self.ctx, "kl_q8_linear_create", self.ctx.h, self.in_features, self.out_features, codes.data_ptr(),
               ld, scales.data_ptr(), None if bias is None else bias.data_ptr(), C.byref(h))
        self.h = h

    @classmethod
    def from_weights(cls, w, bias=None, ctx: Context | None = None) -> "Q8Linear":
        """Quantizes f32 weights [out][in] (anything ``torch.as_tensor`` accepts)
        per output channel: scale = max|w| / 127."""
        ctx = ctx or default_context()
        dev = f"cuda:{ctx.device}"
        w = torch.as_tensor(w).detach().to(device=dev, dtype=torch.float32).contiguous()
        b = None if bias is None else torch.as_tensor(bias).detach().to(device=dev, dtype=torch.float32).contiguous()
        r = quantize_rows_q8(w, ctx=ctx)
        return cls(r.codes, r.scales, b, ctx=ctx)

    def __del__(self):
        if getattr(self, "h", None):
            self.lib.kl_q8_linear_destroy(self.h)

    def forward(self, codes: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = torch.float32,
                out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
        """(codes . W^T) * scales[:, None] * w_scales (+ bias) for codes [rows][in]
        int8 (rows on 16 bytes, as the calls above write them) and scales [rows]
        f32; f32 or bf16 out, added to an f32 ``out`` with ``accumulate``."""
        want(self.ctx, codes, "codes", torch.int8)
        want(self.ctx, scales, "scales", torch.float32)
        ld = _two(codes, "codes")
        rows = codes.shape[0]
        if codes.shape[1] != self.in_features or scales.shape != (rows,) or not scales.is_contiguous():
            raise ValueError("codes must be [rows][in_features], scales contiguous, one for each row")
        if rows == 1:
            ld = -(-ld // 16) * 16  # a single row has no next one
        if rows and (codes.data_ptr() % 16 or ld % 16):
            raise ValueError("the codes' rows must start on 16 bytes")
        if out is None:
            if accumulate:
                raise ValueError("accumulate needs out")
            if out_dtype not in (torch.float32, torch.bfloat16):
                raise ValueError("out_dtype must be float32 or bfloat16")
            out = codes.new_empty((rows, self.out_features), dtype=out_dtype)
            ldo = self.out_features
        else:
            want(self.ctx, out, "out", torch.float32 if accumulate else (torch.float32, torch.bfloat16))
            ldo = _two(out, "out")
            if out.shape != (rows, self.out_features):
                raise ValueError("out must be [rows][out_features]")
        if rows:
            launch(self.ctx, "kl_q8_linear_forward", self.h, codes.data_ptr(), ld, scales.data_ptr(), rows,
                   out.data_ptr(), _lib.DTYPE_BF16 if out.dtype == torch.bfloat16 else _lib.DTYPE_F32, ldo,
                   int(accumulate))
        return out
