"""The norms before and after a block, fused with the block's gate and the residual sum.

    n = rms_norm(h) * post_weight            (h itself without a norm behind the block)
    stream = residual_scale * residual + gate * n
    normed = rms_norm(stream) * pre_weight   (what the next block reads)

``rms_norm`` is the reference's RMSNorm (torchtitan/models/common/rmsnorm.py:14-50), the sum the residual addition
behind attention and feed-forward of its transformer blocks.  A plain pre-norm block has only
`pre_weight`; a block with norms on both sides, a learned scale per channel or a gate per sequence sets the
others.  On the GPU, bf16 and float32 run as one HIP kernel forward and one pass backward; elsewhere
the same formula runs in torch operations.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch
import torch.nn as nn

from .. import _lib, ops
from ..protocols import Module


class _ResidualRMSNorm(torch.autograd.Function):
    """On matrices; `gate` [n, dim] with n dividing the rows."""

    @staticmethod
    def forward(ctx, h, residual, post, gate, pre, scale, eps):
        stream, normed, rstd = ops.residual_norm(h, residual, post, gate, pre, scale, eps, want_rstd=True)
        ctx.save_for_backward(h, residual, post, gate, pre, rstd)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return stream, normed

    @staticmethod
    def backward(ctx, dstream, dnormed):
        if dstream is None and dnormed is None:
            return None, None, None, None, None, None, None
        *operands, rstd = ctx.saved_tensors
        with torch.no_grad():
            grads = ops.residual_norm_bwd(*operands, ctx.scale, rstd, dstream, dnormed, ctx.needs_input_grad[:5])
        # The operands are in the gradients too (but for a plain sum), whether or not the outputs' gradients have gradients.
        inside = operands[2] is not None or operands[3] is not None or dnormed is not None
        if torch.is_grad_enabled() and (inside or any(d is not None and d.requires_grad for d in (dstream, dnormed))):
            grads = [None if g is None else _Refusing.apply(g, torch.empty(0, requires_grad=True)) for g in grads]
        return *grads, None, None


class _Refusing(torch.autograd.Function):
    """Gradients that cannot be differentiated again: asking for it is an error."""

    @staticmethod
    def forward(ctx, grad, _):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("this operator's gradients cannot be differentiated again")


def _in_torch_ops(h, residual, post, gate, pre, scale, eps):
    wide = torch.promote_types(torch.promote_types(h.dtype, residual.dtype), torch.float32)

    def normalised(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)

    n = h.to(wide)
    if post is not None:
        n = normalised(n) * post.to(wide)
    if gate is not None:
        n = n * gate.to(wide)
    total = residual.to(wide) * scale + n
    normed = None if pre is None else (normalised(total) * pre.to(wide)).to(h.dtype)
    return total.to(residual.dtype), normed


def _gate_as_matrix(gate: torch.Tensor, shape: torch.Size) -> torch.Tensor:
    """[n, dim] of a gate of `shape`'s width that is shared by all rows ([dim]) or by the rows of its leading
    dimensions ([batch, 1, dim], [batch, sequence, dim] of [batch, sequence, dim])."""
    lead, dim = list(gate.shape[:-1]), shape[-1]
    while lead and lead[-1] == 1:
        lead.pop()
    if gate.dim() == 0 or gate.shape[-1] != dim or gate.dim() > len(shape) or lead != list(shape[:len(lead)]) or (
            lead and gate.dim() != len(shape)):
        raise ValueError(f"gate must be [{dim}] or have the leading dimensions of {tuple(shape)} up to one and ones behind "
                         f"it, got {tuple(gate.shape)}")
    return gate.reshape(-1, dim)


def residual_rms_norm(h: torch.Tensor, residual: torch.Tensor, *, post_weight: torch.Tensor | None = None,
                      gate: torch.Tensor | None = None, pre_weight: torch.Tensor | None = None,
                      residual_scale: float = 1.0, eps: float = 1e-5):
    """(stream, normed): ``residual_scale * residual + gate * (rms_norm(h) * post_weight)`` in residual's type, and
    ``rms_norm(stream) * pre_weight`` in h's (None without `pre_weight`), all in float32, each rounded once.

    h: output of a block, residual: the stream around it, both [..., dim]; h may be bf16 where the stream is float32.
    post_weight, pre_weight: [dim].  gate: [dim], or with h's dimensions: its leading ones up to some point, ones
    behind it, dim ([batch, 1, dim]: a row for every sequence).  The gradients cannot be differentiated again."""
    tracing = torch.compiler.is_compiling()
    if not tracing and ops.native_rows(h):
        out = _lib.blocks().residual_rms_norm(h, residual, post_weight, gate, pre_weight, residual_scale, eps)
        if out is not None:
            return out
    dim = h.shape[-1] if h.dim() else 0
    if h.dim() == 0 or residual.shape != h.shape:
        raise ValueError(f"h and residual must have one shape with a last dimension, got {tuple(h.shape)} and {tuple(residual.shape)}")
    operands = [t for t in (h, residual, post_weight, gate, pre_weight) if t is not None]
    if not all(t.is_floating_point() for t in operands):
        raise TypeError("operands must be floating-point tensors")
    if any(t.device != h.device for t in operands):
        raise ValueError(f"operands on different devices: {', '.join(str(t.device) for t in operands)}")
    for name, w in (("post_weight", post_weight), ("pre_weight", pre_weight)):
        if w is not None and w.shape != (dim,):
            raise ValueError(f"{name} must be [{dim}], got {tuple(w.shape)}")
    rows = None if gate is None else _gate_as_matrix(gate, h.shape)
    ours = not ops.wrapped(*operands) and all(t.is_cuda and t.dtype in ops.ROW_TYPES for t in operands) and (
        h.dtype == torch.bfloat16 or residual.dtype == torch.float32)
    if not ours or h.numel() == 0 or not (tracing or ops.plain_rows(*operands)):
        return _in_torch_ops(h, residual, post_weight, gate, pre_weight, residual_scale, eps)
    h2, r2 = h.reshape(-1, dim), residual.reshape(-1, dim)
    if tracing:
        from ..compiled import residual_norm_traced  # the same launches as nodes of the graph

        stream, normed = residual_norm_traced(h2, r2, post_weight, rows, pre_weight, float(residual_scale), float(eps))
    elif torch.is_grad_enabled() and any(t.requires_grad for t in operands):
        stream, normed = _ResidualRMSNorm.apply(h2, r2, post_weight, rows, pre_weight, residual_scale, eps)
    else:
        stream, normed, _ = ops.residual_norm(h2, r2, post_weight, rows, pre_weight, residual_scale, eps)
    return stream.view(h.shape), None if normed is None else normed.view(h.shape)


class ResidualRMSNorm(Module):
    """The seam between two blocks as a module: ``forward(h, residual) -> (stream, normed)``.

    `post_norm`: a norm behind the block; `gate`: a learned scale per channel, from `gate_init`; `pre_norm`: the norm in front
    of the next block (without it, behind the last one, `normed` is None)."""

    @dataclass(kw_only=True, slots=True)
    class Config(Module.Config):
        dim: int = field(init=False)  # supplied by build(dim=...)
        post_norm: bool = False
        gate: bool = False
        gate_init: float = 1.0
        pre_norm: bool = True
        residual_scale: float = 1.0
        eps: float = 1e-5

    def __init__(self, config: Config):
        super().__init__()
        vector = lambda wanted: nn.Parameter(torch.ones(config.dim)) if wanted else None
        self.post_weight, self.gate, self.pre_weight = (vector(w) for w in (config.post_norm, config.gate, config.pre_norm))
        self.residual_scale, self.eps, self._gate_init = config.residual_scale, config.eps, config.gate_init
        self.init_weights()

    def forward(self, h: torch.Tensor, residual: torch.Tensor):
        return residual_rms_norm(h, residual, post_weight=self.post_weight, gate=self.gate, pre_weight=self.pre_weight,
                                 residual_scale=self.residual_scale, eps=self.eps)

    def init_weights(self, **kwargs) -> None:
        for w, value in ((self.post_weight, 1.0), (self.gate, self._gate_init), (self.pre_weight, 1.0)):
            if w is not None:
                nn.init.constant_(w, value)
