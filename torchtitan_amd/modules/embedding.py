"""Token embedding with a scale, and its dense gradient by sorted tokens.

``Embedding`` is the first layer of the reference's decoder (torchtitan/models/common/decoder.py:59-155) as
a module that also satisfies the ``Module`` protocol; ``scaled_embedding`` is the function under it.  On the
GPU, bf16 and float32 tables run as one HIP kernel forward and sorted tokens backward; elsewhere
the same formula runs in torch operations.
"""
from __future__ import annotations

from dataclasses import dataclass, field

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _lib, ops
from ..protocols import Module


class _ScaledEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx, first_row, dtype):
        ctx.save_for_backward(ids)
        ctx.call = (weight.shape[0], scale, first_row, padding_idx, weight.dtype)
        return ops.embedding_fwd(ids, weight, scale, first_row, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        (ids,) = ctx.saved_tensors
        return None, ops.embedding_bwd(ids, dout, *ctx.call), None, None, None, None


def _in_torch_ops(ids, weight, scale, padding_idx, first_row, dtype):
    wide = torch.promote_types(weight.dtype, torch.float32)
    row = ids.long() - first_row
    inside = (row >= 0) & (row < weight.shape[0])
    if weight.shape[0] == 0:  # (the sum of no rows: zeros with a gradient of no rows)
        return weight.sum(0).to(dtype).expand(*ids.shape, weight.shape[1]).clone()
    if torch.is_grad_enabled() and weight.requires_grad:  # equal ids' gradients are added up in the table's type
        weight = weight.to(wide)
    values = weight[torch.where(inside, row, 0)].to(wide) * scale
    if padding_idx is not None:
        values = torch.where((ids == padding_idx)[..., None], values.detach(), values)
    return torch.where(inside[..., None], values, 0.0).to(dtype)


def scaled_embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, *, padding_idx: int | None = None,
                     first_row: int = 0, dtype: torch.dtype | None = None) -> torch.Tensor:
    """[*ids.shape, dim] in `dtype` (weight's without one): ``scale * weight[ids - first_row]``, formed in float32 and
    rounded once.

    ids: int64 or int32, any shape.  An id outside the table's rows [first_row, first_row + len(weight)) gives a row of
    zeros and no gradient: the rows of a vocabulary shard add up over the shards.  Tokens whose id is
    `padding_idx` have their row, but no gradient.  weight: [rows, dim].  The gradient is dense, sums of equal ids in
    float32 in an order that depends on the ids alone; it cannot be differentiated again."""
    tracing = torch.compiler.is_compiling()
    if not tracing and (dtype is None or dtype in ops.ROW_TYPES) and ops.native_rows(weight):
        out = _lib.blocks().scaled_embedding(ids, weight, scale, padding_idx, first_row,
                                             (dtype or weight.dtype) == torch.float32)
        if out is not None:
            return out
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must be int64 or int32, got {ids.dtype}")
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"weight must be a floating-point matrix, got {tuple(weight.shape)} {weight.dtype}")
    if ids.device != weight.device:
        raise ValueError(f"ids on {ids.device}, weight on {weight.device}")
    dtype = dtype or weight.dtype
    if (tracing and weight.is_cuda and weight.dtype in ops.ROW_TYPES and dtype in ops.ROW_TYPES
            and not ops.wrapped(weight, ids)):
        from .. import compiled  # noqa: F401  (the same launches as nodes of the graph)

        return torch.ops.torchtitan_amd.embedding_fwd(ids, weight, float(scale), padding_idx, first_row, dtype)
    if tracing or not (ops.plain_rows(weight) and type(ids) is torch.Tensor and dtype in ops.ROW_TYPES):
        return _in_torch_ops(ids, weight, scale, padding_idx, first_row, dtype)
    if torch.is_grad_enabled() and weight.requires_grad:
        return _ScaledEmbedding.apply(ids, weight, scale, padding_idx, first_row, dtype)
    return ops.embedding_fwd(ids, weight, scale, first_row, dtype)


class Embedding(nn.Embedding, Module):
    """``nn.Embedding`` built from a config, times `scale` (for instance the square root of the width)."""

    @dataclass(kw_only=True, slots=True)
    class Config(Module.Config):
        # sizes are not constructor arguments of the config: the parent model supplies them
        num_embeddings: int = field(init=False)
        embedding_dim: int = field(init=False)
        padding_idx: int | None = None
        scale: float = 1.0
        init_std: float = 1.0

    def __init__(self, config: Config):
        nn.Embedding.__init__(self, config.num_embeddings, config.embedding_dim, padding_idx=config.padding_idx)
        self.scale = config.scale
        self._init_std = config.init_std

    def forward(self, ids: torch.Tensor) -> torch.Tensor:
        return scaled_embedding(ids, self.weight, self.scale, padding_idx=self.padding_idx)

    def init_weights(self, **kwargs) -> None:
        override = kwargs.pop("init_std", None)
        nn.init.normal_(self.weight, mean=0.0, std=self._init_std if override is None else override)
        if self.padding_idx is not None:
            with torch.no_grad():
                self.weight[self.padding_idx].zero_()
