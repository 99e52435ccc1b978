"""Token embedding with scaling, and its gradient by sorted tokens.

``scaled_embedding(input_ids, weight, scale)`` is ``scale * weight[input_ids]``, the lookup that
starts a model (with the scale of models whose embeddings are multiplied by sqrt(hidden)). Its
gradient is dense, [V, H] in the weight's dtype, as the fused linear cross-entropy's for the tied
LM head: the tokens are sorted by id and each row is summed once in fp32, in an order that the
ids alone fix, where torch's sums depend on timing or on the batch's order.

Ids outside [0, V) give rows of NaN and no gradient (the layer's rule for labels out of range:
nothing is read out of bounds, and the loss shows it).
"""
from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import ops

__all__ = ["ScaledEmbeddingFunction", "scaled_embedding", "ScaledEmbedding"]


def _forward(input_ids: Tensor, weight: Tensor, scale: float, padding_idx: Optional[int]):
    """(result, contiguous int64 ids, padding row or -1), after the checks of the arguments."""
    if weight.dim() != 2 or weight.shape[1] == 0:
        raise ValueError(f"scaled_embedding: weight must be [V, H], got {tuple(weight.shape)}")
    if input_ids.dtype is not torch.int64:
        if input_ids.dtype is not torch.int32:
            raise TypeError(f"scaled_embedding: ids must be int64 or int32, got {input_ids.dtype}")
        input_ids = input_ids.to(torch.int64)
    if not math.isfinite(scale):
        raise ValueError(f"scaled_embedding: scale must be finite, got {scale}")
    if padding_idx is None:
        padding_idx = -1
    else:
        rows = weight.shape[0]
        if not -rows <= padding_idx < rows:
            raise ValueError(f"scaled_embedding: padding_idx {padding_idx} for {rows} rows")
        padding_idx %= rows
    ids = input_ids.contiguous()
    if weight.is_contiguous():
        w2d, ldw = weight, weight.shape[1]
    else:
        w2d, ldw = ops.as_rows(weight)
    return ops.embedding_forward(ids, w2d, ldw, scale), ids, padding_idx


class ScaledEmbeddingFunction(torch.autograd.Function):
    """forward(input_ids [...], weight [V, H], scale, padding_idx) -> [..., H]; backward gives the
    weight's gradient."""

    @staticmethod
    def forward(ctx, input_ids: Tensor, weight: Tensor, scale: float = 1.0,
                padding_idx: Optional[int] = None) -> Tensor:
        out, ids, padding_idx = _forward(input_ids, weight, scale, padding_idx)
        ctx.save_for_backward(ids)
        ctx.cfg = (weight.shape[0], scale, padding_idx)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout: Tensor):
        if not ctx.needs_input_grad[1]:
            return None, None, None, None
        ids = ctx.saved_tensors[0].contiguous()  # hooks may give it back with other strides
        rows, scale, padding_idx = ctx.cfg
        d2d, ldd = ops.as_rows(dout)
        return None, ops.embedding_backward(ids, d2d, ldd, rows, scale, padding_idx), None, None


def scaled_embedding(input_ids: Tensor, weight: Tensor, scale: float = 1.0,
                     padding_idx: Optional[int] = None) -> Tensor:
    """scale * weight[input_ids]: ids [...] int64 or int32, weight [V, H] fp32/bf16/fp16; the
    result is [..., H] in the weight's dtype, differentiable in weight. Tokens equal to
    padding_idx (negative counts from the end) get their row but give it no gradient."""
    if (weight.requires_grad and torch.is_grad_enabled()) or ops.in_forward_ad():
        return ScaledEmbeddingFunction.apply(input_ids, weight, float(scale), padding_idx)
    return _forward(input_ids, weight, float(scale), padding_idx)[0]


class ScaledEmbedding(nn.Module):
    """An embedding layer on ``scaled_embedding``, initialised as torch's ``nn.Embedding``."""

    def __init__(self, num_embeddings: int, embedding_dim: int, scale: float = 1.0,
                 padding_idx: Optional[int] = None, device: Optional[torch.device] = None,
                 dtype: Optional[torch.dtype] = None):
        super().__init__()
        if padding_idx is not None:
            if not -num_embeddings <= padding_idx < num_embeddings:
                raise ValueError(f"ScaledEmbedding: padding_idx {padding_idx} for "
                                 f"{num_embeddings} rows")
            padding_idx %= num_embeddings
        self.num_embeddings = num_embeddings
        self.embedding_dim = embedding_dim
        self.scale = float(scale)
        self.padding_idx = padding_idx
        self.weight = nn.Parameter(torch.empty(num_embeddings, embedding_dim, device=device,
                                               dtype=dtype))
        with torch.no_grad():
            self.weight.normal_()
            if padding_idx is not None:
                self.weight[padding_idx].zero_()

    def forward(self, input_ids: Tensor) -> Tensor:
        return scaled_embedding(input_ids, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return (f"{self.num_embeddings}, {self.embedding_dim}, scale={self.scale}, "
                f"padding_idx={self.padding_idx}")
