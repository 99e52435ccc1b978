"""Drop-in counterparts of TrainScale's ``kernels/layernorm_kernels.py`` RMSNorm ops.

Reference (``data_pipeline/trainer/``):

* ``RMSLayerNormFunction`` (kernels/layernorm_kernels.py:676-807):
  forward(X, weight, eps, compute_weight_grad) -> Y; backward -> (dX, dW, None, None).
  Its forward rounds x * rstd to the weight dtype before the weight product
  (y = x_norm.to(w.dtype) * w, :189-194): with a 16-bit weight that is a
  second rounding, which the ROUND_TWICE kernel mode reproduces; with an fp32
  weight the product is formed in fp32 and rounded once into the data dtype.
* ``rms_layernorm`` and its alias ``fast_rms_layernorm`` (:1054-1070, :1141).
* ``RMSNorm`` module (:1150-1189).
* ``FusedAddRMSLayerNormFunction`` (:949-1047), ``fused_add_rms_layernorm``
  (:1094-1121) and the ``FusedRMSNorm`` module (:1241-1269): h = X + residual
  in fp32, Y = RMSNorm(h) with the same round-twice numerics, and h rounded to
  the data dtype as ``residual_out``. As in the reference, backward returns
  the same dX for X and residual, computed from dY and the rounded h; the
  gradient arriving at ``residual_out`` is not added and the weight gets no
  gradient (the reference's backward returns None for it).

Not in the reference: ``FusedSandwichRMSNormFunction``, ``fused_sandwich_rms_layernorm`` and the
``FusedSandwichRMSNorm`` module, the boundary between two blocks of models that normalise before
and after each block: the norm of a block's output, its gate, the residual sum and the next
block's norm in one pass, with every gradient.

LayerNorm/Welford and dropout+RMS are not part of this layer.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import ops

DEFAULT_EPS_RMS = 1e-6

__all__ = [
    "RMSLayerNormFunction",
    "rms_layernorm",
    "fast_rms_layernorm",
    "RMSNorm",
    "FusedAddRMSLayerNormFunction",
    "fused_add_rms_layernorm",
    "FusedRMSNorm",
    "FusedSandwichRMSNormFunction",
    "fused_sandwich_rms_layernorm",
    "FusedSandwichRMSNorm",
    "DEFAULT_EPS_RMS",
]


class RMSLayerNormFunction(torch.autograd.Function):
    """RMSNorm with the reference's rounding: y = round(round(x*rstd) * w) for 16-bit w."""

    @staticmethod
    def forward(ctx, X: Tensor, weight: Tensor, eps: float = DEFAULT_EPS_RMS,
                compute_weight_grad: bool = True) -> Tensor:
        orig_shape = X.shape
        x2d, ldx = ops.as_rows(X)
        y, rstd = ops.rmsnorm_forward(x2d, ldx, weight, eps, ops.ROUND_TWICE)
        ctx.save_for_backward(x2d, weight, rstd)
        ctx.orig_shape = orig_shape
        ctx.compute_weight_grad = compute_weight_grad
        return y.view(orig_shape)

    @staticmethod
    def backward(ctx, dY: Tensor) -> Tuple[Optional[Tensor], ...]:
        x2d, weight, rstd = ctx.saved_tensors
        (x2d, ldx), (dy2d, lddy) = ops.as_rows(x2d), ops.as_rows(dY)
        need_dw = bool(ctx.compute_weight_grad and weight is not None and weight.requires_grad)
        dx, dw = ops.rmsnorm_backward(dy2d, lddy, x2d, ldx, weight, rstd, need_dw=need_dw)
        return dx.view(ctx.orig_shape), dw, None, None


def rms_layernorm(X: Tensor, weight: Tensor, eps: float = DEFAULT_EPS_RMS) -> Tensor:
    """RMSNorm (reference: kernels/layernorm_kernels.py:1054-1070)."""
    return RMSLayerNormFunction.apply(X, weight, eps, True)


fast_rms_layernorm = rms_layernorm


class _RMSNormNoWeight(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X: Tensor, eps: float) -> Tensor:
        orig_shape = X.shape
        x2d, ldx = ops.as_rows(X)
        y, rstd = ops.rmsnorm_forward(x2d, ldx, None, eps, ops.ROUND_ONCE)
        ctx.save_for_backward(x2d, rstd)
        ctx.orig_shape = orig_shape
        return y.view(orig_shape)

    @staticmethod
    def backward(ctx, dY: Tensor):
        x2d, rstd = ctx.saved_tensors
        (x2d, ldx), (dy2d, lddy) = ops.as_rows(x2d), ops.as_rows(dY)
        dx, _ = ops.rmsnorm_backward(dy2d, lddy, x2d, ldx, None, rstd, need_dw=False)
        return dx.view(ctx.orig_shape), None


class RMSNorm(nn.Module):
    """RMSNorm module (reference: kernels/layernorm_kernels.py:1150-1189)."""

    def __init__(self, hidden_size: int, eps: float = DEFAULT_EPS_RMS,
                 elementwise_affine: bool = True, device: Optional[torch.device] = None,
                 dtype: torch.dtype = torch.float32):
        super().__init__()
        self.hidden_size = hidden_size
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)

    def forward(self, X: Tensor) -> Tensor:
        if self.elementwise_affine:
            return rms_layernorm(X, self.weight, self.eps)
        return _RMSNormNoWeight.apply(X, self.eps)

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, eps={self.eps}, elementwise_affine={self.elementwise_affine}"


class FusedAddRMSLayerNormFunction(torch.autograd.Function):
    """Residual add + RMSNorm in one pass (reference: kernels/layernorm_kernels.py:949-1047).

    forward(X, residual, weight, eps, store_residual) -> (Y, residual_out or None).
    One kernel reads X and residual once and writes Y and h = X + residual
    (rounded); h is also kept for backward when a gradient is needed and
    store_residual is False (the reference then recomputes X + residual).
    """

    @staticmethod
    def forward(ctx, X: Tensor, residual: Tensor, weight: Tensor, eps: float = DEFAULT_EPS_RMS,
                store_residual: bool = True) -> Tuple[Tensor, Optional[Tensor]]:
        orig_shape = X.shape
        if residual.shape != X.shape:
            raise ValueError(f"fused_add_rms_layernorm: residual {tuple(residual.shape)} != "
                             f"X {tuple(X.shape)}")
        x2d, ldx = ops.as_rows(X)
        r2d, ldr = ops.as_rows(residual)
        need_h = store_residual or any(ctx.needs_input_grad[:2])
        y, h, rstd = ops.add_rmsnorm_forward(x2d, ldx, r2d, ldr, weight, eps, ops.ROUND_TWICE,
                                             store_h=need_h)
        ctx.save_for_backward(h, weight, rstd)
        ctx.orig_shape = orig_shape
        return y.view(orig_shape), (h.view(orig_shape) if store_residual else None)

    @staticmethod
    def backward(ctx, dY: Tensor, _unused: Optional[Tensor]):
        h, weight, rstd = ctx.saved_tensors
        (h, ldh), (dy2d, lddy) = ops.as_rows(h), ops.as_rows(dY)
        dx, _ = ops.rmsnorm_backward(dy2d, lddy, h, ldh, weight, rstd, need_dw=False)
        dx = dx.view(ctx.orig_shape)
        return dx, dx, None, None, None


def fused_add_rms_layernorm(X: Tensor, residual: Tensor, weight: Tensor,
                            eps: float = DEFAULT_EPS_RMS, return_residual: bool = False):
    """Y = RMSNorm(X + residual) * weight (reference: kernels/layernorm_kernels.py:1094-1121);
    with return_residual also returns X + residual."""
    Y, residual_out = FusedAddRMSLayerNormFunction.apply(X, residual, weight, eps,
                                                         return_residual)
    if return_residual:
        return Y, residual_out
    return Y


class FusedRMSNorm(nn.Module):
    """Residual add + RMSNorm module (reference: kernels/layernorm_kernels.py:1241-1269)."""

    def __init__(self, hidden_size: int, eps: float = DEFAULT_EPS_RMS,
                 device: Optional[torch.device] = None, dtype: torch.dtype = torch.float32):
        super().__init__()
        self.hidden_size = hidden_size
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))

    def forward(self, X: Tensor, residual: Tensor, return_residual: bool = False):
        return fused_add_rms_layernorm(X, residual, self.weight, self.eps, return_residual)

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, eps={self.eps}"


def _gate_rows(gate: Tensor, X: Tensor) -> Tensor:
    """A gate that broadcasts over X as [groups, H], group g covering equal runs of X's rows."""
    shape, lead = tuple(gate.shape), tuple(X.shape[:-1])
    if not shape or shape[-1] != X.shape[-1]:
        raise ValueError(f"fused_sandwich_rms_layernorm: gate {shape} for X {tuple(X.shape)}")
    if len(shape) > 1:
        # the leading dimensions of X, then ones: the rows of a group are neighbours
        own = len(shape) == X.dim()
        k = 0
        while own and k < len(lead) and shape[k] == lead[k]:
            k += 1
        if not own or any(n != 1 for n in shape[k:-1]):
            raise ValueError(f"fused_sandwich_rms_layernorm: gate {shape} for X {tuple(X.shape)}: "
                             "expected [H], or X's leading dimensions followed by ones and H")
    return gate.reshape(-1, shape[-1]).contiguous()


def _sandwich_forward(X, residual, post_weight, pre_weight, gate, eps, residual_scale,
                      weight_offset):
    """The results and what the backward needs of one call: (n, h, saved tensors)."""
    if residual.shape != X.shape:
        raise ValueError(f"fused_sandwich_rms_layernorm: residual {tuple(residual.shape)} != "
                         f"X {tuple(X.shape)}")
    g2d = None if gate is None else _gate_rows(gate, X)
    y2d, ldy = ops.as_rows(X)
    x2d, ldx = ops.as_rows(residual)
    post, pre = post_weight.contiguous(), pre_weight.contiguous()
    n, h, rstd = ops.sandwich_norm_forward(y2d, ldy, x2d, ldx, post, pre, g2d, residual_scale,
                                           weight_offset, eps, X.shape)
    return n, h, (y2d, x2d, post, pre, g2d, rstd)


class FusedSandwichRMSNormFunction(torch.autograd.Function):
    """forward(X, residual, post_weight, pre_weight, gate, eps, residual_scale, weight_offset) ->
    (Y, residual_out); differentiable in the five tensors."""

    @staticmethod
    def forward(ctx, X: Tensor, residual: Tensor, post_weight: Tensor, pre_weight: Tensor,
                gate: Optional[Tensor] = None, eps: float = DEFAULT_EPS_RMS,
                residual_scale: float = 1.0, weight_offset: float = 0.0) -> Tuple[Tensor, Tensor]:
        n, h, saved = _sandwich_forward(X, residual, post_weight, pre_weight, gate, eps,
                                        residual_scale, weight_offset)
        ctx.save_for_backward(*saved)
        ctx.set_materialize_grads(False)
        ctx.cfg = (X.shape, None if gate is None else gate.shape, residual_scale,
                   weight_offset)
        return n, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dn: Optional[Tensor], dh: Optional[Tensor]):
        if dn is None and dh is None:
            return (None,) * 8
        y2d, x2d, post, pre, g2d, rstd = ctx.saved_tensors
        shape, gate_shape, residual_scale, weight_offset = ctx.cfg
        if y2d.shape[0] == 0:
            return (*[None if t is None or not need else torch.zeros(s, dtype=t.dtype,
                                                                      device=t.device)
                      for t, need, s in zip((y2d, x2d, post, pre, g2d), ctx.needs_input_grad,
                                            (shape, shape, post.shape, pre.shape, gate_shape))],
                    None, None, None)
        # hooks on saved tensors may give them back with other strides
        (y2d, ldy), (x2d, ldx) = ops.as_rows(y2d), ops.as_rows(x2d)
        post, pre, rstd = post.contiguous(), pre.contiguous(), rstd.contiguous()
        g2d = None if g2d is None else g2d.contiguous()
        (dn, lddn), (dh, lddh) = [(None, 0) if d is None else ops.as_rows(d) for d in (dn, dh)]
        return (*ops.sandwich_norm_backward(
            dn, lddn, dh, lddh, y2d, ldy, x2d, ldx, post, pre, g2d, rstd, residual_scale,
            weight_offset, ctx.needs_input_grad, shape, gate_shape), None, None, None)


def fused_sandwich_rms_layernorm(X: Tensor, residual: Tensor, post_weight: Tensor,
                                 pre_weight: Tensor, gate: Optional[Tensor] = None,
                                 eps: float = DEFAULT_EPS_RMS, residual_scale: float = 1.0,
                                 weight_offset: float = 0.0) -> Tuple[Tensor, Tensor]:
    """The boundary between two blocks with norms before and after each: X is a block's output,
    residual the stream beside it.

        residual_out = residual_scale * residual + gate * RMSNorm(X; post_weight)
        Y            = RMSNorm(residual_out; pre_weight)

    Returns (Y, residual_out): the next block's input and the stream. RMSNorm(x; w) is
    x * rstd * (weight_offset + w); weight_offset 1 is for weights kept as their difference from
    1. gate: None, [H], or X's leading dimensions followed by ones and H ([B, 1, H] for X
    [B, S, H]: one gate for each sequence; the backward holds four fp32 rows of H for each gate
    row, so a gate for every token is possible but costly). fp32 arithmetic; Y comes from the unrounded sum and
    both results are rounded once. The weights share one dtype, X's or fp32; the gate has X's
    dtype or fp32. Differentiable in X, residual, both weights and the gate. H is at most 16384
    for 16-bit X, 8192 for fp32."""
    args = (X, residual, post_weight, pre_weight, gate, float(eps), float(residual_scale),
            float(weight_offset))
    if ops.in_forward_ad() or (torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in args[:5])):
        return FusedSandwichRMSNormFunction.apply(*args)
    return _sandwich_forward(*args)[:2]


class FusedSandwichRMSNorm(nn.Module):
    """The norm after a block and the one before the next, with the residual sum between them
    (``fused_sandwich_rms_layernorm``). layer_gate adds a learned gate of hidden_size channels,
    initialised to gate_init."""

    def __init__(self, hidden_size: int, eps: float = DEFAULT_EPS_RMS, weight_offset: float = 0.0,
                 residual_scale: float = 1.0, layer_gate: bool = False, gate_init: float = 1.0,
                 device: Optional[torch.device] = None, dtype: torch.dtype = torch.float32):
        super().__init__()
        self.hidden_size = hidden_size
        self.eps = eps
        self.weight_offset = weight_offset
        self.residual_scale = residual_scale

        def param(value):
            return nn.Parameter(torch.full((hidden_size,), value, device=device, dtype=dtype))

        self.post_weight = param(1.0 - weight_offset)
        self.pre_weight = param(1.0 - weight_offset)
        if layer_gate:
            self.gate = param(gate_init)
        else:
            self.register_parameter("gate", None)

    def forward(self, X: Tensor, residual: Tensor,
                gate: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
        """gate: a conditioning gate, where the module has no learned one."""
        if gate is not None and self.gate is not None:
            raise ValueError("FusedSandwichRMSNorm: the module has a gate of its own")
        return fused_sandwich_rms_layernorm(X, residual, self.post_weight, self.pre_weight,
                                            self.gate if gate is None else gate, self.eps,
                                            self.residual_scale, self.weight_offset)

    def extra_repr(self) -> str:
        return (f"{self.hidden_size}, eps={self.eps}, weight_offset={self.weight_offset}, "
                f"residual_scale={self.residual_scale}")
