"""Dropout from a counter-based generator: alone, with the residual sum, and with the residual sum
and the next block's RMSNorm, each in one pass. No mask is stored.

An element's random bits follow from (seed, offset, row, column) alone, row counting all leading
dimensions: Philox 4x32-10 under key ``seed``, 16 bits an element (``ts_dropout_rng`` in the C
header). They do not depend on the data type, strides or launch, so the backward forms the mask
again, and so can a recomputation in activation checkpointing.

``rng`` says where the numbers come from:

* ``(seed, offset)``: two integers in [0, 2^64). Different pairs give independent masks; a training
  loop keeps one seed and counts offsets.
* an int64 tensor [2] on the device, (seed, offset), read when the kernels run. This is the form
  for captured graphs: change the tensor between replays, or in the graph after the backward, and
  every replay draws new numbers. It must not change between a forward and its backward (autograd
  notices where it does).
* ``None``: a seed drawn from torch's CPU generator (``torch.manual_seed`` fixes it, checkpointing
  restores it), offset 0. Refused while a graph is captured, whose replays would repeat it.

The probability of dropping is p rounded to a multiple of 2^-16, kept elements are divided by the
exact probability of being kept; a dropped element is 0 whatever its value. Without training, or
where p rounds to 0, nothing is drawn.

The reference's dropout + RMSNorm kernel is kernels/layernorm_kernels.py:556-618.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import ops
from .layernorm_kernels import DEFAULT_EPS_RMS

__all__ = ["FusedDropoutFunction", "fused_dropout", "fused_dropout_add",
           "FusedDropoutAddRMSNormFunction", "fused_dropout_add_rms_layernorm",
           "FusedDropoutAddRMSNorm"]

RngLike = Union[None, Tuple[int, int], Tensor]


def _drop(what: str, p: float, training: bool) -> int:
    """The 16-bit limit below which an element is dropped."""
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p must be in [0, 1], got {p}")
    return round(p * 65536) if training else 0


def _rng(what: str, rng: RngLike, drop: int):
    if drop == 0:
        return (0, 0)
    if rng is None:
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what}: a captured graph would repeat its random numbers; pass "
                               "rng as a device tensor and change it between replays")
        return (int(torch.empty((), dtype=torch.int64, device="cpu").random_()), 0)
    if isinstance(rng, Tensor):
        if rng.dtype is not torch.int64 or rng.shape != (2,) or not rng.is_contiguous():
            raise ValueError(f"{what}: rng must be an int64 tensor [2], got {rng.dtype} "
                             f"{tuple(rng.shape)}")
        return rng
    seed, offset = rng
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError(f"{what}: seed and offset must be in [0, 2^64), got {rng}")
    return (int(seed), int(offset))


def _check_residual(what: str, x: Tensor, residual: Tensor) -> None:
    if residual.shape != x.shape:
        raise ValueError(f"{what}: residual {tuple(residual.shape)} != x {tuple(x.shape)}")
    if residual.dtype is not x.dtype:
        raise TypeError(f"{what}: residual dtype {residual.dtype} != x dtype {x.dtype}")


def _forward(x: Tensor, residual: Optional[Tensor], rng, state: Optional[Tensor]) -> Tensor:
    shape = x.shape
    if x.is_cuda and x.numel() == 0:
        return torch.empty(shape, dtype=x.dtype, device=x.device)
    cols = shape[-1] if shape else 1
    x, ldx = ops.rows_at(x, cols)
    residual, ldr = (None, 0) if residual is None else ops.rows_at(residual, cols)
    return ops.dropout_forward(x, ldx, residual, ldr, rng, state, shape)


class FusedDropoutFunction(torch.autograd.Function):
    """forward(x, residual or None, rng, drop) -> [residual +] dropout(x); differentiable in x and
    residual. rng is (seed, offset) or a device tensor, drop the 16-bit limit."""

    @staticmethod
    def forward(ctx, x: Tensor, residual: Optional[Tensor], rng, drop: int) -> Tensor:
        ctx.rng = ops.dropout_rng(rng, drop)
        state = rng if isinstance(rng, Tensor) else None
        if state is not None:
            ctx.save_for_backward(state)
        return _forward(x, residual, ctx.rng, state)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout: Tensor):
        dx = dout
        if ctx.needs_input_grad[0] and ctx.rng.drop:
            saved = ctx.saved_tensors
            dx = _forward(dout, None, ctx.rng, saved[0].contiguous() if saved else None)
        return (dx if ctx.needs_input_grad[0] else None,
                dout if ctx.needs_input_grad[1] else None, None, None)


def _dropout(what: str, x: Tensor, residual: Optional[Tensor], p: float, rng: RngLike,
             training: bool) -> Tensor:
    drop = _drop(what, p, training)
    if residual is not None:
        _check_residual(what, x, residual)
    rng = _rng(what, rng, drop)
    if ops.in_forward_ad() or (torch.is_grad_enabled() and (
            x.requires_grad or (residual is not None and residual.requires_grad))):
        return FusedDropoutFunction.apply(x, residual, rng, drop)
    return _forward(x, residual, ops.dropout_rng(rng, drop),
                    rng if isinstance(rng, Tensor) else None)


def fused_dropout(x: Tensor, p: float, rng: RngLike = None, training: bool = True) -> Tensor:
    """Dropout of x (fp32, bf16 or fp16, any shape and strides) with probability p, a new tensor.
    Differentiable in x; the module docstring says what rng is."""
    return _dropout("fused_dropout", x, None, p, rng, training)


def fused_dropout_add(x: Tensor, residual: Tensor, p: float, rng: RngLike = None,
                      training: bool = True) -> Tensor:
    """residual + dropout(x), fp32 arithmetic rounded once: a block's output joining the stream.
    Differentiable in both (the residual's gradient is the result's)."""
    return _dropout("fused_dropout_add", x, residual, p, rng, training)


def _norm_forward(x, residual, weight, eps, rng, state):
    shape, w = x.shape, weight.contiguous()
    x, ldx = ops.rows_at(x, shape[-1])
    residual, ldr = ops.rows_at(residual, shape[-1])
    y, h, rstd = ops.dropout_add_rmsnorm_forward(x, ldx, residual, ldr, w, eps, rng, state, shape)
    return y, h, w, rstd


class FusedDropoutAddRMSNormFunction(torch.autograd.Function):
    """forward(x, residual, weight, eps, rng, drop) -> (Y, residual_out); differentiable in the
    three tensors. The backward reads the rounded residual_out."""

    @staticmethod
    def forward(ctx, x: Tensor, residual: Tensor, weight: Tensor, eps: float, rng,
                drop: int) -> Tuple[Tensor, Tensor]:
        ctx.rng = ops.dropout_rng(rng, drop)
        state = rng if isinstance(rng, Tensor) else None
        y, h, w, rstd = _norm_forward(x, residual, weight, eps, ctx.rng, state)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, w, rstd, state)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: Optional[Tensor], dh: Optional[Tensor]):
        if dy is None and dh is None:
            return (None,) * 6
        h, w, rstd, state = ctx.saved_tensors
        needs = ctx.needs_input_grad[:3]
        if h.numel() == 0:
            return (*[torch.zeros(s, dtype=t.dtype, device=t.device) if need else None
                      for need, s, t in zip(needs, (h.shape, h.shape, w.shape), (h, h, w))],
                    None, None, None)
        shape, cols = h.shape, h.shape[-1]
        h, ldh = ops.rows_at(h, cols)
        (dy, lddy), (dh, lddh) = [(None, 0) if d is None else ops.rows_at(d, cols)
                                  for d in (dy, dh)]
        return (*ops.dropout_add_rmsnorm_backward(
            dy, lddy, dh, lddh, h, ldh, w.contiguous(), rstd.contiguous(), ctx.rng,
            None if state is None else state.contiguous(), needs, shape), None, None, None)


def fused_dropout_add_rms_layernorm(x: Tensor, residual: Tensor, weight: Tensor, p: float,
                                    eps: float = DEFAULT_EPS_RMS, rng: RngLike = None,
                                    training: bool = True) -> Tuple[Tensor, Tensor]:
    """The boundary between two blocks of a model trained with dropout:

        residual_out = residual + dropout(x)
        Y            = RMSNorm(residual_out) * weight

    Returns (Y, residual_out), both rounded once, Y from the unrounded sum. x and residual [..., H]
    of one dtype (fp32, bf16, fp16), weight [H] of that dtype or fp32, H at most 16384.
    Differentiable in all three with every gradient, where ``fused_add_rms_layernorm`` keeps to its
    counterpart and drops residual_out's and the weight's. The module docstring says what rng is."""
    what = "fused_dropout_add_rms_layernorm"
    drop = _drop(what, p, training)
    _check_residual(what, x, residual)
    if x.dim() < 1 or weight.shape != (x.shape[-1],) or x.shape[-1] == 0:
        raise ValueError(f"{what}: weight {tuple(weight.shape)} for x {tuple(x.shape)}")
    rng = _rng(what, rng, drop)
    args = (x, residual, weight, float(eps), rng, drop)
    if ops.in_forward_ad() or (torch.is_grad_enabled()
                               and (x.requires_grad or residual.requires_grad
                                    or weight.requires_grad)):
        return FusedDropoutAddRMSNormFunction.apply(*args)
    return _norm_forward(x, residual, weight, float(eps), ops.dropout_rng(rng, drop),
                         rng if isinstance(rng, Tensor) else None)[:2]


class FusedDropoutAddRMSNorm(nn.Module):
    """``fused_dropout_add_rms_layernorm`` with a weight; dropout follows the module's mode."""

    def __init__(self, hidden_size: int, p: float = 0.1, eps: float = DEFAULT_EPS_RMS,
                 device: Optional[torch.device] = None, dtype: torch.dtype = torch.float32):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"FusedDropoutAddRMSNorm: p must be in [0, 1], got {p}")
        self.hidden_size = hidden_size
        self.p = p
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden_size, device=device, dtype=dtype))

    def forward(self, x: Tensor, residual: Tensor, rng: RngLike = None) -> Tuple[Tensor, Tensor]:
        return fused_dropout_add_rms_layernorm(x, residual, self.weight, self.p, self.eps, rng,
                                               self.training)

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, p={self.p}, eps={self.eps}"
