"""Gated feed-forward block: both projections, the activation and the product in one kernel.

``fused_gated_mlp(x, gate, up, down)`` is ``(act(x gate^T) * (x up^T)) down^T``, the block whose
elementwise part alone is ``Fast_SwiGLU``; ``fused_gated_linear`` is the same without the down
projection. Weights have ``nn.Linear``'s layout. bf16 and fp16; the sums are fp32, and what lies
between the products (the gated product forward, the gradients of both projections backward) is
rounded to the data type once, where the unfused block rounds g, u, act(g) and the product.

Where gradients of x, gate or up will follow, the forward keeps the two factors of the backward in
fp32 (up * act'(gate) and act(gate), 8 N F bytes), so that no rounding of the projections adds to the
gradients'; for down's it keeps the gated product (2 N F); beside them x and the weights. Otherwise
only the gated product is formed.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import ops

__all__ = ["ACTIVATIONS", "GatedMLPFunction", "fused_gated_linear", "fused_gated_mlp",
           "FusedGatedMLP"]

# activation -> TS_ACT_*
ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}


def _check(x: Tensor, gate: Tensor, up: Tensor, down: Optional[Tensor], activation: str) -> int:
    what = "fused_gated_linear" if down is None else "fused_gated_mlp"
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"{what}: unknown activation {activation!r} ({', '.join(ACTIVATIONS)})")
    dtype = x.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"{what}: x must be bfloat16 or float16, got {dtype}")
    for name, t in (("gate", gate), ("up", up), ("down", down)):
        if t is not None and t.dtype is not dtype:
            raise TypeError(f"{what}: {name} weight dtype {t.dtype} != x dtype {dtype}")
    xs, gs = x.shape, gate.shape
    if len(xs) < 1 or len(gs) != 2 or gs[1] != xs[-1] or 0 in gs:
        raise ValueError(f"{what}: gate weight {tuple(gs)} for x {tuple(xs)}")
    if up.shape != gs:
        raise ValueError(f"{what}: up weight {tuple(up.shape)} != gate weight {tuple(gs)}")
    if down is not None:
        ds = down.shape
        if len(ds) != 2 or ds[1] != gs[0] or ds[0] == 0:
            raise ValueError(f"{what}: down weight {tuple(ds)} for a gate weight {tuple(gs)}")
    return code


def _2d(t: Tensor) -> Tensor:
    return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _forward(x: Tensor, gate: Tensor, up: Tensor, down: Optional[Tensor], activation: str,
             keep: bool):
    """(result, the activation's code, the backward's factors, gated product)."""
    code = _check(x, gate, up, down, activation)
    factors, act, out = ops.gated_mlp_forward(_2d(x), gate, up, down, code, keep)
    if x.dim() != 2:
        out = out.view(*x.shape[:-1], out.shape[1])
    return out, code, factors, act


class GatedMLPFunction(torch.autograd.Function):
    """forward(x [..., H], gate [F, H], up [F, H], down [O, F] or None, activation) -> [..., O] or
    [..., F]; differentiable in the four tensors."""

    @staticmethod
    def forward(ctx, x: Tensor, gate: Tensor, up: Tensor, down: Optional[Tensor],
                activation: str) -> Tensor:
        needs = ctx.needs_input_grad
        out, ctx.code, factors, act = _forward(x, gate, up, down, activation, any(needs[:3]))
        ctx.save_for_backward(x, gate, up, down, factors, act if needs[3] else None)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout: Tensor):
        x, gate, up, down, factors, act = ctx.saved_tensors
        grads = ops.gated_mlp_backward(
            _2d(x), gate, up, down, ctx.code, factors, act, _2d(dout), ctx.needs_input_grad)
        if grads[0] is not None and x.dim() != 2:
            grads[0] = grads[0].view(x.shape)
        return (*grads, None)


def _apply(x: Tensor, gate: Tensor, up: Tensor, down: Optional[Tensor],
           activation: str) -> Tensor:
    if ops.in_forward_ad() or (torch.is_grad_enabled() and (
            x.requires_grad or gate.requires_grad or up.requires_grad
            or (down is not None and down.requires_grad))):
        return GatedMLPFunction.apply(x, gate, up, down, activation)
    return _forward(x, gate, up, down, activation, False)[0]


def fused_gated_linear(x: Tensor, gate: Tensor, up: Tensor, activation: str = "silu") -> Tensor:
    """act(x @ gate.T) * (x @ up.T): x [..., H], gate and up [F, H], all bf16 or all fp16; the
    result is [..., F]. activation: "silu", "gelu" (the error function's form), "gelu_tanh" or
    "relu". Differentiable in all three. Any sizes and strides; sizes or row strides that are not
    multiples of 8, or rows that do not start at 16 bytes, cost a copy of that operand (one launch for
    all of them)."""
    return _apply(x, gate, up, None, activation)


def fused_gated_mlp(x: Tensor, gate: Tensor, up: Tensor, down: Tensor,
                    activation: str = "silu") -> Tensor:
    """fused_gated_linear(x, gate, up, activation) @ down.T with down [O, F]: [..., O].
    Differentiable in all four tensors, in one backward whose gradients of the projections never
    exist unfused."""
    return _apply(x, gate, up, down, activation)


def watched(layer: nn.Module) -> bool:
    """Whether calling this module does or reports more than its class's forward."""
    return bool("forward" in vars(layer) or layer._forward_hooks or layer._forward_pre_hooks
                or layer._backward_hooks or layer._backward_pre_hooks)


class FusedGatedMLP(nn.Module):
    """A gated feed-forward block on ``fused_gated_mlp`` with the weights of three bias-free
    ``nn.Linear`` layers, under their usual names and with their initialisation. The layers are not
    called: one that is more than its weight's product (an adapter, a bias, a hook) is refused."""

    def __init__(self, hidden_size: int, intermediate_size: int, activation: str = "silu",
                 device: Optional[torch.device] = None, dtype: Optional[torch.dtype] = None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"FusedGatedMLP: unknown activation {activation!r}")
        self.hidden_size = hidden_size
        self.intermediate_size = intermediate_size
        self.activation = activation

        def linear(i, o):
            return nn.Linear(i, o, bias=False, device=device, dtype=dtype)

        self.gate_proj = linear(hidden_size, intermediate_size)
        self.up_proj = linear(hidden_size, intermediate_size)
        self.down_proj = linear(intermediate_size, hidden_size)

    def forward(self, x: Tensor) -> Tensor:
        layers = (self.gate_proj, self.up_proj, self.down_proj)
        for name, layer in zip(("gate_proj", "up_proj", "down_proj"), layers):
            if (not isinstance(layer, nn.Linear) or type(layer).forward is not nn.Linear.forward
                    or layer.bias is not None or watched(layer)):
                raise ValueError(f"FusedGatedMLP: {name} is more than a product with its weight "
                                 "(an adapter, a bias or hooks), which would be lost")
        return fused_gated_mlp(x, *[layer.weight for layer in layers], self.activation)

    def extra_repr(self) -> str:
        return f"{self.hidden_size}, {self.intermediate_size}, activation={self.activation!r}"
