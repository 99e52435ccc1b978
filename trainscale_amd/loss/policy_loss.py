"""Clipped policy loss with a KL term, over token log-probabilities.

What ``chunked_log_softmax`` and ``selective_log_softmax`` return goes in here: the log-probs of
the sampled tokens under the policy, next to those under the sampling policy and a reference, the
advantages and the mask of the completions. It is the objective of the trainer's group-relative
and actor updates (data_pipeline/trainer/rl_training.py:483-600):

    r      = exp(logp - old),  x = ref - logp
    policy = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
    kl     = exp(x) - x - 1
    loss   = sum over the valid tokens of w (policy + kl_coef kl)

with w = 1 / (valid tokens) ("token"), 1 / (valid tokens of the sequence * sequences that have
any) ("sequence"), or 1 ("sum"). The loss, its parts and the gradient come from two launches
forward (one for small batches) and one backward.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
import torch.nn as nn
from torch import Tensor
from torch.autograd.function import once_differentiable

from .. import _lib, ops

__all__ = ["PolicyLoss", "ClippedPolicyLossFunction", "clipped_policy_loss", "ClippedPolicyLoss"]


class PolicyLoss(NamedTuple):
    """0-dim fp32 tensors; only ``loss`` is differentiable."""
    loss: Tensor
    policy_loss: Tensor
    kl: Tensor
    clip_fraction: Tensor


def _rows(t: Tensor) -> Tensor:
    """[B, T] with a unit column stride and rows that do not overlap."""
    if t.is_contiguous():
        return t
    if (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        return t.contiguous()
    return t


def _places(tensors) -> list:
    """Where the tensors' values lie."""
    return [None if t is None else (t.data_ptr(), t.stride()) for t in tensors]


def _logps(name: str, t: Tensor, logps: Tensor) -> Tensor:
    if t.shape != logps.shape:
        raise ValueError(f"clipped_policy_loss: {name} {tuple(t.shape)} != logps "
                         f"{tuple(logps.shape)}")
    if t.dtype is not logps.dtype:
        _lib.dtype_code(t, f"clipped_policy_loss {name}")
        t = t.float()
    return _rows(t)


class ClippedPolicyLossFunction(torch.autograd.Function):
    """forward(logps, old_logps, advantages, mask, ref_logps, clip_low, clip_high, kl_coef,
    reduction) -> (loss, policy_loss, kl, clip_fraction); differentiable in logps through loss."""

    @staticmethod
    def forward(ctx, logps: Tensor, old_logps: Optional[Tensor], advantages: Tensor,
                mask: Optional[Tensor], ref_logps: Optional[Tensor], clip_low: float,
                clip_high: float, kl_coef: float, reduction: str):
        if logps.dim() != 2:
            raise ValueError(f"clipped_policy_loss: logps must be [B, T], got {tuple(logps.shape)}")
        if reduction not in ops.POLICY_REDUCTIONS:
            raise ValueError(f"clipped_policy_loss: unknown reduction {reduction!r}")
        if not (clip_low >= 0 and clip_high >= 0):
            raise ValueError("clipped_policy_loss: clip bounds must be >= 0, got "
                             f"{clip_low}, {clip_high}")
        if not 0 <= kl_coef < float("inf"):
            raise ValueError(f"clipped_policy_loss: kl_coef must be finite and >= 0, got {kl_coef}")
        if kl_coef > 0 and ref_logps is None:
            raise ValueError("clipped_policy_loss: kl_coef needs ref_logps")
        _lib.dtype_code(logps, "clipped_policy_loss logps")
        b, t = logps.shape
        adv = advantages
        if adv.dim() == 2 and adv.shape[0] == b and (
                adv.shape[1] == 1 or (adv.shape[1] == t and adv.stride(1) == 0 and t > 0)):
            adv = adv[:, 0]
        if adv.shape not in ((b,), (b, t)):
            raise ValueError(f"clipped_policy_loss: advantages {tuple(adv.shape)} for logps "
                             f"{tuple(logps.shape)}: expected [B] or [B, T]")
        if adv.dtype is not torch.float32:
            adv = adv.float()
        adv = adv.contiguous() if adv.dim() == 1 else _rows(adv)
        if mask is not None:
            if mask.shape != logps.shape:
                raise ValueError(f"clipped_policy_loss: mask {tuple(mask.shape)} != logps "
                                 f"{tuple(logps.shape)}")
            if mask.dtype is not torch.bool and mask.dtype is not torch.uint8:
                mask = mask != 0
            mask = _rows(mask)
        lp = _rows(logps)
        old = None if old_logps is None else _logps("old_logps", old_logps, logps)
        ref = None if ref_logps is None else _logps("ref_logps", ref_logps, logps)
        dev = _lib.require_gpu("clipped_policy_loss", lp, old, adv, mask, ref)
        inputs = ops.policy_inputs(lp, old, adv, mask, ref, clip_low, clip_high, kl_coef, reduction)
        loss, policy, kl, clipped, weights = ops.policy_loss_forward(inputs, dev)
        ctx.save_for_backward(lp, old, adv, mask, ref, weights)
        # the struct points into these tensors
        ctx.inputs, ctx.places = inputs, _places((lp, old, adv, mask, ref))
        ctx.cfg = (clip_low, clip_high, kl_coef, reduction)
        ctx.mark_non_differentiable(policy, kl, clipped)
        ctx.set_materialize_grads(False)
        return loss, policy, kl, clipped

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss: Optional[Tensor], *_unused):
        if dloss is None or not ctx.needs_input_grad[0]:
            return (None,) * 9
        *saved, weights = ctx.saved_tensors
        inputs = ctx.inputs
        if _places(saved) != ctx.places:
            # hooks on saved tensors have given them back elsewhere or with other strides
            saved = [t if t is None else t.contiguous() if t.dim() == 1 else _rows(t)
                     for t in saved]
            inputs = ops.policy_inputs(*saved, *ctx.cfg)
            weights = weights.contiguous()
        grad = ops.policy_loss_backward(inputs, weights, dloss, saved[0].dtype)
        return (grad, *(None,) * 8)


def clipped_policy_loss(logps: Tensor, old_logps: Optional[Tensor], advantages: Tensor,
                        mask: Optional[Tensor] = None, ref_logps: Optional[Tensor] = None,
                        clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                        reduction: str = "token") -> PolicyLoss:
    """The clipped policy loss of token log-probs [B, T] (module docstring).

    old_logps None: the policy's own values (r = 1, the gradient is that of the ratio).
    advantages: [B] (or [B, 1]), one for each sequence, or [B, T]. mask [B, T]: tokens that count
    (non-zero); what the others hold, NaN and infinities included, does not matter, and their
    gradient is 0. A sequence without any token that counts adds nothing, and "sequence" does
    not count it. ref_logps adds the KL estimate to the result and, times kl_coef, to the loss.
    clip_low >= 1 leaves the ratio unbounded below, clip_high = inf above.

    logps, old_logps, ref_logps: fp32, bf16 or fp16. Returns PolicyLoss(loss, policy_loss, kl,
    clip_fraction), reduced alike (clip_fraction: the tokens whose ratio is clipped); the
    gradient goes to logps only."""
    return PolicyLoss(*ClippedPolicyLossFunction.apply(
        logps, old_logps, advantages, mask, ref_logps, float(clip_low), float(clip_high),
        float(kl_coef), reduction))


class ClippedPolicyLoss(nn.Module):
    """``clipped_policy_loss`` with its settings."""

    def __init__(self, clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0,
                 reduction: str = "token"):
        super().__init__()
        if reduction not in ops.POLICY_REDUCTIONS:
            raise ValueError(f"Invalid reduction: {reduction}")
        self.clip_low = clip_low
        self.clip_high = clip_high
        self.kl_coef = kl_coef
        self.reduction = reduction

    def forward(self, logps: Tensor, old_logps: Optional[Tensor], advantages: Tensor,
                mask: Optional[Tensor] = None, ref_logps: Optional[Tensor] = None) -> PolicyLoss:
        return clipped_policy_loss(logps, old_logps, advantages, mask, ref_logps, self.clip_low,
                                   self.clip_high, self.kl_coef, self.reduction)

    def extra_repr(self) -> str:
        return (f"clip_low={self.clip_low}, clip_high={self.clip_high}, kl_coef={self.kl_coef}, "
                f"reduction='{self.reduction}'")
