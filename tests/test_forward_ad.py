"""Forward-mode differentiation: no operator has its derivative, and none may drop a tangent
without a word. On the CPU, with the launches replaced by plain torch."""
import pytest
import torch
from torch.autograd import forward_ad

from trainscale_amd import _lib, ops
from trainscale_amd.kernels import (FusedSandwichRMSNorm, clip_grad_norm_, clipped_grads,
                                    fused_sandwich_rms_layernorm, get_total_norm, scaled_embedding)
from trainscale_amd.loss import clipped_policy_loss


@pytest.fixture
def launches(monkeypatch):
    monkeypatch.setattr(ops, "embedding_forward", lambda ids, w, ld, scale: w.detach()[ids] * scale)
    monkeypatch.setattr(ops, "sandwich_norm_forward", lambda y, ldy, x, *rest: (
        y.detach().clone(), x.detach().clone(), torch.ones(2, y.shape[0])))


W = torch.randn(5, 4, generator=torch.Generator().manual_seed(0))
IDS = torch.tensor([0, 3, 3])


def calls(dual_at):
    """The operators' calls, argument number dual_at of each a dual tensor."""
    def d(k, t):
        return forward_ad.make_dual(t, torch.ones_like(t)) if k == dual_at else t
    v = torch.ones(4)
    yield lambda: scaled_embedding(IDS, d(0, W))
    yield lambda: fused_sandwich_rms_layernorm(d(0, W), d(1, W), d(2, v), d(3, v), d(4, v))
    yield lambda: FusedSandwichRMSNorm(4)(d(0, W), d(1, W))


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("dual_at", range(5))
def test_tangents_are_refused(launches, dual_at, grad_mode):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        for k, call in enumerate(calls(dual_at)):
            if dual_at > (0, 4, 1)[k]:
                call()  # no argument has a tangent
                continue
            with pytest.raises(RuntimeError, match="jvp"):
                call()


def test_results_without_a_level(launches):
    w = W.clone().requires_grad_()
    assert scaled_embedding(IDS, w).requires_grad
    assert not scaled_embedding(IDS, W).requires_grad
    with torch.no_grad():
        assert not scaled_embedding(IDS, w).requires_grad
    assert torch.equal(scaled_embedding(IDS, W, 2.0), 2 * W[IDS])
    assert fused_sandwich_rms_layernorm(W, W, w[0], w[1])[0].requires_grad
    with torch.no_grad():
        assert not fused_sandwich_rms_layernorm(W, W, w[0], w[1])[0].requires_grad


def test_policy_loss_and_clipping_refuse_tangents(monkeypatch):
    lp, adv = torch.zeros(2, 3), torch.zeros(2)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(lp, lp + 1)
        p = torch.nn.Parameter(torch.zeros(2, 3))
        p.grad = dual
        for call in (lambda: get_total_norm([dual]), lambda: clip_grad_norm_([p], 1.0),
                     lambda: clipped_grads([dual], 1.0, [torch.zeros(2, 3)])):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        monkeypatch.setattr(_lib, "require_gpu", lambda *a: torch.device("cpu"))
        monkeypatch.setattr(ops, "policy_loss_forward", lambda *a: tuple(torch.zeros(5)))
        clipped_policy_loss(lp, lp, adv)
        with torch.no_grad(), pytest.raises(RuntimeError, match="jvp"):
            clipped_policy_loss(dual, lp, adv)
