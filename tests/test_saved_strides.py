"""What a backward addresses is the saved tensor that it got, whose strides hooks on saved tensors
(activation offloading) may have changed: on the CPU, with the launches replaced by stubs that check
the row stride they are given against the tensor's own."""
import pytest
import torch

from trainscale_amd import ops
from trainscale_amd.distributed import tensor_parallel as tp
from trainscale_amd.kernels import (fast_cross_entropy_loss, fused_add_rms_layernorm, rms_layernorm)
from trainscale_amd.kernels.fused_kernels import fast_rms_layernorm
from trainscale_amd.kernels.layernorm_kernels import RMSNorm
from trainscale_amd.loss import selective_log_softmax
from trainscale_amd.loss.sota_losses import CrossEntropyRowsFunction, FusedCrossEntropyLoss

ROWS, COLS = 6, 10


def inside(t, ld):
    assert t.stride(1) == 1 and ld == t.stride(0)
    assert t.storage_offset() + (t.shape[0] - 1) * ld + t.shape[1] <= (
        t.untyped_storage().nbytes() // t.element_size())


@pytest.fixture
def seen(monkeypatch):
    """The backward launches' operands, checked."""
    seen = []

    def rms_backward(dy, lddy, x, ldx, weight, rstd, need_dw):
        inside(x, ldx)
        seen.append(x.clone())
        return torch.zeros_like(x), torch.zeros_like(weight) if need_dw else None

    def ce_backward(x, ld, labels, lse, dloss, grad, ldg, *a, **k):
        inside(x, ld)
        inside(grad, ldg)
        seen.append(x.clone())

    def shard_backward(x, ld, *a):
        inside(x, ld)
        seen.append(x.clone())
        return torch.zeros(x.shape)

    rows = torch.zeros(ROWS)
    stubs = dict(rmsnorm_forward=lambda x, *a: (torch.zeros(x.shape), rows),
                 add_rmsnorm_forward=lambda x, ldx, r, *a, **k: (torch.zeros(x.shape), x + r, rows),
                 rmsnorm_backward=rms_backward, ce_backward=ce_backward,
                 ce_forward=lambda *a, **k: (rows.clone(), rows),
                 ce_vocab_shard_stats=lambda *a: torch.zeros(ROWS, 4),
                 ce_vocab_merge=lambda *a: (rows, rows.clone()),
                 ce_vocab_shard_backward=shard_backward)
    for name, f in stubs.items():
        monkeypatch.setattr(ops, name, f)
    return seen


def moved(how):
    """Saved tensors come back in memory of their own: `packed` or column by column."""
    def unpack(t):
        return t.t().contiguous().t() if how == "columns" and t.dim() == 2 else t
    return torch.autograd.graph.saved_tensors_hooks(
        lambda t: t.clone(memory_format=torch.contiguous_format), unpack)


LABELS = torch.zeros(ROWS, dtype=torch.int64)
CALLS = {
    "fast_rms": lambda x: fast_rms_layernorm(x, torch.ones(COLS)),
    "rms": lambda x: rms_layernorm(x, torch.ones(COLS)),
    "rms_no_weight": lambda x: RMSNorm(COLS, elementwise_affine=False)(x),
    "add_rms": lambda x: fused_add_rms_layernorm(x, x.detach(), torch.ones(COLS)),
    "fast_ce": lambda x: fast_cross_entropy_loss(x, LABELS),
    "ce_rows": lambda x: CrossEntropyRowsFunction.apply(x, LABELS),
    "ce_none": lambda x: FusedCrossEntropyLoss(reduction="none")(x, LABELS),
    "selective": lambda x: selective_log_softmax(x, LABELS),
    "vocab": lambda x: tp.vocab_parallel_cross_entropy(x, LABELS),
}


@pytest.mark.parametrize("how", ["packed", "columns"])
@pytest.mark.parametrize("name", CALLS)
def test_strides_of_saved_tensors(seen, name, how):
    x = torch.arange(ROWS * 17.).view(ROWS, 17)[:, 3:3 + COLS].requires_grad_()
    with moved(how):
        out = CALLS[name](x)
    out.sum().backward()
    want = 2 * x if name == "add_rms" else x
    assert len(seen) == 1 and torch.equal(seen[0], want.detach())
