"""Gradients with saved tensors that hooks hand back packed or with other strides, bit for bit those
without hooks."""
import contextlib

import pytest
import torch

from helpers import BF, F32, same, saved_elsewhere
from trainscale_amd.distributed import tensor_parallel as tp
from trainscale_amd.kernels import fast_cross_entropy_loss, fused_add_rms_layernorm, rms_layernorm
from trainscale_amd.kernels.fused_kernels import fast_rms_layernorm
from trainscale_amd.kernels.layernorm_kernels import RMSNorm
from trainscale_amd.loss import selective_log_softmax
from trainscale_amd.loss.sota_losses import CrossEntropyRowsFunction, FusedCrossEntropyLoss

pytestmark = pytest.mark.gpu
N, C = 37, 1000


def calls(gpu, dtype):
    g = torch.Generator(device=gpu).manual_seed(1)
    w = torch.randn(C, device=gpu, generator=g).to(dtype).requires_grad_()
    r = torch.randn(N, C, device=gpu, generator=g).to(dtype)
    y = torch.randint(0, C, (N,), device=gpu, generator=g)
    return {
        "fast_rms": lambda x: fast_rms_layernorm(x, w), "rms": lambda x: rms_layernorm(x, w),
        "rms_no_weight": lambda x: RMSNorm(C, elementwise_affine=False)(x),
        "add_rms": lambda x: fused_add_rms_layernorm(x, r, w.detach()),
        "fast_ce": lambda x: fast_cross_entropy_loss(x, y),
        "ce_rows": lambda x: CrossEntropyRowsFunction.apply(x, y),
        "ce_none": lambda x: FusedCrossEntropyLoss(reduction="none")(x, y),
        "selective": lambda x: selective_log_softmax(x, y),
        "vocab": lambda x: tp.vocab_parallel_cross_entropy(x, y),
    }, w


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("name", ["fast_rms", "rms", "rms_no_weight", "add_rms", "fast_ce", "ce_rows",
                                  "ce_none", "selective", "vocab"])
def test_gradients(gpu, name, dtype):
    wide = torch.randn(N, C + 24, device=gpu, generator=torch.Generator(device=gpu).manual_seed(2))
    got = []
    for hooks in (contextlib.nullcontext(), torch.autograd.graph.save_on_cpu(), saved_elsewhere()):
        run, w = calls(gpu, dtype)
        # one call of the legacy cross-entropy writes its gradient over its logits
        x = wide.to(dtype).clone()[:, 8:8 + C].requires_grad_()
        with hooks:
            out = run[name](x)
        up = torch.linspace(-1, 1, out.numel(), device=gpu).view(out.shape).to(out.dtype)
        leaves = [x, w] if name in ("fast_rms", "rms") else [x]
        got.append(torch.autograd.grad(out, leaves, up))
    for other in got[1:]:
        assert all(same(a, b) for a, b in zip(got[0], other))
    assert all(bool(t.any()) for t in got[0])
