"""A deep copy of a patched model (a frozen reference policy, moving averages) runs on its own
parameters."""
import copy

import pytest
import torch
import torch.nn as nn

import trainscale_amd.registry as registry
from trainscale_amd.registry import KernelPatcher


class LlamaRMSNorm(nn.Module):
    def __init__(self):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(8))
        self.variance_epsilon = 1e-5

    def forward(self, x):
        return self.weight * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.variance_epsilon)


class LlamaMLP(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate_proj, self.up_proj = nn.Linear(8, 12), nn.Linear(8, 12)
        self.down_proj = nn.Linear(12, 8)

    def forward(self, x):
        return self.down_proj(nn.functional.silu(self.gate_proj(x)) * self.up_proj(x))


class Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.embed, self.norm, self.mlp = nn.Embedding(20, 8), LlamaRMSNorm(), LlamaMLP()

    def forward(self, ids):
        return self.mlp(self.norm(self.embed(ids)))


IDS = torch.tensor([[3, 19, 3], [0, 7, 1]])


def patched(device="cpu"):
    torch.manual_seed(0)
    m = Model().to(device)
    p = KernelPatcher(patch_embedding=True)
    p.patch(m)
    assert len(p.patched_layers) == 3
    return m


def check(device):
    m, ids = patched(device), IDS.to(device)
    want = m(ids).detach().clone()
    frozen = copy.deepcopy(m)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(1.0)
    assert torch.equal(frozen(ids), want) and not torch.equal(m(ids), want)
    frozen(ids).sum().backward()
    assert all(p.grad is None for p in m.parameters())
    assert all(p.grad is not None for p in frozen.parameters())
    again = KernelPatcher(patch_embedding=True)
    again.patch(frozen)
    assert again.patched_layers == []
    twice = copy.deepcopy(frozen)
    assert torch.equal(twice(ids), want)


def test_deep_copy():
    check("cpu")


def test_deep_copy_through_the_kernels_route(monkeypatch):
    # the route that GPU tensors take, with plain torch in the kernels' place
    monkeypatch.setattr(registry, "scaled_embedding", lambda i, w, padding_idx=None: w[i])
    monkeypatch.setattr(registry, "fast_rms_layernorm",
                        lambda x, w, eps: w * x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps))
    monkeypatch.setattr(registry, "swiglu_forward", lambda g, u: nn.functional.silu(g) * u)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True, raising=False)
    check("cpu")


@pytest.mark.gpu
def test_deep_copy_on_the_gpu(gpu):
    check(gpu)
