"""The embedding patch of KernelPatcher: which modules it takes, and that CPU tensors keep the
module's own forward."""
import torch
import torch.nn as nn

from trainscale_amd.registry import KernelPatcher


class Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.plain = nn.Embedding(10, 4, padding_idx=2)
        self.renormed = nn.Embedding(10, 4, max_norm=1.0)
        self.by_freq = nn.Embedding(10, 4, scale_grad_by_freq=True)
        self.sparse = nn.Embedding(10, 4, sparse=True)
        self.own = type("OwnEmbedding", (nn.Embedding,), {})(10, 4)


def test_patch_is_opt_in():
    m = Model()
    assert KernelPatcher().patch(m).plain.forward.__func__ is nn.Embedding.forward
    p = KernelPatcher(patch_embedding=True)
    p.patch(m)
    assert p.patched_layers == [("plain", "Embedding")]
    ids = torch.tensor([[1, 2], [3, 1]])
    out = m.plain(ids)
    assert torch.equal(out, m.plain.weight[ids])
    out.sum().backward()
    assert not m.plain.weight.grad[2].any() and bool((m.plain.weight.grad[1] == 2).all())
    again = KernelPatcher(patch_embedding=True)
    again.patch(m)
    assert again.patched_layers == []
