"""A policy update through the operators around the model (GPU): embedding, blocks with the norms
before and after them, log-probs of the sampled tokens, the clipped policy loss, the backward
pass and the clipping of its gradients.

In fp32 the whole step is compared with float64: every operator's own error is a few 1e-6 of its
terms' magnitudes at most, and some ten of them follow one another in each direction, so the
gradients of a well-conditioned model agree to 1e-4 of their 2-norm.
"""
import math

import pytest
import torch
import torch.nn as nn

from helpers import BF, F32, same
from trainscale_amd.kernels import (FusedSandwichRMSNorm, ScaledEmbedding, clip_grad_norm_,
                                    clipped_grads, get_total_norm, swiglu_forward)
from trainscale_amd.loss import ClippedPolicyLoss, chunked_log_softmax, selective_log_softmax
from trainscale_amd.registry import KernelPatcher

pytestmark = pytest.mark.gpu
EPS = 1e-6
V, H, I, LAYERS, B, T = 300, 96, 160, 2, 3, 37


class Model(nn.Module):
    """Tied embedding, LAYERS gated MLP blocks, each followed by the block boundary."""

    def __init__(self, gpu, dtype):
        super().__init__()
        kw = dict(device=gpu, dtype=dtype)
        self.embed = ScaledEmbedding(V, H, scale=math.sqrt(H), padding_idx=0, **kw)
        self.up = nn.ModuleList(nn.Linear(H, 2 * I, bias=False, **kw) for _ in range(LAYERS))
        self.down = nn.ModuleList(nn.Linear(I, H, bias=False, **kw) for _ in range(LAYERS))
        self.norms = nn.ModuleList(FusedSandwichRMSNorm(H, EPS, weight_offset=1.0, layer_gate=True,
                                                        gate_init=0.5, **kw) for _ in range(LAYERS))
        with torch.no_grad():
            self.embed.weight.mul_(0.2)
            for m in self.norms:
                m.post_weight.normal_(0, 0.1)
                m.pre_weight.normal_(0, 0.1)

    def forward(self, ids):
        stream = self.embed(ids)
        x = stream
        for up, down, norm in zip(self.up, self.down, self.norms):
            gate, lin = up(x).chunk(2, -1)
            x, stream = norm(down(swiglu_forward(gate.contiguous(), lin.contiguous())), stream)
        return x


def batch(gpu, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    ids = torch.randint(1, V, (B, T + 1), device=gpu, generator=g)
    length = torch.tensor([T, T // 2, 0], device=gpu)  # one sequence without a valid token
    mask = torch.arange(T, device=gpu)[None] < length[:, None]
    ids[:, 1:][~mask] = 0  # padding
    adv = torch.randn(B, device=gpu, generator=g)
    noise = 0.2 * torch.randn(2, B, T, device=gpu, generator=g)
    return ids, mask, adv, noise


def log_probs(model, ids):
    h = model(ids[:, :-1])
    w = model.embed.weight
    if w.dtype == F32:
        logits = (h.reshape(-1, H) @ w.t()).view(B, T, V)
        return selective_log_softmax(logits, ids[:, 1:])
    return chunked_log_softmax(h, w, ids[:, 1:], out_dtype=F32)


def step(model, data, loss):
    ids, mask, adv, noise = data
    lp = log_probs(model, ids)
    base = lp.detach()
    return loss(lp, base + noise[0], adv, mask, base + noise[1])


def reference(model, data, beta):
    """The step's loss and gradients in float64, from the definitions."""
    p = {k: v.detach().double().requires_grad_() for k, v in model.named_parameters()}
    ids, mask, adv, noise = data

    def norm(x, w):
        return x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (1 + w)

    w = p["embed.weight"]
    # the padding token's row gets no gradient from the lookup
    stream = math.sqrt(H) * torch.where((ids[:, :-1] == 0)[..., None], w.detach()[ids[:, :-1]],
                                        w[ids[:, :-1]])
    x = stream
    for i in range(LAYERS):
        a, b = (x @ p[f"up.{i}.weight"].t()).chunk(2, -1)
        y = (a * torch.sigmoid(a) * b) @ p[f"down.{i}.weight"].t()
        stream = stream + p[f"norms.{i}.gate"] * norm(y, p[f"norms.{i}.post_weight"])
        x = norm(stream, p[f"norms.{i}.pre_weight"])
    lp = (x @ w.t()).log_softmax(-1).gather(-1, ids[:, 1:, None])[..., 0]
    old, ref = lp.detach() + noise[0], lp.detach() + noise[1]
    r = (lp - old).exp()
    pol = -torch.minimum(r * adv[:, None], r.clamp(0.8, 1.2) * adv[:, None])
    k = torch.expm1(ref - lp) - (ref - lp)
    total = ((pol + beta * k) * mask).sum() / mask.sum()
    return total, dict(zip(p, torch.autograd.grad(total, list(p.values()))))


def test_step_against_float64(gpu):
    torch.manual_seed(1)
    model, data = Model(gpu, F32), batch(gpu)
    out = step(model, data, ClippedPolicyLoss(0.2, 0.2, kl_coef=0.1))
    out.loss.backward()
    want, grads = reference(model, data, 0.1)
    assert abs(float(out.loss) - float(want)) <= 1e-5 * abs(float(want)) + 1e-6
    for k, p in model.named_parameters():
        d = (p.grad.double() - grads[k]).norm()
        assert float(d) <= 1e-4 * float(grads[k].norm()), (k, float(d), float(grads[k].norm()))
    norm = math.sqrt(sum(float(g.square().sum()) for g in grads.values()))
    before = [p.grad.clone() for p in model.parameters()]
    assert abs(float(get_total_norm(before)) - norm) <= 1e-4 * norm
    n = clip_grad_norm_(model.parameters(), 0.5 * norm)
    assert abs(float(n) - norm) <= 1e-4 * norm
    for p, g in zip(model.parameters(), before):
        assert torch.allclose(p.grad, g * (0.5 * norm / (float(n) + 1e-6)), rtol=1e-6, atol=0)


def test_step_in_bf16_with_the_fused_log_probs(gpu):
    torch.manual_seed(2)
    model, data = Model(gpu, BF), batch(gpu, 1)
    loss = ClippedPolicyLoss(0.2, 0.28, kl_coef=0.05, reduction="sequence")
    main = [torch.empty(p.shape, device=gpu) for p in model.parameters()]
    for _ in range(2):
        for p in model.parameters():
            p.grad = None
        out = step(model, data, loss)
        out.loss.backward()
        n = clipped_grads([p.grad for p in model.parameters()], 1.0, main)
        assert math.isfinite(float(n)) and float(n) > 0
        assert all(bool(m.isfinite().all()) and bool(m.any()) for m in main)
        assert float(get_total_norm(main)) <= 1.0 + 1e-5
    _, grads = reference(model, data, 0.05)  # (the same parameters, another reduction: direction)
    g = model.embed.weight.grad.double()
    cos = float((g * grads["embed.weight"]).sum() / (g.norm() * grads["embed.weight"].norm()))
    assert cos > 0.9


def test_step_in_a_graph(gpu):
    torch.manual_seed(3)
    model, data = Model(gpu, BF), batch(gpu, 2)
    data = [t.clone() for t in data]
    loss = ClippedPolicyLoss(kl_coef=0.1)
    params = list(model.parameters())
    main = [torch.empty(p.shape, device=gpu) for p in params]

    def whole():
        out = step(model, data, loss)
        norm = clipped_grads(list(torch.autograd.grad(out.loss, params)), 0.1, main)
        return [v.detach() for v in out] + [norm]

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        whole()
    torch.cuda.current_stream(gpu).wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = whole()
    for rep in range(3):
        for t, v in zip(data, batch(gpu, 10 + rep)):
            t.copy_(v)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in outs] + [m.clone() for m in main]
        ref = whole()
        assert all(same(a, b) for a, b in zip(got, ref + main)), rep


def test_patched_embedding(gpu):
    m = nn.Sequential(nn.Embedding(50, 64, padding_idx=3, device=gpu, dtype=BF))
    ids = torch.randint(0, 50, (4, 100), device=gpu)
    want = m(ids)
    p = KernelPatcher(patch_embedding=True)
    p.patch(m)
    assert p.patched_layers == [("0", "Embedding")]
    out = m(ids)
    assert same(out, want)
    up = torch.randn(4, 100, 64, device=gpu).to(BF)
    (g,) = torch.autograd.grad(out, m[0].weight, up)
    keep = ids.reshape(-1) != 3
    ref = torch.zeros(50, 64, device=gpu, dtype=torch.float64).index_add(
        0, ids.reshape(-1)[keep], up.reshape(-1, 64)[keep].double())
    assert bool(((g.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-4).all())
    assert not g[3].any()


def test_second_derivatives_are_refused(gpu):
    m = Model(gpu, F32)
    out = step(m, batch(gpu), ClippedPolicyLoss(kl_coef=0.1))
    (g,) = torch.autograd.grad(out.loss, m.embed.weight, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
