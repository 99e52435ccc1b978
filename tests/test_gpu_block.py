"""One transformer block in training on the layer's operators: rotary positions with several axes,
attention in plain fp32, dropout with the residual sum and the norm, the gated feed-forward block,
dropout with the residual sum. Its results and every gradient against float64.

The same block is also computed in float64 with every stage's result, and every stage's gradients,
rounded to the data type where a plain program rounds them. Errors of the two runs are sums of the
same kind of independent roundings, thousands for each result, so their 2-norms are alike; the
operators round at fewer places. A wrong mask, angle or factor is off by far more. The bound is 1.25
times the plain program's error: its own spread, one in the root of the smallest result's number of
independent roundings (64 weights of the norm, each a sum over all rows), is within 0.18 at two
standard errors of either.
"""
import pytest
import torch
import torch.nn as nn

from helpers import BF, F16, same
from philox import keep_mask
from trainscale_amd.kernels import (FusedDropoutAddRMSNorm, FusedGatedMLP, MultiAxisRotaryEmbedding,
                                    fused_dropout_add)

pytestmark = pytest.mark.gpu
P, EPS, SEED = 0.1, 1e-6, 77
SCALE = 65536 / (65536 - round(P * 65536))


def attention(q, k, v):
    """[B, S, H, D] tensors, causal, in their own type."""
    q, k, v = [t.transpose(1, 2) for t in (q, k, v)]
    k, v = [t.repeat_interleave(q.shape[1] // t.shape[1], 1) for t in (k, v)]
    s = q @ k.transpose(2, 3).contiguous() / q.shape[-1] ** 0.5
    hide = torch.ones(q.shape[2], q.shape[2], dtype=torch.bool, device=q.device).triu(1)
    return (s.masked_fill(hide, float("-inf")).softmax(-1) @ v).transpose(1, 2).contiguous()


class Block(nn.Module):
    def __init__(self, width, heads, kv_heads, inner, sections, layout):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        new = lambda o: nn.Linear(width, o, bias=False)
        self.q_proj, self.o_proj = new(width), new(width)
        self.k_proj, self.v_proj = new(kv_heads * self.dim), new(kv_heads * self.dim)
        self.rope = MultiAxisRotaryEmbedding(sections, layout=layout)
        self.norm = FusedDropoutAddRMSNorm(width, P, eps=EPS)
        self.mlp = FusedGatedMLP(width, inner)

    def forward(self, x, pos):
        b, s, _ = x.shape
        q, k, v = [m(x).view(b, s, -1, self.dim) for m in (self.q_proj, self.k_proj, self.v_proj)]
        q, k = self.rope(q, k, pos)
        o = attention(q.float(), k.float(), v.float()).to(x.dtype).view(b, s, -1)
        y, h = self.norm(self.o_proj(o), x, rng=(SEED, 0))
        return fused_dropout_add(self.mlp(y), h, P, rng=(SEED, 1))


class Rounded(torch.autograd.Function):
    @staticmethod
    def forward(ctx, t, dtype):
        ctx.dtype = dtype
        return t.to(dtype).to(t.dtype)

    @staticmethod
    def backward(ctx, g):
        return g.to(ctx.dtype).to(g.dtype), None


class Uses(torch.autograd.Function):
    """n uses of one tensor, whose gradients are rounded and added one by one, as autograd adds them
    in the data type. x has 4, and the residual's, of the whole's size, comes first: three roundings
    of 1.66e-3 (one of bf16, rms), the last the result's own. Without the other two the plain dx was
    off by 2.53e-3; (2.53^2 + 2 1.66^2)^(1/2) 1e-3 = 3.45e-3."""
    @staticmethod
    def forward(ctx, t, dtype, n):
        ctx.dtype = dtype
        return tuple(t.clone() for _ in range(n))

    @staticmethod
    def backward(ctx, *grads):
        r = (lambda t: t) if ctx.dtype is None else (lambda t: t.to(ctx.dtype).to(t.dtype))
        total = r(grads[0])
        for g in grads[1:]:
            total = r(total + r(g))
        return total, None, None


def plain(block, x, pos, dtype=None):
    """The block in float64, rounded to `dtype` where a plain program in it rounds."""
    r = (lambda t: t) if dtype is None else (lambda t: Rounded.apply(t, dtype))
    w = {k: v.detach().double().requires_grad_() for k, v in block.named_parameters()}
    x = x.detach().double().requires_grad_()
    b, s, c = x.shape

    def turn(t):
        plan = block.rope.plan
        axis = torch.tensor(plan.axis, device=t.device)
        a = pos[axis].permute(1, 2, 0)[:, :, None].double() * plan.inv_freq.to(t.device)
        lo, hi = t.chunk(2, -1)
        return r(torch.cat((lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()), -1))

    def drop(t, offset):
        keep = torch.from_numpy(keep_mask(b * s, c, SEED, offset, P)).view(b, s, c).to(t.device)
        return torch.where(keep, t * SCALE, 0.0)

    first, *uses = Uses.apply(x, dtype, 4)  # the residual's gradient is there first
    q, k, v = [r(t @ w[f"{n}_proj.weight"].t()).view(b, s, -1, block.dim)
               for n, t in zip("qkv", uses)]
    o = r(attention(turn(q), turn(k), v)).view(b, s, c)
    h = r(drop(r(r(o) @ w["o_proj.weight"].t()), 0) + first)
    y = r(h * (h.square().mean(-1, keepdim=True) + EPS).rsqrt() * w["norm.weight"])
    g, u = [r(r(y) @ w[f"mlp.{n}_proj.weight"].t()) for n in ("gate", "up")]
    a = r(r(g * torch.sigmoid(g)) * u)
    out = r(drop(r(a @ w["mlp.down_proj.weight"].t()), 1) + r(h))
    return out, [x, *w.values()]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("b,s,heads,kv,width,inner,sections,layout", [
    (2, 37, 4, 2, 256, 680, (8, 12, 12), "blocks"), (1, 50, 2, 2, 64, 168, (8, 8), "separate"),
    (3, 101, 8, 1, 512, 1368, (12, 10, 10), "interleaved")])
def test_block(gpu, b, s, heads, kv, width, inner, sections, layout, dtype):
    torch.manual_seed(width)
    block = Block(width, heads, kv, inner, sections, layout).to(gpu, dtype)
    with torch.no_grad():
        block.norm.weight.add_(0.1 * torch.randn(width, device=gpu))
    x = torch.randn(b, s, width, device=gpu).to(dtype).requires_grad_()
    pos = torch.randint(0, 5000, (len(sections), b, s), device=gpu)
    dy = torch.randn(b, s, width, device=gpu).to(dtype)
    runs = []
    for _ in range(2):
        y = block(x, pos)
        runs.append([y.detach(), *torch.autograd.grad(y, [x, *block.parameters()], dy)])
    assert all(same(p, q) for p, q in zip(*runs))
    outs = []
    for rounding in (None, dtype):
        y, leaves = plain(block, x, pos, rounding)
        outs.append([y.detach(), *torch.autograd.grad(y, leaves, dy.double())])
    names = ["y", "x", *dict(block.named_parameters())]
    for name, got, exact, rounded in zip(names, runs[0], *outs):
        assert got.dtype == dtype and got.shape == exact.shape, name
        # a gradient's own last rounding, which the plain run's leaves, in float64, are spared
        own, other = (got.double() - exact).norm(), (rounded.to(dtype).double() - exact).norm()
        assert own <= 1.25 * other, (name, float(own), float(other))
