"""Rotary positions with several axes against float64 on the GPU.

Tolerances, with u = 2^-24. The fraction of a turn is off by 2^-65 of a turn per position. Within an
eighth of a turn it is rounded to fp32 and scaled (2 u of at most 0.79 rad); the polynomials leave
out less than 0.04 u, and evaluating them adds at most 2 u: cos and sin are off by 4 u +
2 pi 2^-65 |pos|. A result of two products and a sum is off by 2 u more of (|x1| + |x2|), and by half a
step of its type.
"""
import contextlib
import math

import pytest
import torch

from helpers import BF, F16, F32, saved_elsewhere, same
from trainscale_amd.kernels import MultiAxisRotaryEmbedding, RopeAxes, apply_rope_axes, \
    apply_rope_theta

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def reference(x, pos, plan, backward=False):
    """The rotation in float64 and its bound before the last rounding."""
    n = len(plan.axis)
    p = pos.to(torch.int64).expand(len(plan.sections), x.shape[0], x.shape[1])
    # angles modulo a turn in two pieces of the position, each exact enough in 64 bits
    axis = torch.tensor(plan.axis, device=x.device)
    f = plan.inv_freq.to(x.device)
    lo, hi = p % 4096, p // 4096
    a = (lo[axis].permute(1, 2, 0) * f) + torch.remainder(
        hi[axis].permute(1, 2, 0).double() * (4096 * f), 2 * math.pi)
    c, s = a.cos()[:, :, None], a.sin()[:, :, None]
    if backward:
        s = -s
    X = x.double()
    if plan.interleaved:
        x1, x2 = X[..., 0:2 * n:2], X[..., 1:2 * n:2]
    else:
        x1, x2 = X[..., :n], X[..., n:2 * n]
    o1, o2 = x1 * c - x2 * s, x2 * c + x1 * s
    # the reference's own angles: 2^-53 of |hi f 4096|, at most |pos f|
    far = p[axis].permute(1, 2, 0)[:, :, None].double().abs()
    e = (6 * U + far * (2 * math.pi * 2.0 ** -65 + 4 * 2.0 ** -53 * f)) * (x1.abs() + x2.abs())
    out, bound = X.clone(), torch.zeros_like(X)
    if plan.interleaved:
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = o1, o2
        bound[..., 0:2 * n:2], bound[..., 1:2 * n:2] = e, e
    else:
        out[..., :n], out[..., n:2 * n] = o1, o2
        bound[..., :n], bound[..., n:2 * n] = e, e
    return out, bound


def check(got, x, pos, plan, what, backward=False):
    want, bound = reference(x, pos, plan, backward)
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    tol = bound * (1 + half(got.dtype)) + half(got.dtype) * want.abs() + tiny
    bad = ~((got.double() - want).abs() <= tol)
    assert got.shape == want.shape and not bad.any(), (what, int(bad.sum()),
                                                       bad.nonzero()[:3].tolist())
    n = 2 * len(plan.axis)
    assert same(got[..., n:].contiguous(), x[..., n:].contiguous()), what


def inputs(gpu, b, s, hq, hk, d, dtype, axes, seed, far=4096):
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *t: torch.randn(*t, device=gpu, generator=g).to(dtype)
    pos = torch.randint(0, far, (axes, b, s), device=gpu, generator=g)
    return r(b, s, hq, d), r(b, s, hk, d) if hk else None, pos, r(b, s, hq, d), \
        r(b, s, hk, d) if hk else None


def run_and_check(args, plan):
    q, k, pos, dq, dk = args
    leaf = [t.detach().requires_grad_() for t in (q, k) if t is not None]
    out = apply_rope_axes(leaf[0], leaf[1] if k is not None else None, pos, plan)
    outs = [t for t in out if t is not None]
    grads = torch.autograd.grad(outs, leaf, [t for t in (dq, dk) if t is not None])
    for t, x, d, g, what in zip(outs, (q, k), (dq, dk), grads, "qk"):
        check(t.detach(), x, pos, plan, what)
        check(g, d, pos, plan, "d" + what, backward=True)
    return [t.detach() for t in outs], grads


PLANS = [dict(sections=(16, 24, 24)), dict(sections=(24, 20, 20), layout="interleaved"),
         dict(sections=(20, 20), layout="separate"), dict(sections=(36,)),
         dict(sections=(3, 2), base=100.0), dict(sections=(18, 18), interleaved=True),
         dict(sections=(1,)), dict(sections=(64, 32, 32, 128), base=1e6)]


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("extra", [0, 8, 3])
def test_plans(gpu, plan, dtype, extra):
    p = RopeAxes(**plan)
    d = 2 * len(p.axis) + extra
    run_and_check(inputs(gpu, 2, 9, 3, 2, d, dtype, len(p.sections), d), p)


@pytest.mark.parametrize("b,s,hq,hk", [(1, 1, 1, 0), (16, 1, 32, 8), (1, 1000, 1, 1),
                                       (3, 333, 32, 8), (2, 17, 64, 64), (5, 1, 2, 0),
                                       (1, 2048, 16, 16), (257, 3, 1, 2)])
@pytest.mark.parametrize("il", [False, True])
def test_shapes(gpu, b, s, hq, hk, il):
    p = RopeAxes((16, 24, 24), interleaved=il)
    run_and_check(inputs(gpu, b, s, hq, hk, 128, BF, 3, s), p)


def test_far_positions(gpu):
    p = RopeAxes((32, 32), base=1e6)
    q, k, pos, dq, dk = inputs(gpu, 2, 40, 4, 2, 128, F32, 2, 3)
    for base in (0, -5000, 1 << 20, 1 << 24, 1 << 31, 1 << 40):
        run_and_check((q, k, pos + base, dq, dk), p)
    # any 64-bit position turns by something: no NaN, lengths kept
    ends = torch.tensor([2 ** 63 - 1, -2 ** 63], device=gpu)
    out, _ = apply_rope_axes(q[:1, :2], None, ends[None].expand(2, 1, 2), p)
    n0 = q[:1, :2].double().square().sum(-1)
    assert ((out.double().square().sum(-1) / n0 - 1).abs() <= 16 * U).all()


def test_one_axis_is_the_layers_rope(gpu):
    """With one axis and positions that fp32 products resolve, the one-axis kernel's results, up to
    its fp32 angles: 2 roundings of an angle below 64 and sincosf's own 4 u."""
    q, _, _, _, _ = inputs(gpu, 2, 64, 4, 0, 64, F32, 1, 4)
    pos = torch.arange(64, device=gpu).view(1, 1, 64)
    got, _ = apply_rope_axes(q, None, pos, RopeAxes((32,)))
    want = apply_rope_theta(q, inplace=False)
    mag = q[..., :32].abs() + q[..., 32:].abs()
    assert ((got - want).abs() <= (2 * 64 + 20) * U * torch.cat([mag, mag], -1)).all()


def test_transpose(gpu):
    """<R q, g> = <q, R' g>, both sides' roundings counted."""
    p = RopeAxes((8, 12, 12))
    q, k, pos, dq, dk = inputs(gpu, 2, 50, 4, 2, 80, F32, 3, 5)
    (oq, ok), (gq, gk) = run_and_check((q, k, pos, dq, dk), p)
    for o, d, x, g in ((oq, dq, q, gq), (ok, dk, k, gk)):
        lhs, rhs = (o.double() * d.double()).sum(), (x.double() * g.double()).sum()
        mag = 2 * float(torch.linalg.vector_norm(x.double()) * torch.linalg.vector_norm(d.double()))
        assert abs(float(lhs - rhs)) <= 2 * 7 * U * mag


def test_layouts(gpu):
    p = RopeAxes((16, 8, 8))
    q, k, pos, dq, dk = inputs(gpu, 3, 20, 4, 2, 72, BF, 3, 6)
    ref, grads = run_and_check((q, k, pos, dq, dk), p)
    both = lambda o: all(same(a, b) for a, b in zip(o, ref))
    qkv = torch.full((3, 20, 9, 72 + 5), float("nan"), dtype=BF, device=gpu)  # unaligned views
    qkv[:, :, :4, 3:75], qkv[:, :, 4:6, 3:75] = q, k
    assert both(apply_rope_axes(qkv[:, :, :4, 3:75], qkv[:, :, 4:6, 3:75], pos, p))
    h = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # heads before tokens
    assert both(apply_rope_axes(h(q), h(k), pos, p))
    last = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)
    assert both(apply_rope_axes(last(q), last(k), pos, p))
    assert both(apply_rope_axes(q, k, pos.int(), p))
    assert both(apply_rope_axes(q, k, pos.permute(1, 2, 0).contiguous().permute(2, 0, 1), p))
    one = pos[:, :1]
    shared = apply_rope_axes(q, k, one.expand(3, 3, 20), p)
    for again in (apply_rope_axes(q, k, one, p), apply_rope_axes(q, k, one[:, 0], p)):
        assert all(same(a, b) for a, b in zip(shared, again))
    # a head shared by broadcasting: its gradient is the sum over its copies
    kk = k[:, :, :1].detach().requires_grad_()
    o, _ = apply_rope_axes(kk.expand(3, 20, 4, 72), None, pos, p)
    (g,) = torch.autograd.grad(o, kk, dq)
    want, _ = apply_rope_axes(k[:, :, :1].expand(3, 20, 4, 72).contiguous(), None, pos, p)
    assert same(o.detach(), want)
    assert ((g.float() - grads[0].float().sum(2, keepdim=True)).abs()
            <= 4 * half(BF) * grads[0].float().abs().sum(2, keepdim=True)).all()


def test_in_place(gpu):
    p = RopeAxes((16, 8, 8))
    q, k, pos, _, _ = inputs(gpu, 3, 20, 4, 2, 72, BF, 3, 7)
    want = apply_rope_axes(q, k, pos, p)
    buf = torch.full((3, 20, 8, 72), float("nan"), dtype=BF, device=gpu)
    buf[:, :, :4], buf[:, :, 5:7] = q, k
    a, b = buf[:, :, :4], buf[:, :, 5:7]
    got = apply_rope_axes(a, b, pos, p, inplace=True)
    assert got[0] is a and got[1] is b and same(a, want[0]) and same(b, want[1])
    assert torch.isnan(buf[:, :, 4]).all() and torch.isnan(buf[:, :, 7]).all()


def test_in_place_is_seen_by_autograd(gpu):
    p = RopeAxes((16, 16))
    q, _, pos, _, _ = inputs(gpu, 2, 9, 4, 0, 64, BF, 2, 8)
    w = torch.ones_like(q, requires_grad=True)
    y = w * q  # keeps q
    apply_rope_axes(q, None, pos, p, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    with torch.inference_mode():
        t = q.clone()
        want = apply_rope_axes(t, None, pos, p)[0]
        assert same(apply_rope_axes(t, None, pos, p, inplace=True)[0], want)


def test_only_one_gradient(gpu):
    p = RopeAxes((16, 16))
    q, k, pos, dq, dk = inputs(gpu, 2, 9, 4, 2, 64, BF, 2, 8)
    _, (gq, gk) = run_and_check((q, k, pos, dq, dk), p)
    leaf = k.detach().requires_grad_()
    oq, ok = apply_rope_axes(q, leaf, pos, p)
    (g,) = torch.autograd.grad(ok, leaf, dk)
    assert same(g, gk)
    leaf = q.detach().requires_grad_()
    oq, ok = apply_rope_axes(leaf, k, pos, p)
    (g,) = torch.autograd.grad(oq, leaf, dq)
    assert same(g, gq)


def test_empty(gpu):
    p = RopeAxes((4, 4))
    pos = torch.zeros(2, 0, 5, dtype=torch.int64, device=gpu)
    q = torch.empty(0, 5, 2, 16, device=gpu, requires_grad=True)
    o, k = apply_rope_axes(q, None, pos, p)
    (g,) = torch.autograd.grad(o, q, torch.empty_like(o))
    assert o.shape == g.shape == q.shape and k is None


def test_module_stream_hooks_and_graph(gpu):
    m = MultiAxisRotaryEmbedding((16, 24, 24), layout="blocks")
    q, k, pos, dq, dk = inputs(gpu, 2, 33, 8, 2, 128, BF, 3, 9)
    ref, grads = run_and_check((q, k, pos, dq, dk), m.plan)
    leaf = [q.requires_grad_(), k.requires_grad_()]

    def step():
        o = m(*leaf, pos)
        return (*o, *torch.autograd.grad(o, leaf, (dq, dk)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for ctx in (contextlib.nullcontext(), saved_elsewhere()):
        with torch.cuda.stream(s), ctx:
            out = step()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(out, (*ref, *grads)))
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            q.mul_(1.5)
            pos.add_(i)
        graph.replay()
        torch.cuda.synchronize()
        want, g = run_and_check((q.detach(), k.detach(), pos, dq, dk), m.plan)
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(out, (*want, *g))), i


def test_far_elements(gpu):
    """Elements past 2^32: the last tokens turn as they do alone."""
    p = RopeAxes((16, 24, 24))
    b, s, h, d = 2, 270000, 64, 128
    pos = torch.arange(s, device=gpu).expand(3, b, s)
    q = torch.zeros(b, s, h, d, dtype=BF, device=gpu)
    tail = inputs(gpu, 1, 40, h, 0, d, BF, 3, 5)[0]
    q[1, -40:] = tail[0]
    out = apply_rope_axes(q, None, pos, p)[0]
    want = apply_rope_axes(tail, None, pos[:, :1, -40:], p)[0]
    assert same(out[1, -40:], want[0]) and not out[0].any() and not out[1, :-40].any()
    apply_rope_axes(q, None, pos, p, inplace=True)
    assert same(q[1, -40:], want[0])


def test_any_position(gpu):
    """Positions out to both ends of int64, against angles in rational arithmetic (2 pi to 200 bits):
    cos and sin are off by 4 u and 2 pi 2^-33."""
    import numpy as np
    from fractions import Fraction
    inv = Fraction(0x28BE60DB9391054A7F09D5F47D4D377036D8A5664F10E410, 1 << 192)  # 1 / (2 pi)
    p = RopeAxes((24, 20, 20), layout="interleaved", base=500000.0)
    base = [1 << 20, 1 << 38, 1 << 40, 1 << 46, -(1 << 52), 1 << 57, 1 << 62, -(1 << 62),
            (1 << 63) - 1, -(1 << 63)]
    pos = np.array([[b // (a + 1) + (a if abs(b) < 1 << 62 else 0) for b in base] for a in range(3)],
                   dtype=np.int64)
    pos[:, -2:] = base[-2:]
    turn = [[float(int(pos[a, s]) * Fraction(f) * inv % 1) for a, f in zip(p.axis, p.inv_freq.tolist())]
            for s in range(len(base))]
    angle = 2 * math.pi * torch.tensor(turn, dtype=torch.float64, device=gpu)[None, :, None]
    q, _, _, dq, _ = inputs(gpu, 1, len(base), 3, 0, 128, F32, 3, 11)
    leaf = q.requires_grad_()
    out, _ = apply_rope_axes(leaf, None, torch.from_numpy(pos).to(gpu), p)
    (grad,) = torch.autograd.grad(out, leaf, dq)
    for got, x, sign in ((out.detach(), q.detach(), 1), (grad, dq, -1)):
        lo, hi = x.double().chunk(2, -1)
        c, s = angle.cos(), sign * angle.sin()
        want = torch.cat((lo * c - hi * s, hi * c + lo * s), -1)
        mag = (lo.abs() + hi.abs()).repeat(1, 1, 1, 2)
        bad = ~((got.double() - want).abs() <= (7 * U + 2 * math.pi * 2.0 ** -33) * mag)
        assert not bad.any(), bad.nonzero()[:3].tolist()
