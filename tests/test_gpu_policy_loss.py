"""Clipped policy loss against float64 on the GPU, values and gradient.

Tolerances, u = 2^-24, for one token: d is exact and rounded once to fp32 (|d| u in the ratio),
exp is good to 2 u and the product rounds once: r A is off by (|d| + 3) u |r A|. The KL estimate:
x is rounded once, which moves it by |x| |exp(x) - 1| u; its series loses at most 16 roundings of
the sum, and above |x| = 1/2 the difference expm1(x) - x is off by 3 u (|expm1(x)| + |x|). Sums are
in double and rounded once. The gradient adds kl_coef expm1(x) (3 u and u |x| exp(x)), the sum and
the products with the weight and the upstream gradient (4 u of the magnitudes). 16-bit gradients
add half a step of their type. Fractions are counts in double, rounded once.
"""
import math

import pytest
import torch

from helpers import BF, F16, F32, Guarded, flat, same, saved_elsewhere
from trainscale_amd import _lib, ops
from trainscale_amd.loss import (ClippedPolicyLoss, chunked_log_softmax, clipped_policy_loss,
                                 selective_log_softmax)

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
REDUCTIONS = ["token", "sequence", "sum"]


def reference(lp, old, adv, mask, ref, low, high, beta, reduction, upstream=1.0):
    """float64 values (loss, policy, kl, clipped, gradient) and their bounds."""
    lp64 = lp.detach().double()
    keep = torch.ones_like(lp64, dtype=torch.bool) if mask is None else mask != 0
    z = torch.zeros_like(lp64)
    lp64 = torch.where(keep, lp64, z)
    d = z if old is None else torch.where(keep, lp64 - old.double(), z)
    A = adv.double()
    A = torch.where(keep, A[:, None].expand_as(lp64) if A.dim() == 1 else A, z)
    r = d.exp()
    free, held = r * A, r.clamp(1 - low, 1 + high) * A
    clipped = held < free
    pol, gpol = -torch.minimum(free, held), torch.where(clipped, z, -free)
    x = z if ref is None else torch.where(keep, ref.double() - lp64, z)
    kl, rise = torch.expm1(x) - x, torch.expm1(x)
    lens = keep.sum(1, keepdim=True).double()
    some = float((lens > 0).sum())
    w = {"token": torch.ones_like(lens) / max(1.0, float(lens.sum())),
         "sequence": torch.where(lens > 0, 1 / lens.clamp(min=1), 0 * lens) / max(1.0, some),
         "sum": torch.ones_like(lens)}[reduction]
    wk = w * keep
    grad = upstream * wk * (gpol - beta * rise)
    e_pol = (d.abs() + 3) * U * torch.maximum(free.abs(), pol.abs())
    e_kl = x.abs() * rise.abs() * U + torch.where(x.abs() < 0.51, 16 * U * kl,
                                                   3 * U * (rise.abs() + x.abs()))
    e_grad = abs(upstream) * wk * (torch.where(clipped, z, e_pol) + beta * (3 * U * rise.abs() + U * x.abs() * x.exp())
                   + 5 * U * (gpol.abs() + beta * rise.abs()))
    # a product of the weights may fall below fp32's normal numbers
    e_grad = e_grad + 2.0 ** -148
    s = lambda v: float((wk * v).sum())
    vals = (s(pol) + beta * s(kl), s(pol), s(kl), s(clipped.double()))
    errs = (s(e_pol) + beta * s(e_kl) + 2 * U * beta * s(kl), s(e_pol), s(e_kl), 0.0)
    return vals, errs, grad, e_grad


def check(got, grad, want, upstream=1.0):
    vals, errs, g, e = want
    for name, a, b, tol in zip(got._fields, got, vals, errs):
        assert a.dtype == F32 and a.dim() == 0
        assert abs(float(a) - b) <= tol + 2 * U * abs(b) + 1e-45, (name, float(a), b, tol)
    fi = torch.finfo(grad.dtype)
    tol = e + fi.eps / 2 * (g.abs() + e) + fi.smallest_normal * fi.eps
    bad = ~((grad.double() - g).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist())


def inputs(gpu, b, t, dtype, per_token=False, ref=True, masked=True, seed=0, spread=0.2):
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=gpu, generator=g)
    lp = -r(b, t).abs() - 0.05
    old = (lp + spread * r(b, t)).to(dtype)
    rf = (lp + 2 * spread * r(b, t)).to(dtype) if ref else None
    adv = r(b, t) if per_token else r(b)
    mask = torch.rand(b, t, device=gpu, generator=g) < 0.7 if masked else None
    if masked and b > 2:
        mask[b // 2] = False
    return lp.to(dtype), old, adv, mask, rf


def run(args, low=0.2, high=0.28, beta=0.04, reduction="token", upstream=None):
    lp, old, adv, mask, ref = args
    lp = lp.detach().requires_grad_()
    out = clipped_policy_loss(lp, old, adv, mask, ref, low, high, beta, reduction)
    up = None if upstream is None else torch.tensor(upstream, device=lp.device)
    (g,) = torch.autograd.grad(out.loss, lp, up)
    check(out, g, reference(lp, old, adv, mask, ref, low, high, beta, reduction,
                            1.0 if upstream is None else upstream))
    return out, g


SHAPES = [(1, 1), (1, 3), (2, 4), (3, 5), (4, 500), (7, 511), (5, 512), (5, 513), (64, 512),
          (65, 512), (33, 2047), (3000, 1), (1000, 9), (1, 70001), (3, 33000)]


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("b,t", SHAPES)
def test_shapes(gpu, b, t, dtype):
    for i, reduction in enumerate(REDUCTIONS):
        run(inputs(gpu, b, t, dtype, per_token=i != 1, seed=b + t + i), reduction=reduction)


@pytest.mark.parametrize("b,t", [(16, 512), (17, 512), (8, 513), (9, 513), (1, 8192), (1, 8193)])
def test_around_the_one_launch_form(gpu, b, t):
    for reduction in REDUCTIONS:
        run(inputs(gpu, b, t, F32, seed=b), reduction=reduction)


@pytest.mark.parametrize("per_token", [False, True])
@pytest.mark.parametrize("ref", [False, True])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("reduction", REDUCTIONS)
def test_options(gpu, per_token, ref, masked, reduction):
    args = inputs(gpu, 6, 300, F32, per_token, ref, masked, seed=3)
    run(args, beta=0.3 if ref else 0.0, reduction=reduction)
    run(args, beta=0.0, reduction=reduction, upstream=-2.5)
    run((args[0], None, *args[2:]), beta=0.1 if ref else 0.0, reduction=reduction)


@pytest.mark.parametrize("low,high", [(0.0, 0.0), (0.2, math.inf), (1.0, 0.2), (3.0, 5.0),
                                      (0.99, 0.01)])
def test_bounds(gpu, low, high):
    run(inputs(gpu, 4, 700, F32, True, seed=5, spread=0.6), low, high)


def test_small_and_large_differences(gpu):
    # the KL estimate of a reference next to the policy, and of one far away
    for spread in (1e-6, 1e-4, 1e-2, 0.25, 2.0, 10.0):
        lp, old, adv, mask, ref = inputs(gpu, 3, 900, F32, True, seed=6, spread=spread)
        run((lp, old, adv, mask, ref), beta=1.0)
    lp, old, adv, mask, ref = inputs(gpu, 2, 40, F32)
    out, g = run((lp, lp.clone(), adv, mask, lp.clone()), beta=1.0)
    assert float(out.kl) == 0.0 and float(out.clip_fraction) == 0.0


def test_next_to_the_border(gpu):
    # ratios a few steps of the log-probs on either side of the bounds: whether they are clipped
    # is decided by the exact difference
    lp = torch.zeros(2, 64, device=gpu)
    steps = torch.arange(-32, 32, device=gpu, dtype=torch.float64) * 2.0 ** -24
    old = torch.stack([-(math.log1p(0.28) + steps), -(math.log1p(-0.2) + steps)]).float()
    for sign in (1.0, -1.0):
        adv = torch.tensor([sign, sign], device=gpu)
        run((lp, old, adv, None, None), beta=0.0)


@pytest.mark.parametrize("b,t", [(5, 300), (200, 700)])
def test_masked_places_do_not_matter(gpu, b, t):
    lp, old, adv, mask, ref = inputs(gpu, b, t, F32, True, seed=8)
    base, g0 = run((lp, old, adv, mask, ref))
    bad = [float("nan"), float("inf"), -float("inf"), torch.finfo(F32).min]
    fill = torch.tensor(bad, device=gpu)[torch.randint(0, 4, (b, t), device=gpu)]
    dirty = [torch.where(mask, v, fill) for v in (lp, old, adv, ref)]
    lp2 = dirty[0].requires_grad_()
    out = clipped_policy_loss(lp2, dirty[1], dirty[2], mask, dirty[3], 0.2, 0.28, 0.04)
    (g,) = torch.autograd.grad(out.loss, lp2)
    assert all(same(p, q) for p, q in zip(base, out)) and same(g, g0)
    assert not g[~mask].any()
    # nothing valid at all
    none = torch.zeros_like(mask)
    for reduction in REDUCTIONS:
        out = clipped_policy_loss(lp2, dirty[1], dirty[2], none, dirty[3], kl_coef=0.04,
                                  reduction=reduction)
        assert all(float(v) == 0.0 for v in out)
        assert not torch.autograd.grad(out.loss, lp2)[0].any()
    # a NaN in a valid place shows
    ok = lp.clone()
    ok[mask.nonzero()[0, 0], mask.nonzero()[0, 1]] = float("nan")
    assert math.isnan(float(clipped_policy_loss(ok, old, adv, mask).loss))


def test_empty(gpu):
    for b, t in ((0, 5), (4, 0), (0, 0)):
        lp = torch.zeros(b, t, device=gpu, requires_grad=True)
        out = clipped_policy_loss(lp, lp.detach(), torch.zeros(b, device=gpu))
        assert all(float(v) == 0.0 for v in out)
        assert torch.autograd.grad(out.loss, lp)[0].shape == (b, t)


def test_against_differences(gpu):
    lp, old, adv, mask, ref = inputs(gpu, 3, 30, F32, True, seed=9)
    _, g = run((lp, old, adv, mask, ref), beta=0.5, reduction="sequence")
    gen = torch.Generator(device=gpu).manual_seed(10)
    dirn = torch.randn(lp.shape, device=gpu, generator=gen, dtype=torch.float64)
    step = 1e-6
    val = lambda v: reference(v, old, adv, mask, ref, 0.2, 0.28, 0.5, "sequence")[0][0]
    diff = (val(lp.double() + step * dirn) - val(lp.double() - step * dirn)) / (2 * step)
    # no ratio lies within a step of its bound (their distances are of the order 1e-3); the
    # difference is off by step^2 and by 1e-16 / step
    got = float((g.double() * dirn).sum())
    e = reference(lp, old, adv, mask, ref, 0.2, 0.28, 0.5, "sequence")[3]
    assert abs(got - diff) <= float(((e + U * g.abs()) * dirn.abs()).sum()) + 1e-8


def test_layouts_and_types(gpu):
    lp, old, adv, mask, ref = inputs(gpu, 9, 333, BF, True, seed=11)
    base, g0 = run((lp, old, adv, mask, ref))

    def inside(t):  # a slice at an odd offset of a wider tensor
        w = torch.zeros(9, 341, dtype=t.dtype, device=gpu)
        w[:, 3:336] = t
        return w[:, 3:336]

    out, g = run([inside(t) for t in (lp, old, adv, mask, ref)])
    assert all(same(p, q) for p, q in zip(base, out)) and same(g, g0)
    out, g = run([t.t().contiguous().t() for t in (lp, old, adv, mask, ref)])
    assert all(same(p, q) for p, q in zip(base, out)) and same(g, g0)
    out, g = run((lp, old.float(), adv, mask.long(), ref.float()))
    assert all(same(p, q) for p, q in zip(base, out)) and same(g, g0)
    a = adv[:, 0].contiguous()
    for shaped in (a, a[:, None], a[:, None].expand(9, 333), a[::1]):
        out, g = run((lp, old, shaped, mask, ref))
        first = first if shaped is not a else out
        assert all(same(p, q) for p, q in zip(first, out))
    run((lp, old, adv.to(BF).float(), mask.to(F32), ref))
    run((lp.float(), old, adv, mask.to(torch.uint8) * 7, ref.half()))  # fp32 logps, 16-bit others


def test_module_twice_and_no_gradient_elsewhere(gpu):
    lp, old, adv, mask, ref = inputs(gpu, 4, 100, F32, seed=12)
    m = ClippedPolicyLoss(0.1, 0.3, 0.2, "sequence")
    lp.requires_grad_()
    old.requires_grad_()
    ref.requires_grad_()
    out = m(lp, old, adv, mask, ref)
    assert out.loss.requires_grad and not out.kl.requires_grad and not out.policy_loss.requires_grad
    g1 = torch.autograd.grad(out.loss, lp, retain_graph=True)[0]
    g2 = torch.autograd.grad(out.loss * 3, lp, retain_graph=True)[0]
    check(out, g1, reference(lp, old.detach(), adv, mask, ref.detach(), 0.1, 0.3, 0.2, "sequence"))
    assert torch.allclose(3 * g1, g2, rtol=1e-6, atol=0)
    out.loss.backward()
    assert same(lp.grad, g1) and old.grad is None and ref.grad is None


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("b,t", [(3, 5), (3, 514), (300, 514)])
def test_stays_inside(gpu, b, t, dtype):
    lib, st = _lib.load(), _lib.stream_handle(gpu)
    lp, old, adv, mask, ref = inputs(gpu, b, t, dtype, True, seed=13)
    G = lambda v, pad, dt: Guarded(b, t, t + pad, dt, gpu, v)
    glp, gold, gref, gadv = G(lp, 1, dtype), G(old, 3, dtype), G(ref, 2, dtype), G(adv, 5, F32)
    gmask = G(mask.to(torch.uint8), 1, torch.uint8)
    p = ops.policy_inputs(glp.t, gold.t, gadv.t, gmask.t, gref.t, 0.2, 0.28, 0.04, "token")
    outs = [flat(1, F32, gpu) for _ in range(4)]
    w, dl, grad = flat(b, F32, gpu), flat(1, F32, gpu, torch.ones(1)), Guarded(b, t, t + 1, dtype, gpu)
    wsb = int(lib.ts_policy_loss_workspace_size(b, t))
    ws = flat(max(wsb, 1), torch.uint8, gpu)
    import ctypes
    _lib.check(lib.ts_policy_loss_fwd(ctypes.byref(p), *[o.p for o in outs], w.p, ws.p, wsb, st), "f")
    _lib.check(lib.ts_policy_loss_bwd(ctypes.byref(p), w.p, dl.p, grad.p, t + 1, st), "b")
    for x in (glp, gold, gref, gadv, gmask, *outs, w, dl, grad, ws):
        assert x.intact()
    ref_out, ref_g = run((lp, old, adv, mask, ref))
    assert all(same(o.t.reshape(()), r) for o, r in zip(outs, ref_out)) and same(grad.t, ref_g)


def test_stream_and_graph(gpu):
    for b, t in ((4, 100), (100, 1000)):
        lp, old, adv, mask, ref = inputs(gpu, b, t, F32, seed=14)
        lp.requires_grad_()

        def step():
            out = clipped_policy_loss(lp, old, adv, mask, ref, kl_coef=0.1, reduction="sequence")
            return [v.detach() for v in out] + list(torch.autograd.grad(out.loss, lp))

        side = torch.cuda.Stream(gpu)
        side.wait_stream(torch.cuda.current_stream(gpu))
        with torch.cuda.stream(side):
            first = step()
        torch.cuda.current_stream(gpu).wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        for rep in range(4):
            if rep:
                with torch.no_grad():
                    lp.copy_(-torch.rand(b, t, device=gpu))
                    adv.copy_(torch.randn(b, device=gpu))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            now = step()
            assert all(same(p, q) for p, q in zip(outs, now)), (b, rep)
            if rep == 0:
                assert all(same(p, q) for p, q in zip(first, now))


def test_on_the_layers_log_probs(gpu):
    # through the log-prob drop-ins: the gradient reaches logits, hidden states and the LM head
    g = torch.Generator(device=gpu).manual_seed(15)
    b, t, h, v = 2, 20, 64, 500
    hid = torch.randn(b, t, h, device=gpu, generator=g).to(BF).requires_grad_()
    head = (0.1 * torch.randn(v, h, device=gpu, generator=g)).to(BF).requires_grad_()
    ids = torch.randint(0, v, (b, t), device=gpu, generator=g)
    adv = torch.randn(b, device=gpu, generator=g)
    lp = chunked_log_softmax(hid, head, ids, out_dtype=F32)
    old = (lp + 0.1).detach()
    out = clipped_policy_loss(lp, old, adv)
    gh, gw, glp = torch.autograd.grad(out.loss, (hid, head, lp))
    check(out, glp, reference(lp, old, adv, None, None, 0.2, 0.2, 0.0, "token"))
    assert bool(gh.any()) and bool(gw.any()) and gh.isfinite().all() and gw.isfinite().all()
    logits = (hid.detach() @ head.detach().t()).requires_grad_()
    lp2 = selective_log_softmax(logits, ids, out_dtype=F32)
    (gl,) = torch.autograd.grad(clipped_policy_loss(lp2, old, adv).loss, logits)
    assert gl.shape == logits.shape and bool(gl.any())


@pytest.mark.parametrize("how", ["moved", "checkpoint"])
def test_saved_tensors_elsewhere(gpu, how):
    from torch.utils.checkpoint import checkpoint
    args = inputs(gpu, 6, 777, F32)
    lp, rest = args[0].detach(), args[1:]

    def loss(x):
        # every operand is formed here: only what is saved keeps it
        old, adv, mask, ref = [t.clone() for t in rest]
        return clipped_policy_loss(x * 1.5, old, adv, mask, ref, 0.2, 0.28, 0.04, "sequence").loss

    def grad(call):
        x = lp.clone().requires_grad_()
        out = call(x)
        # the allocator's free blocks of these sizes are used again
        held = [torch.full_like(lp, float("nan")) for _ in range(8)]
        (g,) = torch.autograd.grad(out, x)
        del held
        return g

    want = grad(loss)
    if how == "checkpoint":
        got = grad(lambda x: checkpoint(loss, x, use_reentrant=False))
    else:
        def moved(x):
            with saved_elsewhere():
                return loss(x)
        got = grad(moved)
    assert torch.isfinite(want).all() and same(got, want)


# Log ratios whose exp leaves fp32's range, and infinite ones
FAR = [0.25, 80.0, 88.0, 89.0, 95.0, 110.0, 800.0, math.inf, -80.0, -89.0, -800.0, -math.inf]


def far_case(gpu, dtype, adv_of, beta, low, high, reduction, upstream):
    """One far log ratio a row, among ordinary tokens: the loss's tensors and the gradient with
    the definition's values in float64 (the policy's term of a token with A = 0 is 0 for any finite
    difference; what is infinite follows float64's arithmetic)."""
    b, t = len(FAR) * (2 if beta else 1), 7
    g = torch.Generator(device=gpu).manual_seed(16)
    lp = -torch.rand(b, t, device=gpu, generator=g)
    old = (lp + 0.1 * torch.randn(b, t, device=gpu, generator=g)).to(dtype)
    ref = (lp + 0.1 * torch.randn(b, t, device=gpu, generator=g)).to(dtype)
    lp = lp.to(dtype)
    lp[:, 3] = 0
    old[:, 3] = ref[:, 3] = 0
    old[:len(FAR), 3] = -torch.tensor(FAR, device=gpu).to(dtype)
    if beta:
        ref[len(FAR):, 3] = torch.tensor(FAR, device=gpu).to(dtype)
    adv = torch.full((b,), float(adv_of), device=gpu)
    lp.requires_grad_()
    out = clipped_policy_loss(lp, old, adv, None, ref if beta else None, low, high, beta, reduction)
    (grad,) = torch.autograd.grad(out.loss, lp, torch.tensor(upstream, device=gpu))

    d, A = lp.detach().double() - old.double(), adv.double()[:, None]
    r = d.exp()
    clipped = ((A > 0) & (r > 1 + high)) | ((A < 0) & (r < 1 - low))
    held = r.clamp(1 - low, 1 + high) if low < 1 else r.clamp(max=1 + high)
    zero = (A == 0) & d.isfinite()
    pol = torch.where(zero, 0.0, -torch.where(clipped, held, r) * A)
    gpol = torch.where(zero | clipped, 0.0, -r * A)
    x = ref.double() - lp.detach().double() if beta else torch.zeros_like(d)
    rise = torch.expm1(x)
    w = upstream * {"sum": 1.0, "token": 1.0 / (b * t), "sequence": 1.0 / (b * t)}[reduction]
    want = w * (gpol - beta * rise if beta else gpol)
    # |d| |r A| and |x| exp(x) are 0 in the limit of minus infinity, where exp gives an exact 0
    e = abs(w) * (torch.where(gpol == 0, 0.0, (d.abs() + 3) * U * gpol.abs())
                  + beta * (3 * U * rise.abs() + U * torch.where(x.isneginf(), 0.0, x.abs() * x.exp()))
                  + 5 * U * (gpol.abs() + beta * rise.abs())
                  # an exp below fp32's normal numbers becomes 0: up to 2^-126, times |A| in r A
                  + 2.0 ** -126 * (1 + A.abs()))
    fi = torch.finfo(dtype)
    tol = e + fi.eps / 2 * (want.abs() + e) + fi.smallest_normal * fi.eps
    rounded = want.to(dtype)  # infinities where the value leaves the type's range
    ok = torch.where(rounded.isfinite(), (grad.double() - want).abs() <= tol,
                     (grad == rounded) | (grad.isnan() & rounded.isnan()))
    assert bool(ok.all()), [(k, grad[k].tolist(), want[k].tolist())
                            for k in (~ok).any(1).nonzero()[:3, 0].tolist()]
    return out, pol, torch.expm1(x) - x, rounded


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("adv", [-1, 0, 1, -1e4])
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_exp_beyond_fp32(gpu, dtype, adv, beta):
    finite = 0
    for low, high in ((0.2, 0.2), (1.0, math.inf)):
        for reduction, upstream in (("sum", 1.0), ("token", 1e-4), ("sequence", -1e-6)):
            *_, want = far_case(gpu, dtype, adv, beta, low, high, reduction, upstream)
            finite += int(want.isfinite().sum())
            assert bool(want.isinf().any() or adv >= 0)
    assert finite > 0


def one_token(gpu, lp, old, adv, ref=None, **k):
    lp, old, adv = [torch.tensor([[v]], device=gpu, dtype=F32) for v in (lp, old, adv)]
    ref = None if ref is None else torch.tensor([[ref]], device=gpu, dtype=F32)
    return clipped_policy_loss(lp, old, adv, None, ref, reduction="sum", **k)


@pytest.mark.parametrize("d", FAR)
def test_loss_of_far_tokens(gpu, d):
    r = float(torch.tensor(d, dtype=torch.float64).exp())
    for adv in (-1.0, 1.0):
        got = one_token(gpu, 0.0, -d, adv)
        want = -min(r * adv, min(max(r, 0.8), 1.2) * adv)
        want = math.inf if want > 3.5e38 else want
        assert float(got.loss) == want or abs(float(got.loss) - want) <= 2 * U * abs(want) + 2.0 ** -149
    got = float(one_token(gpu, 0.0, -d, 0.0).loss)
    assert got == 0.0 or (math.isinf(d) and math.isnan(got))


@pytest.mark.parametrize("b,t", [(3, 50), (70, 600)])  # both forms of the forward
@pytest.mark.parametrize("far", [-math.inf, 1e30])
def test_infinite_kl_that_is_only_watched(gpu, b, t, far):
    lp, old, adv, _, ref = inputs(gpu, b, t, F32, masked=False, seed=17)
    ref[1, 7] = far
    lp.requires_grad_()
    out = clipped_policy_loss(lp, old, adv, None, ref, kl_coef=0.0)
    assert float(out.kl) == math.inf
    want = clipped_policy_loss(lp, old, adv, None, None)
    assert math.isfinite(float(want.loss)) and same(out.loss, want.loss)
    assert same(out.loss, out.policy_loss)
    assert same(*[torch.autograd.grad(o.loss, lp)[0] for o in (out, want)])
    assert float(clipped_policy_loss(lp, old, adv, None, ref, kl_coef=0.1).loss) == math.inf
