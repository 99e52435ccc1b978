"""Norms before and after a block against float64 on the GPU, forward and every gradient.

Tolerances, with u = 2^-24. A row's sum of squares runs through at most 32 products of a lane, 6
steps inside a wave and 16 waves: its square root's reciprocal is off by at most 27 u (plus the
division's and the root's roundings, 4 u in all), relatively, for exact terms. A term of h then
carries at most 35 u of itself, so h is off by at most 35 u M, M = |a x| + |g yhat w|, and rh by
(31 + 35 k) u, k = |M| / |h| in 2-norms: what cancels in h. Every other quantity of the backward is
a product of at most six such factors and a sum of depth 60 at most (columns: 8 steps of a lane, 8
row slots, 8 partial rows, 6 in the tree; more rows are counted), so it is off by at most
K = 6 (66 + 35 k) + 60 + rows / 512 times u times the same quantity formed from magnitudes
(every difference a sum). 16-bit results add half a step of their type.
"""
import contextlib

import pytest
import torch

from helpers import BF, F16, F32, Guarded, flat, same, saved_elsewhere
from trainscale_amd import _lib
from trainscale_amd.kernels import (FusedSandwichRMSNorm, fused_add_rms_layernorm,
                                    fused_sandwich_rms_layernorm)

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


def half(dtype):
    return torch.finfo(dtype).eps / 2


def reference(y, x, post, pre, gate, a, o, dn, dh):
    """Results in float64 and, for each, its error bound before the final rounding."""
    d = torch.float64
    lead = tuple(range(y.dim() - 1))
    leaf = [t.detach().to(d).requires_grad_() if t is not None else None
            for t in (y, x, post, pre, gate)]
    Y, X, P, Q, G = leaf
    ry = 1 / (Y.square().mean(-1, keepdim=True) + EPS).sqrt()
    br = Y * ry * (P + o)
    if G is not None:
        br = br * G
    h = a * X + br
    rh = 1 / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
    n = h * rh * (Q + o)
    dn64 = torch.zeros_like(n) if dn is None else dn.to(d)
    dh64 = torch.zeros_like(n) if dh is None else dh.to(d)
    grads = torch.autograd.grad((n, h), [t for t in leaf if t is not None], (dn64, dh64))
    out = dict(n=n, h=h, **dict(zip([k for k, t in zip(("dy", "dx", "dpost", "dpre", "dgate"), leaf)
                                     if t is not None], grads)))
    with torch.no_grad():
        one = torch.ones((), dtype=d, device=y.device)
        g = one if G is None else G.abs()
        u0, yh = g * (P + o).abs(), (Y * ry).abs()
        w, M = (Q + o).abs(), (a * X).abs() + br.abs()
        k = M.norm(dim=-1, keepdim=True) / h.norm(dim=-1, keepdim=True).clamp(min=1e-30)
        K = (6 * (66 + 35 * k) + 60 + y[..., 0].numel() / 512) * U
        Hm, um, e = M * rh, br.abs(), dn64.abs() * w
        mean = lambda t: t.mean(-1, keepdim=True)
        c1 = mean(e * Hm)
        t = dh64.abs() + rh * (e + Hm * c1)
        c2 = mean((dh64.abs() + rh * e) * um) + rh * c1 * mean(Hm * um)
        bound = dict(h=35 * U * M, n=K * M * rh * w, dx=K * abs(a) * t,
                     dy=K * ry * (t * u0 + yh * c2), dpre=(K * dn64.abs() * Hm).sum(lead),
                     dpost=(K * t * yh * g).sum(lead))
        if G is not None:
            full = K * t * yh * (P + o).abs()
            bound["dgate"] = full.sum_to_size(G.shape)
    return out, bound


def check(got, want, bound, what):
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    tol = bound * (1 + half(got.dtype)) + half(got.dtype) * want.abs() + tiny
    bad = ~((got.double() - want).abs() <= tol)
    assert got.shape == want.shape and not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist())


def inputs(gpu, shape, dtype, wdtype, gate, gdtype, o, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=gpu, generator=g)
    h = shape[-1]
    mean = 1 - o
    gs = {"none": None, "channel": (h,), "batch": (shape[0],) + (1,) * (len(shape) - 2) + (h,),
          "full": shape}[gate]
    return [(0.7 * r(*shape)).to(dtype), (2 * r(*shape)).to(dtype), (mean + 0.1 * r(h)).to(wdtype),
            (mean + 0.1 * r(h)).to(wdtype), None if gs is None else (0.3 + 0.3 * r(*gs)).to(gdtype),
            r(*shape).to(dtype), r(*shape).to(dtype)]


def run_and_check(args, a, o, use=(True, True)):
    y, x, post, pre, gate, dn, dh = args
    leaves = [t.requires_grad_() if t is not None else None for t in (y, x, post, pre, gate)]
    n, h = fused_sandwich_rms_layernorm(y, x, post, pre, gate, EPS, a, o)
    outs = [t for t, k in zip((n, h), use) if k]
    ups = [t for t, k in zip((dn, dh), use) if k]
    grads = torch.autograd.grad(outs, [t for t in leaves if t is not None], ups)
    want, bound = reference(y, x, post, pre, gate, a, o, dn if use[0] else None,
                            dh if use[1] else None)
    names = [k for k, t in zip(("dy", "dx", "dpost", "dpre", "dgate"), leaves) if t is not None]
    for k, v in dict(n=n, h=h, **dict(zip(names, grads))).items():
        check(v.detach(), want[k].detach(), bound[k], k)
    return dict(n=n, h=h, **dict(zip(names, grads)))


WIDTHS = [1, 5, 8, 64, 72, 513, 1000, 1024, 2056, 4096, 4100, 8192]


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(gpu, width, dtype):
    run_and_check(inputs(gpu, (11, width), dtype, dtype, "none", None, 0.0, width), 1.0, 0.0)
    run_and_check(inputs(gpu, (3, 7, width), dtype, F32, "batch", dtype, 1.0, width + 1), 0.5, 1.0)


@pytest.mark.parametrize("width,dtype", [(16384, BF), (16383, F16), (8191, F32), (12000, BF)])
def test_widest(gpu, width, dtype):
    run_and_check(inputs(gpu, (2, 5, width), dtype, dtype, "channel", F32, 0.0, 1), 1.0, 0.0)


@pytest.mark.parametrize("rows", [1, 2, 7, 513, 3000])
@pytest.mark.parametrize("gate", ["none", "channel", "full"])
def test_rows(gpu, rows, gate):
    run_and_check(inputs(gpu, (rows, 264), BF, BF, gate, BF, 1.0, rows), -0.7, 1.0)


@pytest.mark.parametrize("shape", [(1, 1, 128), (600, 1, 128), (1, 1000, 128), (17, 33, 130),
                                   (2, 3, 5, 256), (4, 513, 4096)])
def test_gate_groups(gpu, shape):
    run_and_check(inputs(gpu, shape, BF, BF, "batch", F32, 0.0, 3), 1.0, 0.0)
    run_and_check(inputs(gpu, shape, F32, F32, "batch", F32, 0.0, 4), 1.0, 0.0)


@pytest.mark.parametrize("use", [(True, False), (False, True)])
def test_one_result_used(gpu, use):
    run_and_check(inputs(gpu, (5, 9, 512), BF, F32, "batch", BF, 0.0, 5), 1.0, 0.0, use)


def test_only_some_gradients(gpu):
    y, x, post, pre, gate, dn, dh = inputs(gpu, (3, 40, 256), BF, BF, "batch", BF, 0.0, 6)
    names = ("y", "x", "post", "pre", "gate")
    tensors = dict(zip(names, (y, x, post, pre, gate)))
    full = None
    for wanted in (names, ("y",), ("x",), ("post",), ("pre",), ("gate",), ("x", "gate")):
        t = {k: v.detach().clone().requires_grad_(k in wanted) for k, v in tensors.items()}
        n, h = fused_sandwich_rms_layernorm(t["y"], t["x"], t["post"], t["pre"], t["gate"])
        g = dict(zip(wanted, torch.autograd.grad((n, h), [t[k] for k in wanted], (dn, dh))))
        full = full or g
        assert all(same(g[k], full[k]) for k in wanted), wanted


def test_against_differences(gpu):
    y, x, post, pre, gate, dn, dh = inputs(gpu, (2, 6, 40), F32, F32, "batch", F32, 0.0, 7)
    leaves = [t.requires_grad_() for t in (y, x, post, pre, gate)]
    n, h = fused_sandwich_rms_layernorm(*leaves, EPS, 0.8)
    grads = torch.autograd.grad((n, h), leaves, (dn, dh))
    _, bound = reference(y, x, post, pre, gate, 0.8, 0.0, dn, dh)

    def value(ts):
        Y, X, P, Q, G = ts
        hh = 0.8 * X + G * Y / (Y.square().mean(-1, keepdim=True) + EPS).sqrt() * P
        nn = hh / (hh.square().mean(-1, keepdim=True) + EPS).sqrt() * Q
        return float((nn * dn).sum() + (hh * dh).sum())

    base = [t.detach().double() for t in leaves]
    g = torch.Generator(device=gpu).manual_seed(8)
    for i, name in enumerate(("dy", "dx", "dpost", "dpre", "dgate")):
        dirn = torch.randn(base[i].shape, device=gpu, generator=g, dtype=torch.float64)
        step = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + step * dirn, base[i] - step * dirn
        diff = (value(up) - value(down)) / (2 * step)
        got = float((grads[i].double() * dirn).sum())
        # the kernel's bound along the direction; the difference's own error is step^2 times a
        # third derivative of order 10 n over 500 terms, and 1e-16 / step of its values
        tol = float(((bound[name] + U * grads[i].abs()) * dirn.abs()).sum()) + 1e-6
        assert abs(got - diff) <= tol, (name, got, diff, tol)


def test_layouts_and_determinism(gpu):
    y, x, post, pre, gate, dn, dh = inputs(gpu, (4, 50, 256), BF, BF, "batch", BF, 0.0, 9)
    ref = run_and_check([y, x, post, pre, gate, dn, dh], 1.0, 0.0)

    def strided(t):  # unaligned rows inside a wider buffer of NaN
        w = torch.full((*t.shape[:-1], 263), float("nan"), dtype=t.dtype, device=gpu)
        w[..., 3:259] = t.detach()
        return w[..., 3:259]

    again = run_and_check([strided(t) for t in (y, x)] + [post, pre, gate]
                          + [strided(t) for t in (dn, dh)], 1.0, 0.0)
    assert all(same(ref[k], again[k]) for k in ref)
    t = run_and_check([t.detach().transpose(0, 1).contiguous().transpose(0, 1) for t in (y, x)]
                      + [post.detach(), pre.detach(), gate.detach(), dn, dh], 1.0, 0.0)
    assert all(same(ref[k].contiguous(), t[k].contiguous()) for k in ref)
    # upstream gradients without memory of their own
    n, h = fused_sandwich_rms_layernorm(y, x, post, pre, gate)
    g = torch.autograd.grad(n.float().sum() + h.float().sum(), [y, x, post, pre, gate])
    want, bound = reference(y, x, post, pre, gate, 1.0, 0.0, torch.ones_like(dn), torch.ones_like(dh))
    for k, v in zip(("dy", "dx", "dpost", "dpre", "dgate"), g):
        check(v, want[k], bound[k], k)


def test_empty_and_extreme_rows(gpu):
    y, x, post, pre, gate, dn, dh = inputs(gpu, (0, 5, 64), BF, BF, "batch", BF, 0.0, 1)
    leaves = [t.requires_grad_() for t in (y, x, post, pre, gate)]
    n, h = fused_sandwich_rms_layernorm(*leaves)
    assert n.shape == h.shape == (0, 5, 64)
    for t, g in zip(leaves, torch.autograd.grad((n, h), leaves, (dn, dh))):
        assert g.shape == t.shape and not g.any()
    # zero rows, rows of one value, and rows whose block is tiny beside the stream
    y, x, post, pre, gate, dn, dh = inputs(gpu, (6, 300), F32, F32, "channel", F32, 0.0, 2)
    y[0] = 0
    x[0] = 0
    y[1] = 0
    x[2] = 0
    y[3] *= 1e-4
    x[4] *= 1e3
    y[5] = 3.0
    run_and_check([y, x, post, pre, gate, dn, dh], 1.0, 0.0)
    # a NaN or an infinity stays in its row
    y, x, post, pre, gate, dn, dh = inputs(gpu, (6, 300), BF, BF, "channel", BF, 0.0, 2)
    clean = fused_sandwich_rms_layernorm(y, x, post, pre, gate)
    y[2, 5], x[4, 7] = float("nan"), float("inf")
    n, h = fused_sandwich_rms_layernorm(y, x, post, pre, gate)
    keep = [0, 1, 3, 5]
    assert same(n[keep], clean[0][keep]) and same(h[keep], clean[1][keep])
    assert bool(n[2].isnan().all()) and bool(n[4].isnan().any())


@pytest.mark.parametrize("dtype,width", [(BF, 256), (BF, 259), (F32, 1001), (F16, 4099), (BF, 9001)])
def test_stays_inside(gpu, dtype, width):
    lib, st, code = _lib.load(), _lib.stream_handle(gpu), _lib.DTYPE_CODE[dtype]
    rows, groups = 12, 3
    y, x, post, pre, gate, dn, dh = inputs(gpu, (groups, 4, width), dtype, dtype, "batch", dtype,
                                           0.0, width)
    want, bound = reference(y, x, post, pre, gate, 1.0, 0.0, dn, dh)
    G = lambda t, pad=0: Guarded(rows, width, width + pad, dtype, gpu, t.reshape(rows, width))
    gy, gx, gdn, gdh = G(y, 1), G(x, 3), G(dn, 5), G(dh, 8)
    gp, gq, gg = flat(width, dtype, gpu, post), flat(width, dtype, gpu, pre), flat(
        groups * width, dtype, gpu, gate)
    out = {k: Guarded(rows, width, width + 7, dtype, gpu) for k in ("n", "h", "dy", "dx")}
    par = {k: flat(s, dtype, gpu) for k, s in (("dpost", width), ("dpre", width),
                                               ("dgate", groups * width))}
    ry, rh = flat(rows, F32, gpu), flat(rows, F32, gpu)
    wsb = int(lib.ts_sandwich_norm_bwd_workspace_size(rows, width, groups))
    ws = flat(wsb, torch.uint8, gpu)
    _lib.check(lib.ts_sandwich_norm_fwd(
        gy.p, width + 1, gx.p, width + 3, code, gp.p, gq.p, code, gg.p, code, groups, out["n"].p,
        width + 7, out["h"].p, width + 7, ry.p, rh.p, rows, width, 1.0, 0.0, EPS, st), "fwd")
    _lib.check(lib.ts_sandwich_norm_bwd(
        gdn.p, width + 5, gdh.p, width + 8, gy.p, width + 1, gx.p, width + 3, code, gp.p, gq.p, code,
        gg.p, code, groups, ry.p, rh.p, out["dy"].p, width + 7, out["dx"].p, width + 7,
        par["dpost"].p, par["dpre"].p, par["dgate"].p, rows, width, 1.0, 0.0, ws.p, wsb, st), "bwd")
    for t in (gy, gx, gdn, gdh, gp, gq, gg, ry, rh, ws, *out.values(), *par.values()):
        assert t.intact()
    for k, t in {**out, **par}.items():
        check(t.t.reshape(want[k].shape), want[k].detach(), bound[k], k)


def test_module_and_neighbours(gpu):
    # without norm, gate and scale before the sum the boundary is the fused add + norm that is there
    m = FusedSandwichRMSNorm(128, weight_offset=1.0, layer_gate=True, device=gpu, dtype=F32)
    x = torch.randn(4, 9, 128, device=gpu)
    y = torch.randn(4, 9, 128, device=gpu)
    n, h = m(y, x)
    yn = y / (y.double().square().mean(-1, keepdim=True) + EPS).sqrt().float()
    n2, h2 = fused_add_rms_layernorm(yn, x, torch.ones(128, device=gpu), EPS, return_residual=True)
    assert torch.allclose(n, n2, rtol=1e-5, atol=1e-5) and torch.allclose(h, h2, rtol=1e-5, atol=1e-5)
    (n.sum() + h.sum()).backward()
    assert all(p.grad is not None and p.grad.shape == p.shape for p in m.parameters())


def test_stream_and_graph(gpu):
    y, x, post, pre, gate, dn, dh = inputs(gpu, (2, 300, 512), BF, BF, "batch", BF, 0.0, 11)
    leaves = [t.requires_grad_() for t in (y, x, post, pre, gate)]

    def step():
        n, h = fused_sandwich_rms_layernorm(*leaves)
        return [n.detach(), h.detach(), *torch.autograd.grad((n, h), leaves, (dn, dh))]

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
        with torch.no_grad():
            if rep:
                for t in (y, x, dn, dh):
                    t.copy_(torch.randn(t.shape, device=gpu))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        ref = step()
        assert all(same(p, q) for p, q in zip(outs, ref)), rep
        if rep == 0:
            assert all(same(p, q) for p, q in zip(first, ref))


@pytest.mark.parametrize("width", [256, 263])
def test_saved_tensors_elsewhere(gpu, width):
    y, x, post, pre, gate, dn, dh = inputs(gpu, (4, 50, 256), BF, BF, "batch", BF, 0.0, 21)
    base = [torch.cat([t, t[..., :width - 256]], -1) for t in (y, x)]  # rows of a wider buffer

    def grads(hooks):
        leaves = [t.detach().requires_grad_() for t in (*base, post, pre, gate)]
        with hooks:
            n, h = fused_sandwich_rms_layernorm(leaves[0][..., :256], leaves[1][..., :256],
                                                *leaves[2:], EPS)
        return torch.autograd.grad([n, h], leaves, [dn, dh])

    want, got = grads(contextlib.nullcontext()), grads(saved_elsewhere())
    assert all(same(a, b) for a, b in zip(want, got))
