"""The gated feed-forward block against float64 on the GPU, forward and every gradient.

Tolerances hold for each row of a result, in 2-norms. With u = 2^-24 and h half a step of the data
type: an fp32 sum of K exact products is off by at most K u times the sum of magnitudes. An
activation t of g is off by at most 24 u |g| (the argument of its exponential carries at most 4
roundings, which move t by at most 8 u |g|; the exponential, reciprocal or erfc and two products
add 16 u |t|, and |t| <= |g|), its derivative by 16 u (1 + |g|); |act'| <= 1.2 and |act''| <= 1
carry the error of g on (relu: its derivative is off by 1 where the sign of g is in doubt). The
gated product, dg and du are rounded to the data type once, g and u where they are kept. Products
of matrices carry errors on as |E B|_2 <= |E|_2 times B's spectral norm. Results add h of
themselves.
"""
import copy

import pytest
import torch

from helpers import BF, F16, saved_elsewhere, same
from trainscale_amd.kernels import FusedGatedMLP, fused_gated_linear, fused_gated_mlp

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACTS = ["silu", "gelu", "gelu_tanh", "relu"]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def act64(act, g):
    if act == "silu":
        return g * torch.sigmoid(g)
    if act == "gelu":
        return torch.nn.functional.gelu(g)
    if act == "gelu_tanh":
        return torch.nn.functional.gelu(g, approximate="tanh")
    return torch.relu(g)


def spectral(t):
    """An upper bound on the spectral norm: one squaring of the Gram matrix."""
    m = t.t() @ t if t.shape[0] > t.shape[1] else t @ t.t()
    return float(torch.linalg.matrix_norm(m @ m)) ** 0.25


def rows(t):
    return torch.linalg.vector_norm(t, dim=1)


def product(A, EA, B, EB=None):
    """A B^T with the row-wise bound on its error: A off by EA, B by EB, an fp32 sum."""
    e = rows(EA) * spectral(B) + A.shape[1] * U * rows(A.abs() + EA) * torch.linalg.matrix_norm(B)
    if EB is not None:
        e = e + rows(A.abs() + EA) * torch.linalg.matrix_norm(EB)
    return A @ B.t(), e


def reference(x, wg, wu, wd, act, dy):
    """Results in float64 and the row-wise bounds before the last rounding."""
    h, d = half(x.dtype), torch.float64
    x, wg, wu = x.to(d), wg.to(d), wu.to(d)
    N, H, F = x.shape[0], x.shape[1], wg.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = H * U * (x.abs() @ wg.abs().t()), H * U * (x.abs() @ wu.abs().t())
    gl = g.clone().requires_grad_()
    t = act64(act, gl)
    (dt,) = torch.autograd.grad(t.sum(), gl)
    t = t.detach()
    et = 1.2 * eg + 24 * U * (g.abs() + eg)
    a = t * u
    ea = (et * (u.abs() + eu) + t.abs() * eu) * (1 + U) + U * a.abs()
    ea = ea * (1 + h) + h * a.abs() + tiny(dy.dtype)
    out, bound = {}, {}
    if wd is None:
        out["y"], bound["y"] = a, rows(ea)
        da, eda = dy.to(d), torch.zeros_like(a)
    else:
        wd = wd.to(d)
        out["y"], bound["y"] = product(a, ea, wd)
        dyd = dy.to(d)
        da = dyd @ wd
        eda = wd.shape[0] * U * (dyd.abs() @ wd.abs())
        out["dwd"], bound["dwd"] = product(dyd.t(), torch.zeros_like(dyd.t()), a.t(), ea.t())
    # from the kept, rounded g and u
    eg, eu = eg + h * (g.abs() + eg) + tiny(dy.dtype), eu + h * (u.abs() + eu) + tiny(dy.dtype)
    et = 1.2 * eg + 24 * U * (g.abs() + eg)
    ed = eg + 16 * U * (1 + g.abs() + eg)
    if act == "relu":
        ed = torch.where(g.abs() <= eg, 1.0, 0.0)
    dg, du = da * u * dt, da * t
    A, Ug, D = da.abs() + eda, u.abs() + eu, dt.abs() + ed
    edg = eda * Ug * D + A * eu * D + A * Ug * ed + 2 * U * A * Ug * D
    edu = eda * (t.abs() + et) + A * et + U * A * (t.abs() + et)
    edg = edg * (1 + h) + h * dg.abs() + tiny(dy.dtype)
    edu = edu * (1 + h) + h * du.abs() + tiny(dy.dtype)
    p, q = product(dg, edg, wg.t()), product(du, edu, wu.t())
    out["dx"], bound["dx"] = p[0] + q[0], 2 * (p[1] + q[1])
    out["dwg"], bound["dwg"] = product(dg.t(), edg.t(), x.t())
    out["dwu"], bound["dwu"] = product(du.t(), edu.t(), x.t())
    return out, bound


def check(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    e = rows(got.double() - want)
    tol = bound * (1 + half(got.dtype)) + half(got.dtype) * rows(want) + \
        tiny(got.dtype) * want.shape[1] ** 0.5
    bad = ~(e <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist(), float((e / tol).max()))


def inputs(gpu, n, h, f, o, dtype, seed):
    r = torch.Generator(device=gpu).manual_seed(seed)
    new = lambda *s, std=1.0: (std * torch.randn(*s, device=gpu, generator=r)).to(dtype)
    return [new(n, h), new(f, h, std=1.5 / h ** 0.5), new(f, h, std=h ** -0.5),
            new(o, f, std=f ** -0.5) if o else None, new(n, o or f)]


def run(args, act):
    x, wg, wu, wd, dy = args
    leaf = [t.detach().requires_grad_() if t is not None else None for t in (x, wg, wu, wd)]
    y = (fused_gated_linear(*leaf[:3], activation=act) if wd is None
         else fused_gated_mlp(*leaf, activation=act))
    names = [k for k, t in zip(("dx", "dwg", "dwu", "dwd"), leaf) if t is not None]
    grads = torch.autograd.grad(y, [t for t in leaf if t is not None], dy)
    return dict(y=y.detach(), **dict(zip(names, grads)))


def run_and_check(args, act):
    got = run(args, act)
    want, bound = reference(*args[:4], act, args[4])
    for k, v in got.items():
        check(v, want[k], bound[k], k)
    with torch.no_grad():  # the form that keeps nothing
        x, wg, wu, wd, _ = args
        y = (fused_gated_linear(x, wg, wu, activation=act) if wd is None
             else fused_gated_mlp(x, wg, wu, wd, activation=act))
    check(y, want["y"], bound["y"], "y without gradients")
    return got


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("down", [True, False])
def test_activations(gpu, act, dtype, down):
    run_and_check(inputs(gpu, 200, 192, 320, 136 if down else 0, dtype, 1), act)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 33, 64, 65, 100, 127, 129, 255, 257, 511, 1000])
def test_rows(gpu, n):
    run_and_check(inputs(gpu, n, 256, 512, 256, BF, n), "silu")
    run_and_check(inputs(gpu, n, 128, 384, 0, F16, n + 1), "gelu_tanh")


@pytest.mark.parametrize("h,f,o", [(8, 8, 8), (64, 8, 72), (8, 1000, 16), (72, 264, 520),
                                   (520, 136, 264), (1032, 2056, 776), (4096, 512, 128),
                                   (128, 4104, 1000)])
@pytest.mark.parametrize("n", [3, 70, 300])
def test_sizes(gpu, n, h, f, o):
    run_and_check(inputs(gpu, n, h, f, o, BF, h), "silu")


@pytest.mark.parametrize("h,f,o", [(1, 1, 1), (37, 50, 21), (100, 257, 64), (64, 63, 7)])
@pytest.mark.parametrize("n", [1, 65, 130])
def test_odd_sizes(gpu, n, h, f, o):
    run_and_check(inputs(gpu, n, h, f, o, F16, h), "gelu")
    run_and_check(inputs(gpu, n, h, f, 0, BF, h), "silu")


@pytest.mark.parametrize("n,h,f", [(2048, 1024, 2816), (4100, 768, 2048), (24, 4096, 14336),
                                   (300, 4096, 14336)])
def test_large(gpu, n, h, f):
    run_and_check(inputs(gpu, n, h, f, h, BF, 5), "silu")
