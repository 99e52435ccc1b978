"""The gated feed-forward block against float64 on the GPU, forward and every gradient.

Tolerances hold for each row of a result, in 2-norms. With u = 2^-24 and h half a step of the data
type: an fp32 sum of K exact products is off by at most K u times the sum of magnitudes. An
activation t of g is off by at most 24 u |g| (the argument of its exponential carries at most 4
roundings, which move t by at most 8 u |g|; the exponential, reciprocal or erfc and two products
add 16 u |t|, and |t| <= |g|), its derivative by 16 u (1 + |g|); |act'| <= 1.2 and |act''| <= 1
carry the error of g on (relu: its derivative is off by 1 where the sign of g is in doubt). The
gated product, dg and du are rounded to the data type once; what the backward keeps is fp32. Products
of matrices carry errors on as |E B|_2 <= |E|_2 times B's spectral norm. Results add h of
themselves.
"""
import contextlib
import copy
import ctypes

import pytest
import torch

from helpers import BF, F16, F32, Guarded, saved_elsewhere, same
from trainscale_amd import _lib
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


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 32, 33, 48, 49, 64, 65, 100, 127, 129, 255, 257, 511, 1000])
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


@pytest.mark.parametrize("n", [16, 17, 31, 32, 33, 48, 49, 64])
@pytest.mark.parametrize("h,f,o", [(72, 4104, 4120), (512, 5000, 7000), (4136, 8192, 4096),
                                   (96, 9216, 9224)])
def test_few_rows_of_many_features(gpu, n, h, f, o):
    run_and_check(inputs(gpu, n, h, f, o, BF, n), "silu")


@pytest.mark.parametrize("n,h,f", [(2048, 1024, 2816), (4100, 768, 2048), (24, 4096, 14336),
                                   (300, 4096, 14336)])
def test_large(gpu, n, h, f):
    run_and_check(inputs(gpu, n, h, f, h, BF, 5), "silu")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype,values", [
    (BF, [0.0, 1e-30, 1e-3, 0.3, 1.0, 5.0, 12.0, 30.0, 89.0, 200.0, 1e4, 1e15]),
    (F16, [0.0, 6e-8, 1e-3, 0.3, 1.0, 5.0, 12.0, 30.0, 89.0, 200.0])])
def test_far_activations(gpu, act, dtype, values):
    """A value of g a row, of either sign, alone in its sums."""
    v = torch.tensor(values + [-t for t in values], device=gpu)
    x = torch.zeros(len(v), 8, device=gpu)
    x[:, 0], x[:, 1] = v, 1.5
    wg, wu = torch.zeros(16, 8, device=gpu), torch.zeros(16, 8, device=gpu)
    wg[:, 0], wu[:, 1] = 1, 1
    got = run_and_check([t.to(dtype) for t in (x, wg, wu)] + [None, torch.ones(
        len(v), 16, dtype=dtype, device=gpu)], act)
    assert all(torch.isfinite(t).all() for t in got.values())


def test_largest_values(gpu):
    top = torch.finfo(BF).max
    x = torch.tensor([[top, 1] + [0] * 6, [-top, 1] + [0] * 6], dtype=BF, device=gpu)
    w = torch.eye(8, dtype=BF, device=gpu)
    gate, up = w[:1].expand(8, 8).contiguous(), w[1:2].expand(8, 8).contiguous()
    for act in ACTS:
        y = fused_gated_linear(x, gate, up, act)
        assert (y[0] == top).all() and not y[1].any(), act


@pytest.mark.parametrize("n", [20, 200])
@pytest.mark.parametrize("act", ACTS)
def test_nan_stays_in_its_row(gpu, act, n):
    args = inputs(gpu, n, 64, 128, 72, BF, 7)
    args[0][5], args[0][11] = 0, 0
    ref = run(args, act)
    args[0][5], args[0][11, 3] = float("nan"), float("inf")
    got = run(args, act)
    rest = [i for i in range(n) if i not in (5, 11)]
    for k in ("y", "dx"):
        assert same(got[k][rest], ref[k][rest]), k
        assert got[k][5].isnan().all() and not got[k][11].isfinite().any(), k
    assert got["dwg"].isnan().all() and got["dwd"].isnan().all()


def test_layouts(gpu):
    args = inputs(gpu, 90, 72, 136, 40, BF, 3)
    ref = run(args, "silu")

    def inside(t, left, right):  # rows inside wider ones of NaN
        w = torch.full((t.shape[0], t.shape[1] + left + right), float("nan"), dtype=t.dtype,
                       device=gpu)
        w[:, left:left + t.shape[1]] = t
        return w[:, left:left + t.shape[1]]

    for change in (lambda t: inside(t, 8, 16), lambda t: inside(t, 3, 1), lambda t: inside(t, 4, 4),
                   lambda t: t.t().contiguous().t(),
                   lambda t: torch.stack((t, t * float("nan")), -1)[..., 0]):
        again = run([change(t) for t in args], "silu")
        assert all(same(ref[k], again[k].contiguous()) for k in ref)
    x = args[0].view(2, 45, 72).transpose(0, 1)
    y = fused_gated_mlp(x, *args[1:4])
    assert y.shape == (45, 2, 40) and same(y.transpose(0, 1).reshape(90, 40), ref["y"])
    # an upstream gradient without memory of its own
    leaf = args[0].detach().requires_grad_()
    (g,) = torch.autograd.grad(fused_gated_mlp(leaf, *args[1:4]).sum(), leaf)
    assert same(g, run(args[:4] + [torch.ones_like(args[4])], "silu")["dx"])
    row = args[0][:1].detach().requires_grad_()  # a row broadcast: its gradients are added
    (g,) = torch.autograd.grad(fused_gated_mlp(row.expand(90, 72), *args[1:4]), row, args[4])
    many = run([args[0][:1].repeat(90, 1)] + args[1:], "silu")["dx"]
    assert same(g, many.sum(0, keepdim=True))


def test_one_weight_for_both_projections(gpu):
    x, wg, _, wd, dy = inputs(gpu, 70, 64, 96, 64, BF, 4)
    ref = run([x, wg, wg.clone(), wd, dy], "silu")
    w = wg.detach().requires_grad_()
    (g,) = torch.autograd.grad(fused_gated_mlp(x, w, w, wd), w, dy)
    assert same(g, ref["dwg"] + ref["dwu"])


@pytest.mark.parametrize("n,down", [(20, True), (300, True), (300, False)])
def test_only_some_gradients(gpu, n, down):
    args = inputs(gpu, n, 136, 264, 72 if down else 0, BF, 6)
    ref = run(args, "gelu")
    assert all(same(v, w) for v, w in zip(ref.values(), run(args, "gelu").values()))
    names = ("dx", "dwg", "dwu", "dwd")
    for wanted in range(1, 16 if down else 8):
        leaf = [t.detach().requires_grad_(bool(wanted >> i & 1)) if t is not None else None
                for i, t in enumerate(args[:4])]
        y = (fused_gated_mlp(*leaf, activation="gelu") if down
             else fused_gated_linear(*leaf[:3], activation="gelu"))
        need = [t for t in leaf if t is not None and t.requires_grad]
        got = torch.autograd.grad(y, need, args[4])
        assert all(same(a, ref[names[i]]) for a, i in zip(
            got, [i for i in range(4) if wanted >> i & 1]))


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_against_differences(gpu, act):
    args = inputs(gpu, 40, 64, 72, 56, F16, 8)
    got = run(args, act)
    _, bound = reference(*args[:4], act, args[4])
    exact = [t.double() for t in args]

    def loss(x, wg, wu, wd):
        return float(((act64(act, x @ wg.t()) * (x @ wu.t()) @ wd.t()) * exact[4]).sum())

    r, step = torch.Generator(device=gpu).manual_seed(9), 1e-4
    for i, name in enumerate(("dx", "dwg", "dwu", "dwd")):
        d = torch.randn(args[i].shape, device=gpu, generator=r, dtype=torch.float64)
        d /= d.norm()
        at = lambda s: loss(*[t + s * d if j == i else t for j, t in enumerate(exact[:4])])
        diff = (at(step) - at(-step)) / (2 * step)
        g = got[name].double()
        # Cauchy-Schwarz over the rows' bounds; the difference is off by step^2 / 6 times a third
        # derivative of at most 10 for each of 40 x 56 terms
        tol = float(((bound[name] + 2 * half(F16) * rows(g)) * rows(d)).sum()) + 1e-4
        assert abs(float((g * d).sum()) - diff) <= tol, name


@pytest.mark.parametrize("n", [24, 200])
def test_nothing_outside_is_touched(gpu, n):
    lib, (h, f, o) = _lib.load(), (72, 136, 40)
    val = inputs(gpu, n, h, f, o, BF, n)
    x, wg, wu, wd, dy = [Guarded(*t.shape, t.shape[1] + 8, BF, gpu, t) for t in val]
    keep = [Guarded(n, f, f, F32, gpu) for _ in range(2)]
    act, out = Guarded(n, f, f, BF, gpu), Guarded(n, o, o, BF, gpu)
    grads = [Guarded(*t.shape, t.shape[1], BF, gpu) for t in val[:4]]
    a = _lib.GatedMLPArgs(x.p.value, x.ld, wg.p.value, wg.ld, wu.p.value, wu.ld, wd.p.value, wd.ld,
                          n, h, f, o, 0, _lib.TS_BF16)
    sizes = (lib.ts_gated_mlp_fwd_workspace_size(n, h, f, o),
             lib.ts_gated_mlp_bwd_workspace_size(n, h, f, o))
    ws = [Guarded(1, max(s, 16), max(s, 16), torch.uint8, gpu) for s in sizes]
    st = _lib.stream_handle(gpu)
    assert lib.ts_gated_mlp_fwd(ctypes.byref(a), keep[0].p, keep[1].p, act.p, out.p, ws[0].p,
                                sizes[0], st) == 0, _lib.last_error()
    assert lib.ts_gated_mlp_bwd(ctypes.byref(a), keep[0].p, keep[1].p, act.p, dy.p, dy.ld,
                                *[t.p for t in grads], ws[1].p, sizes[1], st) == 0
    torch.cuda.synchronize()
    assert all(t.intact() for t in (x, wg, wu, wd, dy, act, out, *keep, *grads, *ws))
    got = run(val, "silu")
    for t, k in zip((out, *grads), ("y", "dx", "dwg", "dwu", "dwd")):
        assert same(t.t, got[k]), k


@pytest.mark.parametrize("dtype", [BF, F16])
def test_pad(gpu, dtype):
    """Copies in one launch: of rows, of columns, of neither dense, of one repeated, of none."""
    lib, r = _lib.load(), torch.Generator(device=gpu).manual_seed(1)
    base = torch.randn(400, 401, device=gpu, generator=r).to(dtype)
    views = [base[:67, 1:130], base[3:132, :5].t(), base[::3, ::2], base[:1].expand(70, 401),
             base[:0, :8], base[5:6, 7:8], base[:65, :64].t(), base[2:66, 8:72]]
    sizes = [(67, 136), (8, 136), (134, 201), (72, 408), (3, 8), (1, 1), (64, 65), (64, 64)]
    outs = [Guarded(*s, s[1], dtype, gpu) for s in sizes]
    jobs = [_lib.PadJob(v.data_ptr(), *v.stride(), *v.shape, o.p, *s)
            for v, o, s in zip(views, outs, sizes)]
    assert lib.ts_pad_matrices((_lib.PadJob * 8)(*jobs), 8, _lib.DTYPE_CODE[dtype],
                               _lib.stream_handle(gpu)) == 0, _lib.last_error()
    for v, o, s in zip(views, outs, sizes):
        want = torch.nn.functional.pad(v, (0, s[1] - v.shape[1], 0, s[0] - v.shape[0]))
        assert o.intact() and same(o.t, want), s


def test_empty(gpu):
    _, wg, wu, wd, _ = inputs(gpu, 1, 16, 24, 8, BF, 1)
    leaf = [torch.empty(3, 0, 16, dtype=BF, device=gpu).requires_grad_()] + [
        t.requires_grad_() for t in (wg, wu, wd)]
    y = fused_gated_mlp(*leaf)
    assert y.shape == (3, 0, 8)
    for g, t in zip(torch.autograd.grad(y, leaf, torch.empty_like(y)), leaf):
        assert g.shape == t.shape and not g.any()
    assert fused_gated_linear(leaf[0], wg, wu).shape == (3, 0, 24)
    assert fused_gated_linear(torch.ones(16, dtype=BF, device=gpu), wg, wu).shape == (24,)


def test_module_streams_and_hooks(gpu):
    m = FusedGatedMLP(72, 200, "gelu_tanh", dtype=F16, device=gpu)
    x, _, _, _, dy = inputs(gpu, 130, 72, 200, 72, F16, 5)
    weights = [m.gate_proj.weight, m.up_proj.weight, m.down_proj.weight]
    ref = run([x, *weights, dy], "gelu_tanh")
    for ctx in (contextlib.nullcontext(), saved_elsewhere()):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        leaf = x.detach().requires_grad_()
        with torch.cuda.stream(s), ctx:
            y = m(leaf)
            g = torch.autograd.grad(y, [leaf, *weights], dy)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert same(y.detach(), ref["y"])
        assert all(same(a, ref[k]) for a, k in zip(g, ("dx", "dwg", "dwu", "dwd")))
    other = copy.deepcopy(m)
    assert same(other(x).detach(), ref["y"])
    assert str(m).startswith("FusedGatedMLP(\n  72, 200, activation='gelu_tanh'")


def test_graphs(gpu):
    """Two captured graphs, of few rows and of many with K slots, replayed in turn."""
    sets = [inputs(gpu, n, 520, 1032, 264, BF, n) for n in (9, 260)]
    leaves = [[t.requires_grad_() for t in args[:4]] for args in sets]

    def step(i):
        y = fused_gated_mlp(*leaves[i])
        return (y, *torch.autograd.grad(y, leaves[i], sets[i][4]))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for i in range(2):
            step(i)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(step(i))
    for rep in range(4):
        for i in range(2):
            with torch.no_grad():
                sets[i][0].mul_(-1.25)
                sets[i][4].mul_(1.5)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = run(sets[i], "silu")
            assert all(same(a.detach(), b) for a, b in zip(outs[i], want.values())), (rep, i)


def test_far_elements(gpu):
    """More than 2^32 features in all; gradients of the first and last rows alone."""
    n, h, f = 66000, 8, 1 << 16
    x, wg, wu, _, _ = inputs(gpu, n, h, f, 0, BF, 2)
    ends = list(range(32)) + list(range(n - 32, n))
    dy = torch.zeros(n, f, dtype=BF, device=gpu)
    dy[ends] = torch.randn(64, f, device=gpu).to(BF)
    got = run([x, wg, wu, None, dy], "silu")
    want, bound = reference(x[ends], wg, wu, None, "silu", dy[ends])
    for k in ("y", "dx"):
        check(got[k][ends], want[k], bound[k], k)
    assert not got["dx"][32:-32].any()
    for k in ("dwg", "dwu"):  # the other rows add exact zeros
        check(got[k], want[k], bound[k], k)


@pytest.mark.parametrize("down", [True, False])
def test_keeps_what_the_gradients_read(gpu, down):
    """The fp32 factors are kept for gradients of x, gate and up, the gated product for down's."""
    n, h, f = 200, 64, 136
    args = inputs(gpu, n, h, f, 72 if down else 0, BF, 6)
    ref = run(args, "silu")
    given = {t.data_ptr() for t in args[:4] if t is not None}
    for wanted in range(1, 16 if down else 8):
        leaf = [t.detach().requires_grad_(bool(wanted >> i & 1)) if t is not None else None
                for i, t in enumerate(args[:4])]
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
            y = (fused_gated_mlp(*leaf) if down else fused_gated_linear(*leaf[:3]))
        new = [t for t in kept if t.data_ptr() not in given]
        assert sum(t.numel() * t.element_size() for t in new) == \
            (8 * n * f if wanted & 7 else 0) + (2 * n * f if wanted & 8 else 0), wanted
        need = [i for i in range(4) if wanted >> i & 1]
        for g, i in zip(torch.autograd.grad(y, [leaf[i] for i in need], args[4]), need):
            assert same(g, ref[("dx", "dwg", "dwu", "dwd")[i]]), (wanted, i)


@pytest.mark.parametrize("wanted", [1, 6, 8, 9, 14])
@pytest.mark.parametrize("n,h,f,o", [(256, 2048, 5632, 2048), (1000, 768, 2048, 264),
                                     (2045, 768, 2048, 768), (130, 4096, 1032, 8)])
def test_plans_of_some_gradients(gpu, n, h, f, o, wanted):
    """Frozen operands: the others' gradients, on tiles and K slots of their own."""
    args = inputs(gpu, n, h, f, o, BF, n)
    want, bound = reference(*args[:4], "silu", args[4])
    leaf = [t.detach().requires_grad_(bool(wanted >> i & 1)) for i, t in enumerate(args[:4])]
    names = [k for i, k in enumerate(("dx", "dwg", "dwu", "dwd")) if wanted >> i & 1]
    need = [t for t in leaf if t.requires_grad]
    runs = [torch.autograd.grad(fused_gated_mlp(*leaf), need, args[4]) for _ in range(2)]
    for k, g, again in zip(names, *runs):
        check(g, want[k], bound[k], k)
        assert same(g, again), k
