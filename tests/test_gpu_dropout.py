"""Counter-based dropout against float64 on the GPU, alone, with the residual sum and with the norm.

Tolerances, with u = 2^-24 and half a step of the type for every rounded result. D(x) is one product
with a scale rounded to fp32 (2 u), h adds a sum (u): 3 u M, M = |residual| + |D(x)|. A row's sum of
squares has at most 32 products of a lane, 6 steps inside a wave and 8 waves: with the division and
the root, rstd is off by (27 + 3 k) u, k = |M| / |h| in 2-norms being what cancels in h. y is a
product of three such factors: (40 + 4 k) u M rstd |w|. The backward reads the rounded h, so hat is
off by eh = (half + (32 + 6 k) u) M rstd; its row mean c1 by mean |e| (eh + 50 u M rstd); t and dw as
these propagate. dw adds a row for each step of a workgroup, its row slots, 32 partial rows a slice
and 32 slices: (rows / 512 + 120) u of its magnitudes.
"""
import contextlib
import copy

import pytest
import torch

from helpers import BF, F16, F32, Guarded, same, saved_elsewhere
from philox import keep_mask
from trainscale_amd.kernels import (FusedDropoutAddRMSNorm, fused_dropout, fused_dropout_add,
                                    fused_dropout_add_rms_layernorm, fused_add_rms_layernorm)

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6
RNG = (0x123456789ABCDEF, 42)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def mask_of(shape, p, gpu, rng=RNG):
    cols = shape[-1]
    rows = 1
    for n in shape[:-1]:
        rows *= n
    return torch.from_numpy(keep_mask(rows, cols, *rng, p)).view(shape).to(gpu)


def check(got, want, bound, what):
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    tol = bound * (1 + half(got.dtype)) + half(got.dtype) * want.abs() + tiny
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:3].tolist())


def inputs(gpu, shape, dtype, wdtype, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=gpu, generator=g)
    return [(0.7 * r(*shape)).to(dtype), (2 * r(*shape)).to(dtype),
            (1 + 0.1 * r(shape[-1])).to(wdtype), r(*shape).to(dtype), r(*shape).to(dtype)]


def scale_of(p):
    drop = round(p * 65536)
    return 0.0 if drop == 65536 else 65536 / (65536 - drop)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 1), (5, 13), (4, 64), (129, 72),
                                   (2, 3, 1000), (33, 4100), (1, 100003)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_plain_and_add(gpu, shape, dtype, p):
    x, res, _, dy, _ = inputs(gpu, shape, dtype, dtype, len(shape))
    keep, s = mask_of(shape, p, gpu), scale_of(p)
    D = lambda t: torch.where(keep, t.double() * s, 0.0)
    x.requires_grad_(), res.requires_grad_()
    y = fused_dropout(x, p, rng=RNG)
    (dx,) = torch.autograd.grad(y, x, dy)
    check(y.detach(), D(x.detach()), 2 * U * D(x.detach()).abs(), "y")
    check(dx, D(dy), 2 * U * D(dy).abs(), "dx")
    assert not y[~keep].any() and not dx[~keep].any()
    h = fused_dropout_add(x, res, p, rng=RNG)
    dx2, dres = torch.autograd.grad(h, (x, res), dy)
    M = D(x.detach()).abs() + res.detach().double().abs()
    check(h.detach(), res.detach().double() + D(x.detach()), 3 * U * M, "h")
    assert same(dx2, dx) and same(dres, dy)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -17, 2.0 ** -16, 0.25, 0.9, 1 - 2.0 ** -16, 1.0])
def test_probabilities(gpu, p):
    x = torch.full((40, 520), 3.0, device=gpu)
    x[3, 7] = float("nan")
    y = fused_dropout(x, p, rng=RNG)
    keep = mask_of(x.shape, p, gpu)
    want = torch.where(keep, x.double() * scale_of(p), 0.0)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    check(y.nan_to_num(), want.nan_to_num(), 2 * U * want.nan_to_num().abs(), "y")
    assert same(fused_dropout(x, p, rng=RNG, training=False), x)


def reference(x, res, w, p, dy, dh):
    """Results of the norm in float64 and their bounds before the last rounding."""
    d, hf = torch.float64, half(x.dtype)
    shape, cols = x.shape, x.shape[-1]
    keep, s = mask_of(shape, p, x.device), scale_of(p)
    D = lambda t: torch.where(keep, t * s, 0.0)
    X, R, W = x.detach().to(d), res.detach().to(d), w.detach().to(d)
    h, M = R + D(X), R.abs() + D(X).abs()
    rh = 1 / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
    k = M.norm(dim=-1, keepdim=True) / h.norm(dim=-1, keepdim=True).clamp(min=1e-30)
    hat, Mr = h * rh, M * rh
    out = dict(h=h, y=hat * W)
    bound = dict(h=3 * U * M, y=(40 + 4 * k) * U * Mr * W.abs())
    DY = torch.zeros_like(h) if dy is None else dy.to(d)
    DH = torch.zeros_like(h) if dh is None else dh.to(d)
    e = DY * W
    c1 = (e * hat).mean(-1, keepdim=True)
    t = DH + rh * (e - hat * c1)
    eh = (hf + (32 + 6 * k) * U) * Mr
    ec = (e.abs() * (eh + 50 * U * Mr)).mean(-1, keepdim=True)
    C1 = (e.abs() * Mr).mean(-1, keepdim=True)
    et = rh * (eh * (c1.abs() + ec) + Mr * ec) + (40 + 4 * k) * U * rh * (e.abs() + Mr * C1) \
        + 2 * U * (DH.abs() + rh * (e.abs() + Mr * C1))
    rows = h.numel() // cols
    out.update(dres=t, dx=D(t), dw=(DY * hat).reshape(-1, cols).sum(0))
    bound.update(dres=et, dx=D(et) * (1 + U) + 2 * U * D(t).abs(),
                 dw=(DY.abs() * (eh + (rows / 512 + 120) * U * Mr)).reshape(-1, cols).sum(0))
    return out, bound


def run(args, p, rng=RNG, use=(True, True)):
    x, res, w, dy, dh = args
    leaf = [t.detach().requires_grad_() for t in (x, res, w)]
    y, h = fused_dropout_add_rms_layernorm(*leaf, p, EPS, rng=rng)
    outs = [t for t, k in zip((y, h), use) if k]
    ups = [t for t, k in zip((dy, dh), use) if k]
    grads = torch.autograd.grad(outs, leaf, ups)
    return dict(y=y.detach(), h=h.detach(), dx=grads[0], dres=grads[1], dw=grads[2])


def run_and_check(args, p, use=(True, True)):
    got = run(args, p, RNG, use)
    want, bound = reference(*args[:3], p, args[3] if use[0] else None, args[4] if use[1] else None)
    for k, v in got.items():
        check(v, want[k], bound[k], k)
    return got


WIDTHS = [1, 5, 8, 64, 72, 250, 256, 512, 513, 1000, 1024, 2048, 2056, 4096, 4100, 8192, 16384]


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(gpu, width, dtype):
    run_and_check(inputs(gpu, (11, width), dtype, dtype, width), 0.1)
    run_and_check(inputs(gpu, (3, 7, width), dtype, F32, width + 1), 0.5)


@pytest.mark.parametrize("rows", [1, 2, 31, 33, 513, 3000])
@pytest.mark.parametrize("width", [64, 200, 264, 768, 1600])
def test_rows(gpu, rows, width):
    run_and_check(inputs(gpu, (rows, width), BF, BF, rows), 0.1)


@pytest.mark.parametrize("rows,width,dtype", [(16391, 2048, BF), (65601, 512, F16),
                                              (16400, 4090, BF), (16385, 1030, F32)])
def test_many_rows(gpu, rows, width, dtype):
    run_and_check(inputs(gpu, (rows, width), dtype, F32, rows), 0.1)


@pytest.mark.parametrize("use", [(True, False), (False, True)])
def test_one_result_used(gpu, use):
    run_and_check(inputs(gpu, (5, 9, 512), BF, F32, 5), 0.1, use)


def test_only_some_gradients(gpu):
    args = inputs(gpu, (3, 40, 256), F16, F16, 6)
    full = run(args, 0.2)
    for wanted in (("x",), ("res",), ("w",), ("x", "w")):
        t = {k: v.detach().clone().requires_grad_(k in wanted)
             for k, v in zip(("x", "res", "w"), args)}
        y, h = fused_dropout_add_rms_layernorm(t["x"], t["res"], t["w"], 0.2, EPS, rng=RNG)
        g = torch.autograd.grad((y, h), [t[k] for k in wanted], args[3:])
        assert all(same(a, full["d" + k]) for a, k in zip(g, wanted)), wanted


def test_against_differences(gpu):
    args = inputs(gpu, (6, 40), F32, F32, 7)
    x, res, w, dy, dh = args
    got = run(args, 0.3)
    _, bound = reference(x, res, w, 0.3, dy, dh)
    keep, s = mask_of(x.shape, 0.3, gpu), scale_of(0.3)

    def value(ts):
        h = ts[1] + torch.where(keep, ts[0] * s, 0.0)
        y = h / (h.square().mean(-1, keepdim=True) + EPS).sqrt() * ts[2]
        return float((y * dy).sum() + (h * dh).sum())

    base = [t.double() for t in (x, res, w)]
    g = torch.Generator(device=gpu).manual_seed(8)
    for i, name in enumerate(("dx", "dres", "dw")):
        dirn = torch.randn(base[i].shape, device=gpu, generator=g, dtype=torch.float64)
        step = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + step * dirn, base[i] - step * dirn
        diff = (value(up) - value(down)) / (2 * step)
        have = float((got[name].double() * dirn).sum())
        # the kernel's bound along the direction; the difference's own error is step^2 times a
        # third derivative of order 10 n over 240 terms, and 1e-16 / step of its values
        tol = float(((bound[name] + U * got[name].abs()) * dirn.abs()).sum()) + 1e-6
        assert abs(have - diff) <= tol, (name, have, diff, tol)


def test_without_dropout_the_norm_is_the_layers(gpu):
    x, res, w, _, _ = inputs(gpu, (50, 1024), F32, F32, 9)
    y, h = fused_dropout_add_rms_layernorm(x, res, w, 0.4, EPS, training=False)
    y2, h2 = fused_add_rms_layernorm(x, res, w, EPS, return_residual=True)
    assert same(h, h2)
    assert (y - y2).abs().max() <= 64 * U * y2.abs().max()


def test_layouts(gpu):
    args = inputs(gpu, (4, 50, 200), BF, BF, 10)
    ref = run(args, 0.1)

    def strided(t):  # unaligned rows inside a wider buffer of NaN
        w = torch.full((*t.shape[:-1], 211), float("nan"), dtype=t.dtype, device=gpu)
        w[..., 3:203] = t.detach()
        return w[..., 3:203]

    again = run([strided(t) for t in args[:2]] + [args[2]] + [strided(t) for t in args[3:]], 0.1)
    assert all(same(ref[k], again[k]) for k in ref)
    t = run([t.transpose(0, 1).contiguous().transpose(0, 1) for t in args[:2]] + args[2:], 0.1)
    assert all(same(ref[k].contiguous(), t[k].contiguous()) for k in ref)
    assert same(fused_dropout(strided(args[0]), 0.1, RNG), fused_dropout(args[0], 0.1, RNG))
    assert same(fused_dropout_add(strided(args[0]), strided(args[1]), 0.1, RNG), ref["h"])
    # upstream gradients without memory of their own
    x = args[0].detach().requires_grad_()
    (g,) = torch.autograd.grad(fused_dropout(x, 0.1, RNG).float().sum(), x)
    assert same(g, fused_dropout(torch.ones_like(x), 0.1, RNG))


def test_nothing_outside_is_touched(gpu):
    import ctypes
    from trainscale_amd import _lib
    lib, r = _lib.load(), ctypes.byref(_lib.DropoutRng(*RNG, 0, 6554))
    for dtype, cols in ((BF, 72), (F32, 71), (F16, 517)):
        code, g = _lib.DTYPE_CODE[dtype], torch.Generator(device=gpu).manual_seed(cols)
        rows, ld = 9, cols + 5
        val = [torch.randn(rows, cols, device=gpu, generator=g).to(dtype) for _ in range(4)]
        x, res, dy, dh = [Guarded(rows, cols, ld, dtype, gpu, v) for v in val]
        w = Guarded(1, cols, cols, dtype, gpu, torch.ones(cols, device=gpu).to(dtype))
        out = Guarded(rows, cols, ld, dtype, gpu)
        packed = [Guarded(rows, cols, cols, dtype, gpu) for _ in range(4)]  # y, h, dx, dres
        rstd = Guarded(1, rows, rows, F32, gpu)
        dw = Guarded(1, cols, cols, dtype, gpu)
        st = _lib.stream_handle(gpu)
        n = lib.ts_dropout_add_rmsnorm_bwd_workspace_size(rows, cols)
        ws = Guarded(1, n, n, torch.uint8, gpu)
        assert lib.ts_dropout_fwd(x.p, ld, res.p, ld, out.p, ld, code, rows, cols, r, st) == 0
        assert lib.ts_dropout_add_rmsnorm_fwd(x.p, ld, res.p, ld, code, w.p, code, packed[0].p,
                                              packed[1].p, rstd.p, rows, cols, EPS, r, st) == 0
        assert lib.ts_dropout_add_rmsnorm_bwd(dy.p, ld, dh.p, ld, packed[1].p, cols, code, w.p,
                                              code, rstd.p, packed[2].p, packed[3].p, dw.p, rows,
                                              cols, r, ws.p, n, st) == 0
        torch.cuda.synchronize()
        assert all(t.intact() for t in (x, res, dy, dh, w, out, rstd, dw, ws, *packed))
        got = run(val[:2] + [w.t[0]] + val[2:], 0.1)
        assert same(packed[0].t, got["y"]) and same(packed[2].t, got["dx"])
        assert same(out.t, got["h"]) and same(dw.t[0], got["dw"])


def test_numbers_from_a_tensor(gpu):
    args = inputs(gpu, (30, 264), BF, BF, 11)
    state = torch.tensor([RNG[0], RNG[1]], device=gpu)
    by_value, by_tensor = run(args, 0.1), run(args, 0.1, state)
    assert all(same(by_value[k], by_tensor[k]) for k in by_value)
    x = args[0].detach().requires_grad_()
    y = fused_dropout(x, 0.1, state)
    state.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, x, args[3])
    # as signed 64-bit values
    big = (2 ** 64 - 5, 2 ** 63 + 9)
    s = torch.tensor([-5, 9 - 2 ** 63], device=gpu)
    assert same(fused_dropout(x.detach(), 0.1, big), fused_dropout(x.detach(), 0.1, s))


def test_numbers_from_torch(gpu):
    x = torch.ones(50, 1000, device=gpu)
    torch.manual_seed(3)
    a, b = fused_dropout(x, 0.5), fused_dropout(x, 0.5)
    torch.manual_seed(3)
    assert same(a, fused_dropout(x, 0.5)) and not same(a, b)
    # 50000 draws of probability 1/2: within 5 standard errors
    assert abs(float((a == 0).float().mean()) - 0.5) < 5 * 0.5 / 50000 ** 0.5


def test_module_streams_and_hooks(gpu):
    m = FusedDropoutAddRMSNorm(256, 0.1, dtype=BF).to(gpu)
    x, res, _, dy, dh = inputs(gpu, (20, 256), BF, BF, 12)
    with torch.no_grad():
        m.weight.copy_(1 + 0.1 * torch.randn(256, device=gpu))
    ref = run([x, res, m.weight, dy, dh], 0.1)
    for ctx in (contextlib.nullcontext(), saved_elsewhere()):
        leaf = [x.detach().requires_grad_(), res.detach().requires_grad_()]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s), ctx:
            y, h = m(*leaf, rng=RNG)
            g = torch.autograd.grad((y, h), [*leaf, m.weight], (dy, dh))
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert same(y, ref["y"]) and same(h, ref["h"])
        assert all(same(a, ref[k]) for a, k in zip(g, ("dx", "dres", "dw")))
    m.eval()
    y, h = m(x, res, rng=RNG)
    assert same(h, (x.float() + res.float()).to(BF))


def test_empty(gpu):
    x = torch.empty(0, 64, device=gpu, requires_grad=True)
    w = torch.ones(64, device=gpu, requires_grad=True)
    y, h = fused_dropout_add_rms_layernorm(x, x.detach(), w, 0.1)
    gx, gw = torch.autograd.grad((y, h), (x, w), (torch.empty(0, 64, device=gpu),) * 2)
    assert y.shape == gx.shape == (0, 64) and not gw.any()
    assert fused_dropout(torch.empty(3, 0, device=gpu), 0.5).shape == (3, 0)
    assert fused_dropout(torch.ones((), device=gpu), 0.5, RNG).shape == ()


def test_graph(gpu):
    x, res, w, dy, dh = inputs(gpu, (64, 512), BF, BF, 13)
    state = torch.tensor([7, 0], device=gpu)
    leaf = [t.requires_grad_() for t in (x, res, w)]

    def step():
        y, h = fused_dropout_add_rms_layernorm(*leaf, 0.1, EPS, rng=state)
        return (y, h, *torch.autograd.grad((y, h), leaf, (dy, dh)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        state[1:].add_(1)
        with pytest.raises(RuntimeError, match="captured graph"):
            fused_dropout(dy, 0.1)
    seen = []
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = run([x, res, w, dy, dh], 0.1, rng=(7, i))
        torch.cuda.synchronize()
        assert all(same(a, want[k]) for a, k in zip(out, ("y", "h", "dx", "dres", "dw"))), i
        seen.append(out[1].detach().clone())
    assert not same(seen[0], seen[1])


def test_far_elements(gpu):
    """Elements past 2^32 in a tensor, whose counters pass 2^29."""
    rows, cols = (1 << 32) // 4096 + 3, 4096
    x = torch.ones(rows, cols, dtype=BF, device=gpu)
    y = fused_dropout(x, 0.5, RNG)
    from philox import philox
    import numpy as np
    n = np.arange((rows - 2) * 512, rows * 512, dtype=np.uint64)
    words = philox([n & np.uint64(2 ** 32 - 1), n >> np.uint64(32), np.full_like(n, RNG[1]),
                    np.zeros_like(n)], (RNG[0] % 2 ** 32, RNG[0] >> 32))
    bits = np.stack([v >> np.uint64(s) & np.uint64(0xFFFF) for v in words for s in (0, 16)], -1)
    keep = torch.from_numpy((bits.reshape(2, cols) >= 32768)).to(gpu)
    assert torch.equal(y[-2:] != 0, keep)


def test_far_rows_of_the_norm(gpu):
    """Elements past 2^32: the sum as the operator without the norm forms it (whose far mask the test
    above holds to the generator), the last rows' norm and gradients by their formulas."""
    rows, cols, p = (1 << 32) // 4096 + 40, 4096, 0.25
    x = torch.full((rows, cols), 0.5, dtype=BF, device=gpu).requires_grad_()
    res = torch.zeros(rows, cols, dtype=BF, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(3)
    res[-32:] = torch.randn(32, cols, device=gpu, generator=g).to(BF)
    w = torch.ones(cols, device=gpu, requires_grad=True)
    y, h = fused_dropout_add_rms_layernorm(x, res.requires_grad_(), w, p, EPS, rng=RNG)
    plain = fused_dropout_add(x.detach(), res.detach(), p, RNG)
    assert torch.equal(h.detach(), plain)
    keep = (plain - res.detach() != 0)[-32:]
    del plain
    dy = torch.zeros_like(y)
    dy[-32:] = torch.randn(32, cols, device=gpu, generator=g).to(BF)
    dx, dres, dw = torch.autograd.grad(y, (x, res, w), dy)
    assert not dx[:-32].any() and not dres[:-32].any()
    X, R, DY = [t[-32:].detach().double() for t in (x, res, dy)]
    H = R + torch.where(keep, X * scale_of(p), 0.0)
    rh = 1 / (H.square().mean(-1, keepdim=True) + EPS).sqrt()
    k, M = (H - R).abs() + R.abs(), half(BF)
    check(y[-32:].detach(), H * rh, 60 * U * k * rh, "y")
    # the backward's hat comes from the rounded h: off by half a step of it
    hat = H * rh
    c1 = (DY * hat).mean(-1, keepdim=True)
    t = rh * (DY - hat * c1)
    eh = (M + 60 * U) * k * rh
    ec = (DY.abs() * (eh + 50 * U * hat.abs())).mean(-1, keepdim=True)
    et = rh * (eh * (c1.abs() + ec) + hat.abs() * ec) + 60 * U * rh * (DY.abs() + k * rh * c1.abs())
    check(dres[-32:], t, et, "dres")
    check(dx[-32:], torch.where(keep, t * scale_of(p), 0.0), et * scale_of(p) * (1 + U)
          + 2 * U * t.abs() * scale_of(p), "dx")
    check(dw, (DY * hat).sum(0), (DY.abs() * (eh + 220 * U * k * rh)).sum(0), "dw")


def test_far_rows_apart(gpu):
    """The same of rows with gaps, whose place is divided out of the group's number."""
    x = torch.ones((1 << 32) // 4088 + 9, 4096, dtype=BF, device=gpu)[:, :4088]
    assert x.numel() > 1 << 32
    assert torch.equal(fused_dropout(x, 0.5, RNG), fused_dropout(x.contiguous(), 0.5, RNG))
