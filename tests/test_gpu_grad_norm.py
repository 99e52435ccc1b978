"""Global gradient norm and clipping against float64 on the GPU.

Tolerances: the squares of one 16-byte vector (8 values at most) are summed in fp32, all
positive, so that sum is off by at most 8 * 2^-24 of itself, everything after it is double; the
square root halves that, and the fp32 result is rounded once: NORM = 5 * 2^-24. A clipped value
takes the norm's 4 * 2^-24, the factor's rounding and its own: 6 * 2^-24 in fp32, and for 16-bit
outputs half a step of theirs plus 5 * 2^-24.
"""
import math

import pytest
import torch

from helpers import BF, F16, F32, flat, same
from trainscale_amd import _lib, ops
from trainscale_amd.kernels import (clip_grad_norm_, clip_grads_with_norm_, clipped_grads,
                                    get_total_norm)

pytestmark = pytest.mark.gpu
NORM = 5 * 2.0 ** -24
SIZES = [1, 3, 7, 8, 9, 0, 255, 4096, 32768, 32769, 65537, 98309]


def out_tol(dtype):
    return 6 * 2.0 ** -24 if dtype == F32 else torch.finfo(dtype).eps / 2 + 5 * 2.0 ** -24


def norm64(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def make(gpu, sizes, dtypes, seed=0, std=1e-2, off=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        buf = torch.randn(n + off, device=gpu, generator=g) * std
        out.append(buf.to(dtypes[i % len(dtypes)])[off:])
    return out


def params_of(grads):
    ps = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros_like(g))
        p.grad = g
        ps.append(p)
    return ps


def check_clipped(got, ref, coef, what=""):
    want = ref.double() * coef
    bad = (got.double() - want).abs() > out_tol(got.dtype) * want.abs() + (
        torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps)
    assert not bad.any(), (what, int(bad.sum()))


@pytest.mark.parametrize("dtypes", [[F32], [BF], [F16], [F32, BF, F16]])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_norm(gpu, dtypes, off):
    ts = make(gpu, SIZES, dtypes, seed=off, off=off)
    n = get_total_norm(ts)
    want = norm64(ts)
    assert n.dtype == F32 and n.dim() == 0
    assert abs(float(n) - want) <= NORM * want
    assert same(n, get_total_norm(ts))  # the same sums every time


@pytest.mark.parametrize("count", [1, 128, 129, 300])
def test_many_tensors(gpu, count):
    ts = make(gpu, [(k * 37) % 5000 + 1 for k in range(count)], [BF, F32], seed=count)
    want = norm64(ts)
    assert abs(float(get_total_norm(ts)) - want) <= NORM * want
    out = [torch.empty(t.shape, device=gpu) for t in ts]
    n = clipped_grads(ts, 0.25, out)
    assert abs(float(n) - want) <= NORM * want
    for t, o in zip(ts, out):
        check_clipped(o, t, min(1.0, 0.25 / (want + 1e-6)))


def test_norm_formed_in_a_launch_of_its_own(gpu):
    # more partial sums than the scaling's workgroups add up themselves: full launches of 3 types
    per = 16 * 1024 * 2049
    ts = [torch.full((per // 4,), 1e-3, device=gpu),
          torch.full((per // 2,), 1e-3, device=gpu, dtype=BF),
          torch.full((per // 2 + 1,), 1e-3, device=gpu, dtype=F16)]
    want = math.sqrt(sum(t.numel() * float(t[0].double()) ** 2 for t in ts))
    n = clip_grad_norm_(params_of(ts), 1.0)
    assert abs(float(n) - want) <= NORM * want
    for t, v in zip(ts, (1e-3, BF, F16)):
        first = torch.tensor(1e-3, dtype=t.dtype).double()
        check_clipped(t[:1000].cpu(), first.expand(1000), 1.0 / (want + 1e-6))
        assert bool((t == t[0]).all())


@pytest.mark.parametrize("dtypes", [[F32], [BF], [F16], [BF, F32, F16]])
@pytest.mark.parametrize("off", [0, 1])
def test_clip_in_place(gpu, dtypes, off):
    ts = make(gpu, SIZES, dtypes, seed=3, std=1.0, off=off)
    ref = [t.clone() for t in ts]
    want = norm64(ref)
    ps = params_of(ts)
    versions = [t._version for t in ts]
    n = clip_grad_norm_(ps, 2.0)
    assert abs(float(n) - want) <= NORM * want
    for t, r, v in zip(ts, ref, versions):
        check_clipped(t, r, 2.0 / (want + 1e-6))
        assert t._version > v
    # below the limit the gradients keep their bits
    now = [t.clone() for t in ts]
    clip_grad_norm_(ps, 1e6)
    assert all(same(a, b) for a, b in zip(ts, now))


def test_norm_of_other_ranks(gpu):
    ts = make(gpu, SIZES, [BF, F32], seed=5)
    ref = [t.clone() for t in ts]
    clip_grads_with_norm_(params_of(ts), 1.0, torch.tensor([8.0], device=gpu, dtype=torch.float64))
    for t, r in zip(ts, ref):
        check_clipped(t, r, 1.0 / (8.0 + 1e-6))


def test_norm_is_one_of_the_values(gpu):
    t = make(gpu, [70001], [F32], seed=6)[0]
    t[4321] = 8.0
    ref = t.clone()
    clip_grads_with_norm_(params_of([t]), 1.0, t[4321])
    check_clipped(t, ref, 1.0 / (8.0 + 1e-6))


@pytest.mark.parametrize("value,dtype", [(1e30, F32), (3e38, BF), (1e-30, F32), (1e-42, F32),
                                         (1e-40, BF), (6e-8, F16), (65504.0, F16)])
def test_squares_beyond_fp32(gpu, value, dtype):
    t = torch.full((5003,), value, dtype=dtype, device=gpu)
    t[::3] *= -0.5
    t[1::7] = 0
    want = norm64([t])
    if want > torch.finfo(F32).max:
        assert float(get_total_norm([t])) == math.inf
        t = t[:1]
        want = norm64([t])
    got = float(get_total_norm([t]))
    assert abs(got - want) <= NORM * want + 2.0 ** -150
    out = torch.empty(t.shape, device=gpu)
    clipped_grads([t], 1.0, [out])
    check_clipped(out, t, min(1.0, 1.0 / (want + 1e-6)))


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n", [5003, 1 << 23])  # few partial sums, and a launch of their own
def test_norm_beyond_fp32(gpu, n, dtype):
    def fresh():
        t = torch.full((n,), 3e38, dtype=dtype, device=gpu)
        t[::3] *= -0.5
        t[7] = 1.0
        return t

    for kind in range(4):
        t = fresh()
        if kind == 0:
            n_got = clip_grad_norm_(params_of([t]), 1.0)
        elif kind == 1:
            t2, t = t, torch.full((n,), float("nan"), device=gpu)
            n_got = clipped_grads([t2], 1.0, [t])
        elif kind == 2:
            n_got = get_total_norm([t])
            clip_grads_with_norm_(params_of([t]), 1.0, n_got)
        else:
            with pytest.raises(RuntimeError, match="non-finite"):
                clip_grad_norm_(params_of([t]), 1.0, error_if_nonfinite=True)
            assert same(t, fresh())
            continue
        assert float(n_got) == math.inf
        assert not t.any(), kind  # x * (1 / inf), as torch's arithmetic has it


@pytest.mark.parametrize("n", [70001, (1 << 22) + 5])
def test_same_factor_on_every_path(gpu, n):
    for seed in range(4):
        src = make(gpu, [n, 333, n], [F32, BF, F16], seed=seed, std=1.0)
        one, two, three = [[t.clone() for t in src] for _ in range(3)]
        norm = clip_grad_norm_(params_of(one), 1.0)
        clip_grads_with_norm_(params_of(two), 1.0, norm)
        assert same(norm, clip_grad_norm_(params_of(three), 1.0, error_if_nonfinite=True))
        assert same(norm, get_total_norm(src))
        for a, b, c in zip(one, two, three):
            assert same(a, b) and same(a, c)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_nonfinite_as_torch(gpu, bad, dtype):
    ts = make(gpu, [100, 5001], [dtype], seed=1)
    ts[1][4321] = bad
    ours, theirs = params_of(ts), params_of([t.float().clone() for t in ts])
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_(ours, 1.0, error_if_nonfinite=True)
    assert torch.equal(ours[0].grad, ts[0])  # raised before anything was scaled
    n = clip_grad_norm_(ours, 1.0)
    # the elementwise arithmetic of torch's clipping
    coef = (1.0 / (torch.linalg.vector_norm(torch.cat([p.grad for p in theirs])) + 1e-6)).clamp(max=1)
    assert math.isnan(float(n)) if math.isnan(bad) else float(n) == math.inf
    for p, q in zip(ours, theirs):
        want = q.grad * coef
        assert torch.equal(p.grad.float().isnan(), want.isnan())
        assert torch.equal(p.grad.float().nan_to_num(), want.nan_to_num())


def test_layouts(gpu):
    g = torch.Generator(device=gpu).manual_seed(9)
    base = torch.randn(40, 60, device=gpu, generator=g)
    dense = torch.randn(8, 16, 5, device=gpu, generator=g).permute(2, 0, 1)
    strided = base[:, 10:33]
    ref = [dense.clone(), strided.clone()]
    keep = base.clone()
    want = norm64(ref)
    assert abs(float(get_total_norm([dense, strided])) - want) <= NORM * want
    ps = [torch.nn.Parameter(torch.zeros(t.shape, device=gpu)) for t in ref]
    for p, t in zip(ps, (dense, strided)):
        p.grad = t
    clip_grad_norm_(ps, 0.5)
    for t, r in zip((dense, strided), ref):
        check_clipped(t, r, 0.5 / (want + 1e-6))
    keep[:, 10:33] = base[:, 10:33]
    assert torch.equal(keep, base)  # the columns beside the slice
    out = [torch.empty(t.shape, device=gpu) for t in ref]
    n = norm64([dense, strided])
    clipped_grads([dense, strided], 0.1, out)
    for o, t in zip(out, (dense, strided)):
        check_clipped(o, t, 0.1 / (n + 1e-6))


@pytest.mark.parametrize("count", [2, 40, 200])
def test_strided_gradients_over_several_launches(gpu, count):
    # the copies of strided gradients are read by the last launches, while the first ones write
    # their partial sums
    def make_list():
        g = torch.Generator(device=gpu).manual_seed(count)
        ts = []
        for k in range(count):
            dtype = (F32, BF, F16)[k % 3]
            t = torch.randn(300 + k, 57, device=gpu, generator=g).to(dtype)
            ts.append(t[:, 5:40] if k % 4 else t)
        return ts

    ts = make_list()
    want = norm64(ts)
    for _ in range(3):
        assert abs(float(get_total_norm(ts)) - want) <= NORM * want
    ref = [t.clone() for t in ts]
    n = clip_grad_norm_(params_of(ts), 1.0, error_if_nonfinite=True)
    assert abs(float(n) - want) <= NORM * want
    for t, r in zip(ts, ref):
        check_clipped(t, r, 1.0 / (want + 1e-6))


def test_same_parameter_and_shared_memory(gpu):
    t = torch.full((1000,), 1.0, device=gpu)
    p = params_of([t])[0]
    n = clip_grad_norm_([p, p], 1.0)
    assert abs(float(n) - math.sqrt(1000)) <= NORM * math.sqrt(1000)
    check_clipped(t, torch.ones(1000, device=gpu), 1 / (math.sqrt(1000) + 1e-6))
    a, b = params_of([t[:600], t[500:]])
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_([a, b], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_grads_with_norm_(params_of([t[:1].expand(5)]), 1.0, torch.ones((), device=gpu))
    with pytest.raises(ValueError, match="share memory"):
        clipped_grads([t[:500], t[500:]], 1.0, [t[500:], t[:500]])
    with pytest.raises(ValueError, match="contiguous"):
        clipped_grads([t[:500]], 1.0, [torch.empty(1000, device=gpu)[::2]])
    with pytest.raises(TypeError, match="output dtype"):
        clipped_grads([t], 1.0, [torch.empty(1000, device=gpu, dtype=BF)])
    with pytest.raises(ValueError, match="output"):
        clipped_grads([t], 1.0, [torch.empty(999, device=gpu)])
    before = t.clone()
    n = clipped_grads([t], 0.25, [t])  # its own output
    check_clipped(t, before, 0.25 / (norm64([before]) + 1e-6))
    assert abs(float(get_total_norm([t, t])) - math.sqrt(2) * norm64([t])) <= 1e-6


@pytest.mark.parametrize("src,dst", [(F32, F32), (BF, BF), (F16, F16), (BF, F32), (F16, F32)])
@pytest.mark.parametrize("n", [1, 7, 9, 32768, 65543])
def test_stays_inside(gpu, src, dst, n):
    x = make(gpu, [n], [src], std=1.0, seed=n)[0]
    gx, go, gn = flat(n, src, gpu, x), flat(n, dst, gpu), flat(1, F32, gpu)
    want = norm64([x])
    lib = _lib.load()
    wsb = int(lib.ts_grad_norm_workspace_size(1))
    gw = flat(wsb, torch.uint8, gpu)
    li, lo = ops.HostList([gx.t]), ops.HostList([go.t])
    p, k, d, o, od = map(ops._host, (li.ptr, li.numel, li.code, lo.ptr, lo.code))
    _lib.check(lib.ts_grad_clip(p, o, k, d, od, 1, 0.5, gn.p, gw.p, wsb, _lib.stream_handle(gpu)),
               "clip")
    assert gx.intact() and go.intact() and gn.intact() and gw.intact()
    assert abs(float(gn.t) - want) <= NORM * want
    check_clipped(go.t.reshape(-1), x, min(1.0, 0.5 / (want + 1e-6)))
    gn2 = flat(1, F32, gpu)
    _lib.check(lib.ts_grad_norm(p, k, d, 1, gn2.p, gw.p, wsb, _lib.stream_handle(gpu)), "norm")
    assert same(gn2.t, gn.t) and gn2.intact() and gw.intact()
    _lib.check(lib.ts_grad_scale(p, o, k, d, od, 1, gn.p, 0.5, _lib.stream_handle(gpu)), "scale")
    assert go.intact()
    check_clipped(go.t.reshape(-1), x, min(1.0, 0.5 / (want + 1e-6)))


def test_other_stream_and_graph(gpu):
    ts = make(gpu, [5000, 70001, 3], [BF, F32], seed=2)
    fresh = [t.clone() for t in ts]
    ps = params_of(ts)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        n1 = clip_grad_norm_(ps, 0.5)
    torch.cuda.current_stream(gpu).wait_stream(side)
    torch.cuda.synchronize()
    eager = [t.clone() for t in ts]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n2 = clip_grad_norm_(ps, 0.5)
    for rep in range(4):
        for t, f in zip(ts, fresh):
            t.copy_(f * (1 + rep))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in ts]
        for t, f in zip(ts, fresh):
            t.copy_(f * (1 + rep))
        n3 = clip_grad_norm_(ps, 0.5)
        assert same(n2, n3)
        assert all(same(a, b) for a, b in zip(got, ts)), rep
        if rep == 0:
            assert same(n1, n3) and all(same(a, b) for a, b in zip(got, eager))


def test_strided_gradients_beside_one_another(gpu):
    buf = torch.randn(50, 90, device=gpu, generator=torch.Generator(device=gpu).manual_seed(4))
    keep = buf.clone()

    def parts(t):
        return [t[:, :30], t[:20, 30:77], t[20:, 30:77:2], t[20:, 31:77:2], t[:, 80:]]

    want = norm64(parts(keep))
    n = clip_grad_norm_(params_of(parts(buf)), 1.0)
    assert abs(float(n) - want) <= NORM * want
    for t, r in zip(parts(buf), parts(keep)):
        check_clipped(t, r, 1.0 / (want + 1e-6))
    assert same(buf[:, 77:80], keep[:, 77:80])
    now = buf.clone()
    for grads in ([buf, buf[:, :4]], [buf[:, :6], buf[:, 3:9]], [buf[:, :4]] * 2,
                  [buf.view(-1).as_strided((5, 5), (3, 1))]):
        for call in (lambda p: clip_grad_norm_(p, 1e-3),
                     lambda p: clip_grad_norm_(p, 1e-3, error_if_nonfinite=True),
                     lambda p: clip_grads_with_norm_(p, 1e-3, torch.ones((), device=gpu))):
            with pytest.raises(ValueError, match="share memory"):
                call(params_of(grads))
    assert same(buf, now)
