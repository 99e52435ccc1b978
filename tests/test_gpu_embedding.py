"""Embedding forward and gradient against float64 on the GPU.

Tolerances: the forward is one fp32 product rounded once more (fp32: 2^-24; 16-bit: half a step
plus 2^-24). A gradient row of n tokens is an fp32 sum; its additions run through at most
DEPTH = 2 * 31 tokens, 2 * 63 chunk sums, n / 256 sums of sums and the 2 * 31 additions inside
those, so it is off by at most (DEPTH + n / 256) 2^-24 times the sum of the magnitudes, plus the
rounding of the scale's product (2^-24) and of the result.
"""
import pytest
import torch

from helpers import BF, F16, F32, Guarded, flat, same, saved_elsewhere
from trainscale_amd import _lib
from trainscale_amd.kernels import ScaledEmbedding, scaled_embedding

pytestmark = pytest.mark.gpu
DEPTH = 2 * 31 + 2 * 63 + 2 * 31


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def grad64(ids, dout, rows, scale, padding=None):
    """(gradient, sum of magnitudes, tokens) of every row in float64."""
    keep = (ids >= 0) & (ids < rows)
    if padding is not None:
        keep &= ids != padding
    ids, dout = ids[keep], dout[keep].double()
    z = torch.zeros(rows, dout.shape[1], dtype=torch.float64, device=dout.device)
    return (scale * z.index_add(0, ids, dout), abs(scale) * z.index_add(0, ids, dout.abs()),
            torch.bincount(ids, minlength=rows)[:, None])


def check_grad(got, ids, dout, scale=1.0, padding=None):
    want, mag, n = grad64(ids, dout, got.shape[0], scale, padding)
    tol = (DEPTH + n / 256 + 1) * 2.0 ** -24 * mag + (half_step(got.dtype) + 2.0 ** -24) * want.abs()
    tol += torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist())
    assert not got[(n == 0)[:, 0]].any()  # rows without a token


def inputs(gpu, n, rows, h, dtype, kind="random", seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    w = torch.randn(rows, h, device=gpu, generator=g).to(dtype)
    d = torch.randn(n, h, device=gpu, generator=g).to(dtype)
    if kind == "random":
        ids = torch.randint(0, rows, (n,), device=gpu, generator=g)
    elif kind == "same":
        ids = torch.full((n,), rows - 1, device=gpu, dtype=torch.int64)
    elif kind == "few":  # long runs that begin and end inside chunks
        ids = torch.randint(0, min(rows, 5), (n,), device=gpu, generator=g) * (rows // 5)
    elif kind == "sorted":
        ids = (torch.arange(n, device=gpu) * rows) // n
    else:  # skewed, the most frequent ids neighbours
        ids = (rows ** torch.rand(n, device=gpu, generator=g, dtype=torch.float64)).long() - 1
    return ids.clamp_(0, rows - 1), w, d


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("n,rows,h", [(1, 1, 1), (1, 3, 8), (5, 7, 64), (16, 1000, 4096),
                                      (33, 100, 72), (7, 50, 1000), (3, 20, 8200), (130, 64, 257),
                                      (300, 11, 7)])
def test_forward(gpu, n, rows, h, dtype):
    ids, w, _ = inputs(gpu, n, rows, h, dtype, seed=h)
    assert same(scaled_embedding(ids, w), w[ids])
    out = scaled_embedding(ids, w, scale=1.7)
    want = w[ids].double() * 1.7
    # 1.7 reaches the kernel as fp32; below the type's smallest normal number a step is
    # smallest_normal * eps whatever the value, so a rounding is off by up to half of that
    tol = (half_step(dtype) + 2 * 2.0 ** -24) * want.abs()
    tol += torch.finfo(dtype).smallest_normal * half_step(dtype)
    assert out.dtype == dtype and bool(((out.double() - want).abs() <= tol).all())


def test_forward_shapes_and_ids(gpu):
    ids, w, _ = inputs(gpu, 24, 50, 96, BF)
    x = scaled_embedding(ids.view(2, 3, 4), w)
    assert x.shape == (2, 3, 4, 96) and same(x.view(24, 96), w[ids])
    assert same(scaled_embedding(ids.int(), w), w[ids])
    assert same(scaled_embedding(ids[::2], w), w[ids[::2]])  # strided ids
    wide = torch.randn(50, 200, device=gpu).to(BF)
    assert same(scaled_embedding(ids, wide[:, 3:99]), wide[ids, 3:99])  # strided, unaligned rows
    assert same(scaled_embedding(ids, wide.t()[:, :50].contiguous().t()), wide[ids, :200])
    assert scaled_embedding(ids[:0], w).shape == (0, 96)
    assert same(scaled_embedding(ids[3], w), w[ids[3]])  # one id without a dimension
    wr = w.clone().requires_grad_()
    (g,) = torch.autograd.grad(scaled_embedding(ids[3], wr), wr, w[1])
    assert same(g[ids[3]], w[1]) and int(g.any(1).sum()) == 1
    bad = torch.tensor([-1, 50, 3, 1 << 40, -(1 << 40)], device=gpu)
    out = scaled_embedding(bad, w)
    assert bool(out[[0, 1, 3, 4]].isnan().all()) and same(out[2], w[3])


BWD = [(1, 1, 1, "random"), (1, 5, 8, "random"), (31, 3, 64, "same"), (32, 3, 64, "same"),
       (33, 40, 72, "few"), (64, 9, 130, "few"), (1024, 1000, 96, "skewed"),
       (2047, 13, 100, "few"), (2048, 2000, 40, "random"), (2049, 2000, 40, "random"),
       (2049, 6, 264, "same"), (5000, 30, 1000, "few"), (8191, 50257, 64, "skewed"),
       (8192, 50257, 72, "random"), (8193, 3000, 72, "few"),
       (63, 30, 8, "few"), (65, 30, 8, "few"), (4097, 3000, 72, "few"), (8191, 1, 40, "same"), (5000, 70000, 2048, "skewed"),
       (6001, (1 << 20) + 5, 64, "random"), (16384, 3000, 520, "skewed"), (4500, 1 << 20, 8, "random"), (70000, 17, 9, "few"),
       (300001, 1025, 3, "skewed"), (300000, 2, 8, "same"), (4096, 4096, 2056, "sorted"),
       (2500, 300, 4097, "skewed")]


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("n,rows,h,kind", BWD)
def test_gradient(gpu, n, rows, h, kind, dtype):
    ids, w, d = inputs(gpu, n, rows, h, dtype, kind, seed=n + h)
    if dtype == F16:
        d = d / 64  # sums within fp16's range
    w.requires_grad_()
    (g,) = torch.autograd.grad(scaled_embedding(ids, w, 0.5), w, d)
    assert g.dtype == dtype and g.shape == w.shape
    check_grad(g, ids, d, 0.5)
    # the order of the sums is the ids' alone
    assert same(g, torch.autograd.grad(scaled_embedding(ids, w, 0.5), w, d)[0])


@pytest.mark.parametrize("n", [100, 3000])
@pytest.mark.parametrize("pad", [0, 7, -1])
def test_padding_and_outside(gpu, n, pad):
    rows = 40
    ids, w, d = inputs(gpu, n, rows, 80, BF, seed=n)
    ids[::3] = pad % rows
    ids[1::10] = -1
    ids[2::10] = rows
    ids[5] = 1 << 40
    d[::3] = float("nan")  # what reaches a padded or an unknown token stays out of the gradient
    d[1::10] = float("inf")
    d[2::10] = float("nan")
    d[5] = float("nan")
    ids[0::30] = pad % rows
    w.requires_grad_()
    out = scaled_embedding(ids, w, padding_idx=pad)
    (g,) = torch.autograd.grad(out, w, d)
    keep = (ids >= 0) & (ids < rows) & (ids != pad % rows)
    check_grad(g, ids[keep], d[keep])
    assert bool(keep.any()) and bool(d[keep].isfinite().all())


def test_gradient_against_differences(gpu):
    # the output is linear in the weight: a step's difference is the directional derivative
    ids, w, d = inputs(gpu, 500, 60, 24, F32, "skewed")
    w.requires_grad_()
    (g,) = torch.autograd.grad(scaled_embedding(ids, w, 3.0), w, d)
    dirn = torch.randn_like(w)
    with torch.no_grad():
        diff = (scaled_embedding(ids, w + 0.5 * dirn, 3.0).double()
                - scaled_embedding(ids, w - 0.5 * dirn, 3.0).double())
    got, want = float((g.double() * dirn).sum()), float((diff * d).sum())
    # both sides are sums of 12000 products whose terms carry a few fp32 roundings each
    scale = float((diff.abs() * d.abs()).sum()) + 3 * float((w.abs()[ids] * d.abs()).sum())
    assert abs(got - want) <= (DEPTH + 8) * 2.0 ** -24 * scale


def test_gradient_layouts(gpu):
    ids, w, d = inputs(gpu, 600, 50, 96, BF, "skewed")
    w.requires_grad_()
    ref = torch.autograd.grad(scaled_embedding(ids, w), w, d)[0]
    wide = torch.full((600, 131), float("nan"), device=gpu, dtype=BF)
    wide[:, 5:101] = d
    assert same(ref, torch.autograd.grad(scaled_embedding(ids, w), w, wide[:, 5:101])[0])
    out = scaled_embedding(ids.view(6, 100), w)
    assert same(ref, torch.autograd.grad(out, w, d.view(6, 100, 96))[0])
    # an upstream gradient without memory of its own
    out = scaled_embedding(ids, w)
    (g,) = torch.autograd.grad(out.float().sum(), w)
    check_grad(g, ids, torch.ones_like(d))
    # a weight whose columns are strided keeps its gradient's shape and values
    wt = w.detach().t().contiguous().t().requires_grad_()
    assert same(ref, torch.autograd.grad(scaled_embedding(ids, wt), wt, d)[0].contiguous())
    empty = torch.autograd.grad(scaled_embedding(ids[:0], w), w, d[:0])[0]
    assert not empty.any()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("n,rows,h", [(70, 9, 64), (70, 9, 67), (2100, 30, 1000), (2100, 5, 8193)])
def test_stays_inside(gpu, n, rows, h, dtype):
    lib = _lib.load()
    st = _lib.stream_handle(gpu)
    ids, w, d = inputs(gpu, n, rows, h, dtype, "skewed", seed=h)
    code = _lib.DTYPE_CODE[dtype]
    gw, go = Guarded(rows, h, h + 5, dtype, gpu, w), Guarded(n, h, h + 3, dtype, gpu)
    gi = torch.full((n + 200,), 1 << 50, dtype=torch.int64, device=gpu)
    gi[100:100 + n] = ids
    ip = _lib.ptr(gi[100:])
    _lib.check(lib.ts_embedding_fwd(ip, n, gw.p, h + 5, code, rows, h, 1.0, go.p, h + 3, st), "fwd")
    assert same(go.t, w[ids]) and go.intact() and gw.intact()
    gd, gg = Guarded(n, h, h + 7, dtype, gpu, d), flat(rows * h, dtype, gpu)
    wsb = int(lib.ts_embedding_bwd_workspace_size(n, rows, h))
    ws = flat(wsb, torch.uint8, gpu)
    _lib.check(lib.ts_embedding_bwd(ip, n, gd.p, h + 7, code, rows, h, 1.0, -1, gg.p, ws.p, wsb, st),
               "bwd")
    assert gg.intact() and ws.intact() and gd.intact()
    check_grad(gg.t.view(rows, h), ids, d)


def test_module_stream_and_graph(gpu):
    m = ScaledEmbedding(100, 64, scale=8.0, padding_idx=3, device=gpu, dtype=BF)
    ids, _, d = inputs(gpu, 2500, 100, 64, BF, "skewed")
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        (g1,) = torch.autograd.grad(m(ids), m.weight, d)
    torch.cuda.current_stream(gpu).wait_stream(side)
    check_grad(g1, ids, d, 8.0, 3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    sids, sd = ids.clone(), d.clone()
    with torch.cuda.graph(graph):
        out = m(sids)
        (g2,) = torch.autograd.grad(out, m.weight, sd)
    for rep in range(4):
        sids.copy_(torch.randint(0, 100, (2500,), device=gpu) if rep else ids)
        sd.copy_(d * (rep + 1))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        (g3,) = torch.autograd.grad(m(sids), m.weight, sd)
        assert same(g2, g3) and same(out, m(sids)), rep


def test_saved_ids_elsewhere(gpu):
    ids, w, d = inputs(gpu, 600, 50, 96, BF, "skewed")
    w.requires_grad_()
    want = torch.autograd.grad(scaled_embedding(ids.view(20, 30), w), w, d.view(20, 30, 96))[0]
    with saved_elsewhere():
        out = scaled_embedding(ids.view(20, 30).clone(), w)
    assert same(want, torch.autograd.grad(out, w, d.view(20, 30, 96))[0])
