"""The gated feed-forward block without a GPU: refusals of the entry points and of the functions,
workspace sizes, and the module."""
import ctypes

import pytest
import torch

from trainscale_amd import _lib
from trainscale_amd.kernels import FusedGatedMLP, fused_gated_linear, fused_gated_mlp

OK, INVALID, DTYPE, SHAPE, WORKSPACE = 0, -1, -2, -3, -4
FAKE = 0x1000  # never dereferenced: every call below fails validation


def args(**kw):
    a = dict(x=FAKE, ldx=64, w_gate=FAKE, ld_gate=64, w_up=FAKE, ld_up=64, w_down=FAKE,
             ld_down=128, N=16, H=64, F=128, O=64, activation=0, dtype=_lib.TS_BF16)
    return _lib.GatedMLPArgs(**{**a, **kw})


def fwd(a, gate=FAKE, up=FAKE, act=FAKE, out=FAKE, ws=FAKE, wsb=1 << 40):
    p = None if a is None else ctypes.byref(a)
    return _lib.load().ts_gated_mlp_fwd(p, gate, up, act, out, ws, wsb, None)


def bwd(a, gate=FAKE, up=FAKE, act=FAKE, dout=FAKE, ldd=64, dx=FAKE, dwg=FAKE, dwu=FAKE, dwd=FAKE,
        ws=FAKE, wsb=1 << 40):
    p = None if a is None else ctypes.byref(a)
    return _lib.load().ts_gated_mlp_bwd(p, gate, up, act, dout, ldd, dx, dwg, dwu, dwd, ws, wsb,
                                        None)


BAD = [(dict(dtype=_lib.TS_F32), DTYPE), (dict(dtype=9), DTYPE), (dict(activation=4), INVALID),
       (dict(activation=-1), INVALID), (dict(N=-1), SHAPE), (dict(H=0), SHAPE),
       (dict(F=0), SHAPE), (dict(O=0), SHAPE), (dict(H=60), SHAPE), (dict(F=100), SHAPE),
       (dict(O=12), SHAPE), (dict(ldx=56), SHAPE), (dict(ldx=68), SHAPE),
       (dict(ld_gate=32), SHAPE), (dict(ld_up=32), SHAPE), (dict(ld_down=64), SHAPE),
       (dict(ld_up=(1 << 21) + 8), SHAPE), (dict(H=1 << 22, ldx=1 << 22), SHAPE),
       (dict(N=(1 << 31) + 1), SHAPE), (dict(x=None), INVALID), (dict(w_up=None), INVALID),
       (dict(x=FAKE + 8), INVALID), (dict(w_down=FAKE + 2), INVALID)]


@pytest.mark.parametrize("kw,code", BAD)
def test_operands_are_checked(kw, code):
    assert fwd(args(**kw)) == code, _lib.last_error()
    assert bwd(args(**kw)) == code, _lib.last_error()


def test_buffers_are_checked():
    assert fwd(None) == INVALID and bwd(None) == INVALID
    assert fwd(args(), act=None) == INVALID
    assert fwd(args(), out=None) == INVALID
    assert fwd(args(w_down=None)) == INVALID  # an out without w_down
    assert fwd(args(), gate=None) == INVALID and fwd(args(), up=None) == INVALID
    assert fwd(args(), act=FAKE + 4) == INVALID and fwd(args(), ws=FAKE + 4) == INVALID
    assert fwd(args(N=0)) == OK  # no rows: nothing to do
    assert bwd(args(N=0)) == SHAPE
    for k in ("gate", "up", "act", "dout"):
        assert bwd(args(), **{k: None}) == INVALID
        assert bwd(args(), **{k: FAKE + 2}) == INVALID
    assert bwd(args(), ldd=56) == SHAPE and bwd(args(), ldd=68) == SHAPE
    assert bwd(args(w_down=None), ldd=128) == INVALID  # dw_down without w_down
    assert bwd(args(), dwd=FAKE + 8) == INVALID
    need = _lib.load().ts_gated_mlp_bwd_workspace_size(16, 64, 128, 64)
    assert need >= 2 * 2 * 16 * 128
    assert bwd(args(), wsb=need - 1) == WORKSPACE and bwd(args(), ws=None) == WORKSPACE


def test_workspace_sizes():
    lib = _lib.load()
    for n, h, f, o in ((0, 64, 64, 64), (4, 0, 64, 64), (4, 64, 0, 0), (4, 64, 64, -1)):
        assert lib.ts_gated_mlp_fwd_workspace_size(n, h, f, o) == 0
        assert lib.ts_gated_mlp_bwd_workspace_size(n, h, f, o) == 0
    assert lib.ts_gated_mlp_fwd_workspace_size(100, 64, 64, 0) == 0


def test_pad_is_checked():
    lib = _lib.load()

    def pad(count=1, dtype=_lib.TS_BF16, jobs=True, **kw):
        j = dict(src=FAKE, row_stride=4, col_stride=1, rows=2, cols=4, dst=FAKE, dst_rows=2,
                 dst_cols=8)
        return lib.ts_pad_matrices((_lib.PadJob * 9)(*[_lib.PadJob(**{**j, **kw})] * 9) if jobs
                                   else None, count, dtype, None)

    assert pad(0) == OK and pad(rows=0, dst_rows=0) == OK and pad(0, jobs=False) == OK
    assert pad(9) == INVALID and pad(-1) == INVALID and pad(jobs=False) == INVALID
    assert pad(dtype=_lib.TS_F32) == DTYPE
    for kw in (dict(rows=3), dict(cols=9), dict(rows=-1), dict(cols=-1), dict(row_stride=-4),
               dict(col_stride=-1), dict(dst_rows=1 << 41), dict(dst_rows=1 << 31),
               dict(dst_rows=1 << 40, dst_cols=1 << 40)):
        assert pad(**kw) == SHAPE, kw
    for kw in (dict(src=None), dict(dst=None), dict(src=FAKE + 1), dict(dst=FAKE + 1)):
        assert pad(**kw) == INVALID, kw
    assert pad(8, dst_rows=1 << 25, dst_cols=1 << 8) == SHAPE  # together more than a launch


BF = torch.bfloat16


@pytest.mark.parametrize("x,g,u,d,act,error", [
    ((4, 8), (16, 8), (16, 8), (8, 16), "swish", ValueError),
    ((4, 8), (16, 9), (16, 9), (8, 16), "silu", ValueError),
    ((4, 8), (16, 8), (15, 8), (8, 16), "silu", ValueError),
    ((4, 8), (16, 8), (16, 8), (8, 15), "silu", ValueError),
    ((4, 8), (16, 8), (16, 8), (0, 16), "silu", ValueError),
    ((4, 0), (16, 0), (16, 0), (8, 16), "silu", ValueError),
    ((4, 8), (0, 8), (0, 8), (8, 0), "silu", ValueError),
    ((), (16, 8), (16, 8), (8, 16), "silu", ValueError),
    ((4, 8), (16, 8, 1), (16, 8, 1), (8, 16), "silu", ValueError),
])
def test_functions_refuse(x, g, u, d, act, error):
    with pytest.raises(error, match="fused_gated_mlp"):
        fused_gated_mlp(*[torch.zeros(s, dtype=BF) for s in (x, g, u, d)], activation=act)


def test_types_and_devices():
    x, w, d = torch.zeros(4, 8, dtype=BF), torch.zeros(16, 8, dtype=BF), torch.zeros(8, 16, dtype=BF)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        fused_gated_mlp(x.float(), w.float(), w.float(), d.float())
    with pytest.raises(TypeError, match="up weight dtype"):
        fused_gated_linear(x, w, w.half())
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fused_gated_mlp(x, w, w, d)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fused_gated_linear(x, w.requires_grad_(), w)


def test_module():
    m = FusedGatedMLP(24, 56, "gelu", dtype=BF)
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "gate_proj.weight": (56, 24), "up_proj.weight": (56, 24), "down_proj.weight": (24, 56)}
    with pytest.raises(ValueError, match="activation"):
        FusedGatedMLP(24, 56, "tanh")


def test_operands_of_gradients_not_asked_for():
    """What only skipped gradients would read may be NULL (no workspace: refused before a launch)."""
    assert bwd(args(), act=None, dwd=None, wsb=0) == WORKSPACE
    down = dict(gate=None, up=None, dx=None, dwg=None, dwu=None)
    assert bwd(args(N=4096), wsb=0, **down) == WORKSPACE  # sums of K slots
    for k in ("dx", "dwg", "dwu"):
        others = {n: None for n in ("dx", "dwg", "dwu", "dwd") if n != k}
        assert bwd(args(), gate=None, **others) == INVALID
        assert bwd(args(), up=None, **others) == INVALID
        assert bwd(args(), act=None, wsb=0, **others) == WORKSPACE


def test_workspace_of_gradients_not_asked_for():
    """Frozen weights: no room for sums of their gradients; the one size for all is enough for each."""
    lib = _lib.load()
    size, some = lib.ts_gated_mlp_bwd_workspace_size, lib.ts_gated_mlp_bwd_grads_workspace_size
    for n, h, f, o in ((300, 2048, 5632, 2048), (2045, 768, 2048, 768), (2048, 4096, 14336, 4096),
                       (64, 4096, 14336, 4096), (1000, 96, 200, 0), (8192, 4096, 14336, 4096)):
        most = [some(n, h, f, o, g) for g in range(1, 16)]
        assert size(n, h, f, o) == max(most) and some(n, h, f, o, 0) == 0
        dg = 2 * ((2 * n * f + 255) // 256 * 256)
        assert dg <= some(n, h, f, o, 1) <= dg + 16 * n * h * 4 + 1024
        assert some(n, h, f, o, 8) <= 8 * o * f * 4 + 256  # no dg, du
    assert some(0, 64, 64, 64, 15) == some(4, 64, 64, -1, 15) == 0
    need = some(2045, 768, 2048, 768, 1)
    a = args(N=2045, H=768, F=2048, O=768, ldx=768, ld_gate=768, ld_up=768, ld_down=2048)
    others = dict(dwg=None, dwu=None, dwd=None, ldd=768)
    assert bwd(a, wsb=need - 1, **others) == WORKSPACE


def test_module_refuses_projections_that_are_more_than_their_weight():
    """The module multiplies by its projections' weights; what else a projection has come to do
    would be lost."""
    nn = torch.nn

    class Adapter(nn.Module):  # around a linear layer, its weight in reach
        def __init__(self, base):
            super().__init__()
            self.base, self.weight, self.bias = base, base.weight, None

        def forward(self, t):
            return self.base(t) + t.sum()

    class Other(nn.Linear):
        def forward(self, t):
            return 2 * super().forward(t)

    def own_forward(m):
        m.up_proj.forward = lambda t: t

    changes = [lambda m: setattr(m, "gate_proj", Adapter(m.gate_proj)), own_forward,
               lambda m: setattr(m, "down_proj", nn.Linear(56, 24, dtype=BF)),
               lambda m: setattr(m, "up_proj", Other(24, 56, bias=False, dtype=BF)),
               lambda m: m.gate_proj.register_forward_hook(lambda *a: None),
               lambda m: m.down_proj.register_forward_pre_hook(lambda *a: None),
               lambda m: m.up_proj.register_full_backward_hook(lambda *a: None)]
    for change in changes:
        m = FusedGatedMLP(24, 56, dtype=BF)
        change(m)
        with pytest.raises(ValueError, match="FusedGatedMLP: (gate|up|down)_proj"):
            m(torch.zeros(2, 24, dtype=BF))
    # a weight that is computed is a weight all the same
    m = FusedGatedMLP(24, 56, dtype=BF)
    nn.utils.parametrizations.weight_norm(m.up_proj)
    for plain in (m, FusedGatedMLP(24, 56, dtype=BF)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            plain(torch.zeros(2, 24, dtype=BF))
