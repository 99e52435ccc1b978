"""KernelPatcher(fuse_mlp=True): which blocks it takes, which calls keep the module's own forward."""
import copy
import types

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from trainscale_amd import registry
from trainscale_amd.registry import KernelPatcher

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class LlamaMLP(nn.Module):
    def __init__(self, h=24, i=40, act=None, bias=False, dtype=F32, device=None):
        super().__init__()
        new = lambda a, b: nn.Linear(a, b, bias=bias, dtype=dtype, device=device)
        self.gate_proj, self.up_proj, self.down_proj = new(h, i), new(h, i), new(i, h)
        if act is not None:
            self.act_fn = act

    def forward(self, x):
        act = getattr(self, "act_fn", F.silu)
        return self.down_proj(act(self.gate_proj(x)) * self.up_proj(x))


class PlainMLP(nn.Module):
    def __init__(self):
        super().__init__()
        self.gate_proj = nn.Linear(4, 4)


def taken(m, x, monkeypatch):
    """Whether the patched forward hands the call to the fused block, and with what activation."""
    calls = []
    monkeypatch.setattr(registry, "fused_gated_mlp",
                        lambda x, g, u, d, activation: calls.append(activation) or x)
    m(x)
    return calls[0] if calls else None


class OnGpu(torch.Tensor):
    """A host tensor that says it is on a GPU, to look at the choice without one."""
    is_cuda = True


def fake(dtype=BF):
    return torch.zeros(2, 24, dtype=dtype).as_subclass(OnGpu)


def test_opt_in():
    assert KernelPatcher().fuse_mlp is False
    m = nn.Sequential(LlamaMLP(), PlainMLP())
    x = torch.randn(3, 24)
    want = m[0](x)
    p = KernelPatcher(fuse_mlp=True)
    p.patch(m)
    assert p.patched_layers == [("0", "LlamaMLP")]
    assert m[0].forward.__qualname__.startswith("auto_patch_fused_mlp")
    assert torch.equal(m[0](x), want)  # CPU tensors keep the module's forward
    other = copy.deepcopy(m[0])
    with torch.no_grad():
        other.down_proj.weight.zero_()
    assert not other(x).any() and torch.equal(m[0](x), want)
    plain = nn.Sequential(LlamaMLP())
    KernelPatcher().patch(plain)
    assert plain[0].forward.__qualname__.startswith("auto_patch_mlp")


@pytest.mark.parametrize("act,name", [
    (None, "silu"), (nn.SiLU(), "silu"), (F.silu, "silu"), (nn.GELU(), "gelu"), (F.gelu, "gelu"),
    (nn.GELU(approximate="tanh"), "gelu_tanh"), (nn.ReLU(), "relu"), (F.relu, "relu"),
    (nn.Tanh(), None), (torch.tanh, None), (lambda t: t, None)])
def test_activation(act, name, monkeypatch):
    m = LlamaMLP(act=act, dtype=BF)
    registry.auto_patch_fused_mlp(m)
    assert taken(m, fake(), monkeypatch) == name


def test_transformers_activations(monkeypatch):
    acts = pytest.importorskip("transformers.activations").ACT2FN
    for key, name in (("silu", "silu"), ("gelu", "gelu"), ("gelu_pytorch_tanh", "gelu_tanh"),
                      ("relu", "relu"), ("quick_gelu", None)):
        m = LlamaMLP(act=acts[key], dtype=BF)
        registry.auto_patch_fused_mlp(m)
        assert taken(m, fake(), monkeypatch) == name, key


def test_other_projections(monkeypatch):
    class Adapter(nn.Linear):
        pass

    def hooked(m):
        m.up_proj.register_forward_hook(lambda *a: None)

    def adapted(m):
        m.gate_proj = Adapter(24, 40, bias=False, dtype=BF)

    def replaced(m):
        m.down_proj.forward = lambda t: t

    def biased(m):
        m.down_proj.bias = nn.Parameter(torch.zeros(24, dtype=BF))

    def other_type(m):
        m.up_proj.to(F32)

    def scaled(m):
        nn.utils.parametrizations.weight_norm(m.up_proj)

    for change in (hooked, adapted, replaced, biased, other_type, scaled):
        m = LlamaMLP(dtype=BF)
        registry.auto_patch_fused_mlp(m)
        assert taken(m, fake(), monkeypatch) == "silu"
        change(m)
        ran = []
        m._trainscale_amd_forward = lambda x: ran.append(1)
        assert taken(m, fake(), monkeypatch) is None and ran, change.__name__


def test_other_calls(monkeypatch):
    m = LlamaMLP(dtype=BF)
    registry.auto_patch_fused_mlp(m)
    m._trainscale_amd_forward = lambda x: x
    assert taken(m, torch.zeros(2, 24, dtype=BF), monkeypatch) is None
    assert taken(m, fake(F16), monkeypatch) is None
    assert taken(m, fake(F32), monkeypatch) is None
    monkeypatch.setattr(torch, "is_autocast_enabled", lambda device: True)
    monkeypatch.setattr(torch, "get_autocast_dtype", lambda device: F16)
    assert taken(m, fake(), monkeypatch) is None
    monkeypatch.setattr(torch, "get_autocast_dtype", lambda device: BF)
    assert taken(m, fake(), monkeypatch) == "silu"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F16])
def test_patched_block_on_the_gpu(gpu, dtype):
    torch.manual_seed(0)
    m = LlamaMLP(136, 360, nn.GELU(approximate="tanh"), dtype=dtype, device=gpu)
    exact = LlamaMLP(136, 360, nn.GELU(approximate="tanh"), dtype=torch.float64, device=gpu)
    exact.load_state_dict(m.state_dict())
    registry.auto_patch_fused_mlp(m)
    x = torch.randn(2, 35, 136, device=gpu).to(dtype)
    dy = torch.randn(2, 35, 136, device=gpu).to(dtype)
    out = {}
    for block, t in ((m, x.clone()), (exact, x.double())):
        t.requires_grad_()
        y = block(t)
        y.backward(dy.to(y.dtype))
        out[block] = [y.detach(), t.grad] + [p.grad for p in block.parameters()]
    # three roundings of half a step (the gated product or both gradients, the result), as norms
    for got, want in zip(out[m], out[exact]):
        assert got.dtype == dtype
        err = (got.double() - want).norm() / want.norm()
        assert err <= 4 * torch.finfo(dtype).eps / 2, err


@pytest.mark.parametrize("register", ["register_forward_hook", "register_forward_pre_hook",
                                      "register_full_backward_hook",
                                      "register_full_backward_pre_hook", "register_backward_hook"])
def test_hooks_of_the_activation(register, monkeypatch):
    m = LlamaMLP(act=nn.SiLU(), dtype=BF)
    registry.auto_patch_fused_mlp(m)
    m._trainscale_amd_forward = lambda x: x
    hook = getattr(m.act_fn, register)(lambda *a: None)
    assert taken(m, fake(), monkeypatch) is None
    hook.remove()
    assert taken(m, fake(), monkeypatch) == "silu"


class NamedActMLP(LlamaMLP):
    """A block of a registered shape that keeps its activation under another name."""

    def __init__(self, name, act):
        super().__init__(dtype=BF)
        setattr(self, name, act)


class MethodMLP(LlamaMLP):
    def activation(self, t):
        return F.gelu(t)


@pytest.mark.parametrize("name,act", [
    ("act", nn.GELU()), ("act", F.gelu), ("activation", torch.tanh), ("activation_function", F.gelu),
    ("hidden_act", "gelu"), ("non_linearity", F.gelu), ("dropout", nn.Dropout(0.1)),
    ("norm", nn.LayerNorm(40))])
@pytest.mark.parametrize("act_fn", [None, nn.SiLU()])
def test_blocks_with_more_in_them(name, act, act_fn, monkeypatch):
    """What else a block holds may be part of its forward: the block keeps it, unless act_fn says
    which activation it is and the rest is no layer."""
    m = NamedActMLP(name, act)
    if act_fn is not None:
        m.act_fn = act_fn
    registry.auto_patch_fused_mlp(m)
    m._trainscale_amd_forward = lambda x: x
    layer = isinstance(act, nn.Module)
    assert taken(m, fake(), monkeypatch) == ("silu" if act_fn is not None and not layer else None)


def test_activation_as_a_method(monkeypatch):
    m = MethodMLP(dtype=BF)
    registry.auto_patch_fused_mlp(m)
    m._trainscale_amd_forward = lambda x: x
    assert taken(m, fake(), monkeypatch) is None


def test_transformers_blocks(monkeypatch):
    """The registered blocks of the model library are still taken."""
    pytest.importorskip("transformers")
    from transformers.models.llama.modeling_llama import LlamaMLP as Theirs
    for act, name in (("silu", "silu"), ("gelu_pytorch_tanh", "gelu_tanh"), ("tanh", None)):
        m = Theirs(types.SimpleNamespace(hidden_size=24, intermediate_size=40, mlp_bias=False,
                                         hidden_act=act)).to(BF)
        registry.auto_patch_fused_mlp(m)
        m._trainscale_amd_forward = lambda x: x
        assert taken(m, fake(), monkeypatch) == name


@pytest.mark.parametrize("register", ["register_module_forward_hook",
                                      "register_module_forward_pre_hook",
                                      "register_module_full_backward_hook",
                                      "register_module_full_backward_pre_hook"])
def test_hooks_of_every_module(register, monkeypatch):
    """Hooks for all modules (counters, profilers) fire for the projections too."""
    m = LlamaMLP(dtype=BF)
    registry.auto_patch_fused_mlp(m)
    m._trainscale_amd_forward = lambda x: x
    hook = getattr(nn.modules.module, register)(lambda *a: None)
    try:
        assert taken(m, fake(), monkeypatch) is None
    finally:
        hook.remove()
    assert taken(m, fake(), monkeypatch) == "silu"
