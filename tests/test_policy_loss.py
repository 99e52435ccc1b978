"""Clipped policy loss on the CPU: host checks of the C ABI and the Python refusals."""
import ctypes
import math
import re

import pytest
import torch

from trainscale_amd import _lib
from trainscale_amd.loss import ClippedPolicyLoss, clipped_policy_loss

TS_OK, INVALID, DTYPE, SHAPE, WORKSPACE = 0, -1, -2, -3, -4
FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: every call below ends on the host


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def inputs(**k):
    a = dict(logp=0x1000, ld_logp=100, old=0x2000, ld_old=100, ref=0x3000, ld_ref=100, adv=0x4000,
             ld_adv=1, mask=0x5000, ld_mask=100, rows=700, tokens=100, clip_low=0.2, clip_high=0.2,
             kl_coef=0.1, dtype=1, old_dtype=1, ref_dtype=0, adv_per_token=0, reduction=0)
    a.update(k)
    return _lib.PolicyInputs(**a)


def test_forward_validation(lib):
    need = lib.ts_policy_loss_workspace_size(700, 100)
    assert need == 700 * 24
    assert lib.ts_policy_loss_workspace_size(4, 500) == 0 and lib.ts_policy_loss_workspace_size(0, 5) == 0

    def f(outs=(FAKE,) * 4, weights=FAKE, ws=FAKE, wsb=need, **k):
        return lib.ts_policy_loss_fwd(ctypes.byref(inputs(**k)), *outs, weights, ws, wsb, None)

    assert lib.ts_policy_loss_fwd(None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, need, None) == INVALID
    assert f(dtype=5) == DTYPE and f(old_dtype=2) == DTYPE and f(ref_dtype=2) == DTYPE
    assert f(rows=-1) == SHAPE and f(tokens=-1) == SHAPE
    assert f(rows=1 << 40, tokens=1 << 20) == SHAPE
    assert f(rows=1, tokens=1 << 31) == SHAPE
    for name in ("ld_logp", "ld_old", "ld_ref", "ld_mask"):
        assert f(**{name: 99}) == SHAPE
    assert f(ld_adv=0) == SHAPE and f(adv_per_token=1, ld_adv=99) == SHAPE
    for name in ("logp", "adv"):
        assert f(**{name: None}) == INVALID
    assert f(logp=0x1001) == INVALID and f(ref=0x3002) == INVALID and f(adv=0x4002) == INVALID
    assert f(ref=None) == INVALID  # kl_coef without a reference
    for bad in (-0.1, math.nan):
        assert f(clip_low=bad) == INVALID and f(clip_high=bad) == INVALID
        assert f(kl_coef=bad) == INVALID
    assert f(kl_coef=math.inf) == INVALID
    assert f(reduction=3) == INVALID and f(reduction=-1) == INVALID
    assert f(outs=(FAKE, None, FAKE, FAKE)) == INVALID and f(weights=None) == INVALID
    assert f(ws=None) == WORKSPACE and f(wsb=need - 1) == WORKSPACE
    assert f(ws=ctypes.c_void_p(0x1004)) == WORKSPACE


def test_small_batches_need_no_workspace(lib):
    # one round of the waves of one workgroup, 512 tokens of a row each
    size = lib.ts_policy_loss_workspace_size
    assert size(16, 512) == size(8, 513) == size(1, 8192) == size(5, 1025) == 0
    assert size(17, 512) == 17 * 24 and size(9, 513) == 18 * 24 and size(1, 8193) == 17 * 24


def test_backward_validation(lib):
    def f(weights=FAKE, dloss=FAKE, grad=FAKE, ld=100, **k):
        return lib.ts_policy_loss_bwd(ctypes.byref(inputs(**k)), weights, dloss, grad, ld, None)

    assert f(weights=None) == INVALID and f(dloss=None) == INVALID and f(grad=None) == INVALID
    assert f(ld=99) == SHAPE and f(grad=ctypes.c_void_p(0x1001)) == INVALID
    assert f(dtype=9) == DTYPE
    assert f(rows=0) == TS_OK and f(tokens=0) == TS_OK


def test_struct_is_the_headers():
    text = _lib.HEADER_PATH.read_text()
    body = re.sub(r"/\*.*?\*/", "", text[text.index("typedef struct {"):], flags=re.S)
    body = body[body.index("{") + 1:body.index("}")]
    names = [re.sub(r".*[ *]", "", v.strip()) for line in body.split(";") for v in line.split(",")]
    assert [n for n in names if n] == [name for name, _ in _lib.PolicyInputs._fields_]
    assert ctypes.sizeof(_lib.PolicyInputs) == 12 * 8 + 3 * 8 + 5 * 4 + 4


def test_python_refusals():
    lp = torch.zeros(3, 5)
    adv = torch.zeros(3)
    f = lambda **k: clipped_policy_loss(k.pop("lp", lp), k.pop("old", lp), k.pop("adv", adv), **k)
    with pytest.raises(RuntimeError, match="GPU"):
        f()
    with pytest.raises(ValueError, match="logps must be"):
        f(lp=lp[0])
    with pytest.raises(ValueError, match="reduction"):
        f(reduction="mean")
    with pytest.raises(ValueError, match="reduction"):
        ClippedPolicyLoss(reduction="mean")
    with pytest.raises(ValueError, match="clip bounds"):
        f(clip_low=-1)
    with pytest.raises(ValueError, match="clip bounds"):
        f(clip_high=math.nan)
    with pytest.raises(ValueError, match="kl_coef"):
        f(kl_coef=-0.1)
    with pytest.raises(ValueError, match="needs ref_logps"):
        f(kl_coef=0.1)
    with pytest.raises(ValueError, match="old_logps"):
        f(old=lp[:2])
    with pytest.raises(ValueError, match="ref_logps"):
        f(ref_logps=lp[:, :4])
    with pytest.raises(ValueError, match="mask"):
        f(mask=torch.ones(3))
    for shape in ((5,), (1, 5), (3, 4), ()):
        with pytest.raises(ValueError, match="advantages"):
            f(adv=torch.zeros(shape))
    with pytest.raises(TypeError, match="dtype"):
        f(lp=lp.double())
    with pytest.raises(TypeError, match="dtype"):
        f(old=lp.double())
