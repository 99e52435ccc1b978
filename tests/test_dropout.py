"""Dropout without a GPU: the generator against published vectors, refusals of the entry points and
of the functions, workspace sizes, the module."""
import ctypes

import numpy as np
import pytest
import torch

from philox import bits16, keep_mask, philox
from trainscale_amd import _lib
from trainscale_amd.kernels import (FusedDropoutAddRMSNorm, fused_dropout, fused_dropout_add,
                                    fused_dropout_add_rms_layernorm)
from trainscale_amd.kernels.dropout_kernels import _rng

OK, INVALID, DTYPE, SHAPE, WORKSPACE = 0, -1, -2, -3, -4
FAKE = 0x1000  # never dereferenced: every call below fails validation


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_against_published_vectors(counter, key, want):
    assert tuple(int(w[0]) for w in philox(counter, key)) == want


def test_mask_statistics():
    b = bits16(64, 1000, 12345, 0)
    # 64000 draws of a mean of 32767.5: within 5 standard errors
    assert abs(b.mean() - 32767.5) < 5 * 65536 / 12 ** 0.5 / 64000 ** 0.5
    m = keep_mask(64, 1000, 12345, 0, 0.1)
    assert abs(m.mean() - 0.9) < 5 * 0.3 / 64000 ** 0.5 + 2 ** -17
    assert not np.array_equal(m, keep_mask(64, 1000, 12345, 1, 0.1))
    # columns past the last whole group of 8 use a group of their own
    assert np.array_equal(bits16(3, 13, 5, 7)[:, :8], bits16(3, 16, 5, 7)[:, :8])


def rng(**kw):
    return ctypes.byref(_lib.DropoutRng(**{**dict(seed=1, offset=2, state=None, drop=6554), **kw}))


def fwd(x=FAKE, ldx=64, res=FAKE, ldr=64, out=FAKE, ldo=64, dtype=1, rows=4, cols=64, r=None):
    return _lib.load().ts_dropout_fwd(x, ldx, res, ldr, out, ldo, dtype, rows, cols,
                                      rng() if r is None else r, None)


def test_dropout_entry_is_checked():
    assert fwd(dtype=7) == DTYPE
    assert fwd(rows=-1) == SHAPE and fwd(cols=-1) == SHAPE
    assert fwd(x=None) == INVALID and fwd(out=None) == INVALID
    assert fwd(ldx=63) == SHAPE and fwd(ldr=63) == SHAPE and fwd(ldo=63) == SHAPE
    assert fwd(r=rng(drop=-1)) == INVALID and fwd(r=rng(drop=65537)) == INVALID
    assert fwd(r=rng(state=FAKE + 4)) == INVALID
    assert _lib.load().ts_dropout_fwd(FAKE, 64, None, 0, FAKE, 64, 1, 4, 64, None, None) == INVALID
    assert fwd(rows=1 << 40, cols=64) == SHAPE
    assert fwd(rows=0, x=None, out=None) == OK and fwd(cols=0, x=None, out=None) == OK


def norm_fwd(x=FAKE, ldx=64, res=FAKE, ldr=64, dtype=1, w=FAKE, wdtype=1, y=FAKE, h=FAKE,
             rstd=FAKE, rows=4, cols=64, eps=1e-6, r=None):
    return _lib.load().ts_dropout_add_rmsnorm_fwd(x, ldx, res, ldr, dtype, w, wdtype, y, h, rstd,
                                                  rows, cols, eps, rng() if r is None else r, None)


def norm_bwd(dy=FAKE, lddy=64, dh=FAKE, lddh=64, h=FAKE, ldh=64, dtype=1, w=FAKE, wdtype=1,
             rstd=FAKE, dx=FAKE, dres=FAKE, dw=FAKE, rows=4, cols=64, r=None, ws=FAKE,
             wsb=1 << 40):
    return _lib.load().ts_dropout_add_rmsnorm_bwd(dy, lddy, dh, lddh, h, ldh, dtype, w, wdtype,
                                                  rstd, dx, dres, dw, rows, cols,
                                                  rng() if r is None else r, ws, wsb, None)


def test_norm_entries_are_checked():
    for call in (norm_fwd, norm_bwd):
        assert call(dtype=7) == DTYPE and call(wdtype=2) == DTYPE
        assert call(rows=-1) == SHAPE and call(cols=0) == SHAPE and call(cols=16385) == SHAPE
        assert call(w=None) == INVALID and call(r=rng(drop=70000)) == INVALID
    for k in ("x", "res", "y", "h", "rstd"):
        assert norm_fwd(**{k: None}) == INVALID, k
    assert norm_fwd(ldx=63) == SHAPE and norm_fwd(ldr=63) == SHAPE
    assert norm_fwd(eps=-1.0) == INVALID and norm_fwd(eps=float("nan")) == INVALID
    assert norm_fwd(rows=0, x=None) == OK
    assert norm_bwd(rows=0) == SHAPE
    assert norm_bwd(h=None) == INVALID and norm_bwd(rstd=None) == INVALID
    assert norm_bwd(dy=None, dh=None) == INVALID
    for k in ("lddy", "lddh", "ldh"):
        assert norm_bwd(**{k: 63}) == SHAPE
    need = _lib.load().ts_dropout_add_rmsnorm_bwd_workspace_size(4, 64)
    assert need >= 64 * 4
    assert norm_bwd(wsb=need - 1) == WORKSPACE and norm_bwd(ws=None) == WORKSPACE
    assert norm_bwd(ws=FAKE + 8) == WORKSPACE
    size = _lib.load().ts_dropout_add_rmsnorm_bwd_workspace_size
    assert size(0, 64) == size(4, 0) == size(4, 16385) == 0


def test_functions_refuse():
    x, w = torch.zeros(4, 64), torch.ones(64)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="p must be"):
            fused_dropout(x, p)
        with pytest.raises(ValueError, match="p must be"):
            FusedDropoutAddRMSNorm(64, p)
    for rng_ in ((-1, 0), (0, 1 << 64), (1 << 64, 0)):
        with pytest.raises(ValueError, match="seed and offset"):
            fused_dropout(x, 0.5, rng=rng_)
    for rng_ in (torch.zeros(2), torch.zeros(3, dtype=torch.int64),
                 torch.zeros(4, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError, match="rng must be"):
            fused_dropout(x, 0.5, rng=rng_)
    with pytest.raises(ValueError, match="residual"):
        fused_dropout_add(x, x[:2], 0.5)
    with pytest.raises(TypeError, match="residual dtype"):
        fused_dropout_add(x, x.half(), 0.5)
    with pytest.raises(ValueError, match="weight"):
        fused_dropout_add_rms_layernorm(x, x, torch.ones(63), 0.5)
    with pytest.raises(ValueError, match="weight"):
        fused_dropout_add_rms_layernorm(x[:, :0], x[:, :0], w[:0], 0.5)
    for call in (lambda: fused_dropout(x, 0.5), lambda: fused_dropout_add(x, x, 0.5),
                 lambda: fused_dropout_add_rms_layernorm(x, x, w, 0.5),
                 lambda: fused_dropout(x.requires_grad_(), 0.5)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


@pytest.mark.parametrize("device", ["meta", "cpu"])
def test_seed_is_drawn_on_the_cpu(device):
    """rng=None draws from torch's CPU generator whatever the default device."""
    torch.manual_seed(5)
    want = [_rng("test", None, 100) for _ in range(3)]
    torch.manual_seed(5)
    with torch.device(device):
        assert [_rng("test", None, 100) for _ in range(3)] == want
    assert len(set(want)) == 3
