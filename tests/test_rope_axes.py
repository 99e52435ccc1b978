"""Rotary positions with several axes without a GPU: the plan, refusals of the entry point and of
the functions."""
import copy
import ctypes
import pickle
from fractions import Fraction

import pytest
import torch

from trainscale_amd import _lib
from trainscale_amd.kernels import (MultiAxisRotaryEmbedding, RopeAxes, apply_rope_axes)
from trainscale_amd.kernels.rope_kernels import _axes_positions, _turn_parts, _turns

OK, INVALID, DTYPE, SHAPE = 0, -1, -2, -3
FAKE = 0x1000


def inverse_two_pi(bits):
    """floor(2^bits / (2 pi)) by Machin's formula."""
    one = 1 << bits + 64

    def atan_inv(n):
        total = term = one // n
        k, sign = 3, -1
        while term:
            term //= n * n
            total += sign * (term // k)
            k, sign = k + 2, -sign
        return total

    pi = 4 * (4 * atan_inv(5) - atan_inv(239))
    return (one << bits) // (2 * pi)


def test_turns():
    c = Fraction(inverse_two_pi(256), 1 << 256)
    for f in (1.0, 0.75, 1e-8, 3.7e-5, -0.2, 12345.678, 0.0, 2.0 ** -70):
        want = Fraction(f) * c % 1 * 2 ** 64
        assert min((_turns(f) - want) % 2 ** 64, (want - _turns(f)) % 2 ** 64) <= Fraction(51, 100)


def test_plans():
    p = RopeAxes((16, 24, 24), base=1e6)
    assert p.axis == (0,) * 16 + (1,) * 24 + (2,) * 24
    want = 1.0 / (1e6 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))
    assert torch.equal(p.inv_freq, want.double())
    q = RopeAxes((24, 20, 20), layout="interleaved")
    assert q.axis[:60] == (0, 1, 2) * 20 and q.axis[60:] == (0,) * 4
    s = RopeAxes((20, 20), layout="separate")
    assert s.axis == (0,) * 20 + (1,) * 20 and torch.equal(s.inv_freq[:20], s.inv_freq[20:])
    own = torch.linspace(1, 2, 4, dtype=torch.float64)
    assert torch.equal(RopeAxes((2, 2), inv_freq=own).inv_freq, own)
    for r in (pickle.loads(pickle.dumps(q)), copy.deepcopy(q)):
        assert r.axis == q.axis and list(r._turns_c) == list(q._turns_c)


@pytest.mark.parametrize("args", [
    dict(sections=()), dict(sections=(4, 0)), dict(sections=(200, 57)),
    dict(sections=(8, 12, 12), layout="interleaved"), dict(sections=(4, 4), layout="rows"),
    dict(sections=(2, 2), inv_freq=torch.ones(3)),
    dict(sections=(1, 1), inv_freq=torch.tensor([1.0, float("inf")])),
])
def test_plans_refuse(args):
    with pytest.raises(ValueError, match="RopeAxes"):
        RopeAxes(**args)


def entry(**kw):
    n = kw.get("R", 64) // 2
    turns, axis = (ctypes.c_uint64 * max(n, 1))(), (ctypes.c_int32 * max(n, 1))()
    a = dict(q_in=FAKE, q_out=FAKE, k_in=FAKE, k_out=FAKE, Hq=4, Hk=2, B=2, S=3, D=64, R=64,
             position_ids=FAKE, turns=ctypes.addressof(turns), axis=ctypes.addressof(axis), axes=3,
             dtype=1, interleaved=0, backward=0)
    return _lib.load().ts_rope_axes(ctypes.byref(_lib.RopeAxesArgs(**{**a, **kw})), None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=5), DTYPE), (dict(B=-1), SHAPE), (dict(S=-1), SHAPE), (dict(Hq=-1), SHAPE),
    (dict(D=0), SHAPE), (dict(R=0), SHAPE), (dict(R=31), SHAPE), (dict(R=66), SHAPE),
    (dict(R=514, D=1024), SHAPE), (dict(D=8192), SHAPE), (dict(Hq=4096), SHAPE),
    (dict(axes=0), INVALID), (dict(axes=256), INVALID), (dict(interleaved=2), INVALID),
    (dict(backward=-1), INVALID), (dict(turns=None), INVALID), (dict(axis=None), INVALID),
    (dict(q_out=None), INVALID), (dict(k_in=None), INVALID), (dict(position_ids=None), INVALID),
    (dict(B=1 << 40, S=1 << 20), SHAPE), (dict(B=0), OK), (dict(S=0), OK),
    (dict(Hq=0, Hk=0), OK),
])
def test_entry_is_checked(kw, code):
    assert entry(**kw) == code, _lib.last_error()


def test_entry_checks_the_axes():
    assert _lib.load().ts_rope_axes(None, None) == INVALID
    axis = (ctypes.c_int32 * 32)(*[0] * 31, 3)
    assert entry(axis=ctypes.addressof(axis)) == INVALID
    axis[31] = -1
    assert entry(axis=ctypes.addressof(axis)) == INVALID


def test_functions_refuse():
    p = RopeAxes((4, 4))
    q, k = torch.zeros(2, 3, 4, 16), torch.zeros(2, 3, 1, 16)
    pos = torch.zeros(2, 2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="expected"):
        apply_rope_axes(q[0], k, pos, p)
    with pytest.raises(ValueError, match="at least 16"):
        apply_rope_axes(q[..., :8], k[..., :8], pos, p)
    for bad in (k[:1], k.half(), torch.zeros(2, 3, 1, 24)):
        with pytest.raises(ValueError, match="apply_rope_axes: k"):
            apply_rope_axes(q, bad, pos, p)
    for bad in (pos[:1], pos[:, :, :2], pos[0, :1], torch.zeros(2, 3, 3, dtype=torch.int64)):
        with pytest.raises(ValueError, match="position_ids"):
            apply_rope_axes(q, k, bad, p)
    with pytest.raises(TypeError, match="position_ids"):
        apply_rope_axes(q, k, pos.float(), p)
    with pytest.raises(ValueError, match="gradients"):
        apply_rope_axes(q.clone().requires_grad_(), k, pos, p, inplace=True)
    with pytest.raises(ValueError, match="contiguous head"):
        apply_rope_axes(q.transpose(2, 3).contiguous().transpose(2, 3), None, pos, p, inplace=True)
    with pytest.raises(ValueError, match="expanded"):
        apply_rope_axes(q[:, :, :1].expand_as(q), None, pos, p, inplace=True)
    with pytest.raises(ValueError, match="same memory"):
        apply_rope_axes(q, q[:, :, :1], pos, p, inplace=True)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        MultiAxisRotaryEmbedding((4, 4))(q, k, pos)
    assert _axes_positions(pos[:, 0], 2, 2, 3).shape == (2, 2, 3)
    assert _axes_positions(pos[:, :1].int(), 2, 2, 3).shape == (2, 2, 3)


def test_every_position_is_exact():
    """The fraction of a turn as the kernel forms it, 64-bit product and rest, at any int64 position:
    off by 2^63 times half of 2^-96, and 2^-64 for the rest's own rounding."""
    c = Fraction(inverse_two_pi(256), 1 << 256)
    plan = RopeAxes((32, 32), base=500000.0)
    for i, f in enumerate(plan.inv_freq.tolist()):
        turns, rest = plan._turns_c[i], plan._rest_c[i]
        for pos in (1, 5000, -1 << 24, (1 << 40) + 17, (1 << 46) - 3, -(1 << 52) - 1, 1 << 62,
                    (1 << 63) - 1, -1 << 63):
            got = (pos * turns + (pos * rest >> 32)) % (1 << 64)
            off = (Fraction(got, 1 << 64) - pos * Fraction(f) * c) % 1
            assert min(off, 1 - off) <= Fraction(1, 1 << 33), (f, pos)


def test_rest_of_a_turn():
    c = Fraction(inverse_two_pi(256), 1 << 256)
    for f in (1.0, 0.75, 1e-8, 3.7e-5, -0.2, 12345.678, 0.0, 2.0 ** -70):
        turns, rest = _turn_parts(f)
        off = (Fraction(turns, 1 << 64) + Fraction(rest, 1 << 96) - Fraction(f) * c) % 1
        assert min(off, 1 - off) <= Fraction(51, 100 << 96) and -1 << 31 <= rest < 1 << 31
