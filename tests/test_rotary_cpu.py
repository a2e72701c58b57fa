"""Rotary frequencies against their formulas, their table, and what the entry
points refuse before any device work."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest

FAKE = 1 << 20  # an aligned address


@pytest.fixture()
def L(llk):
    return llk.lib()


def table(llk, *a, **kw):
    return llk.RotaryTable(*a, device="cpu", **kw)


@pytest.mark.parametrize("rot", [2, 34, 64, 128, 1024])
def test_frequencies(llk, rot):
    i = np.arange(rot // 2)
    plain = 10000.0 ** (-2 * i / rot)
    close = dict(rtol=1e-13, atol=0)
    assert np.allclose(table(llk, rot).frequencies, plain, **close)
    assert np.allclose(table(llk, rot, scaling="linear", factor=4.0).frequencies, plain / 4, **close)
    if rot > 2:
        base = 10000.0 * 4.0 ** (rot / (rot - 2))
        assert np.allclose(table(llk, rot, scaling="base", factor=4.0).frequencies,
                           base ** (-2 * i / rot), **close)
    t = table(llk, rot, scaling="yarn", factor=4.0, trained=2048)
    low = max(math.floor(rot * math.log(2048 / (64 * math.pi)) / (2 * math.log(10000))), 0)
    high = min(math.ceil(rot * math.log(2048 / (2 * math.pi)) / (2 * math.log(10000))), rot - 1)
    r = np.clip((i - low) / max(high - low, 0.001), 0, 1)
    assert np.allclose(t.frequencies, r * plain / 4 + (1 - r) * plain, **close)
    assert math.isclose(t.attention_factor, 0.1 * math.log(4) + 1)
    t = table(llk, rot, scaling="yarn", factor=4.0, trained=2048, attention_factor=1.0)
    assert t.attention_factor == 1.0
    t = table(llk, rot, scaling="bands", factor=4.0, trained=2048)
    r = np.clip((2048 * plain / (2 * math.pi) - 1) / 3, 0, 1)
    assert np.allclose(t.frequencies, (1 - r) * plain / 4 + r * plain, **close)
    assert t.attention_factor == 1.0


def test_turns(llk):
    """f / (2 pi) modulo 1 to 2^-64."""
    from fractions import Fraction
    f = [1.0, 2 * math.pi, 0.0, -1.0, 1e-12, 12345.678, 1e15]
    got = [int(t) % (1 << 64) for t in llk.RotaryTable.from_frequencies(f, device="cpu").turns]
    # pi to 120 bits: 4 (4 atan(1/5) - atan(1/239)) by its series
    def atan_inv(n):
        return sum(Fraction((-1) ** k, (2 * k + 1) * n ** (2 * k + 1)) for k in range(60))
    two_pi = 8 * (4 * atan_inv(5) - atan_inv(239))
    for x, t in zip(f, got):
        want = Fraction(x) / two_pi
        want = (want - math.floor(want)) * (1 << 64)
        # 64 bits of the quotient: half of its last, and 2^-64 of it from 2 pi's
        near = 1 + abs(Fraction(x) / two_pi) * 2
        off = abs(want - t)
        assert min(off, (1 << 64) - off) <= near, x


def _params(**kw):
    from dslcompiler_amd._lib import RotaryParams
    d = dict(rotary_dim=64, base=10000.0, scaling=0, factor=2.0, trained=2048.0, fast=32.0, slow=1.0)
    d.update(kw)
    return RotaryParams(*d.values())


def test_frequency_refusals(L, llk):
    f, a = (C.c_double * 512)(), C.c_double()
    assert L.llk_rotary_frequencies(_params(), f, a) == 0
    assert L.llk_rotary_frequencies(None, f, a) == -1
    assert L.llk_rotary_frequencies(_params(), None, a) == -1
    assert L.llk_rotary_frequencies(_params(), f, None) == -1
    for rot in (0, -2, 3, 1026):
        assert L.llk_rotary_frequencies(_params(rotary_dim=rot), f, a) == -2, rot
    nan, inf = float("nan"), float("inf")
    for bad in (dict(base=1.0), dict(base=nan), dict(base=inf), dict(scaling=5), dict(scaling=-1),
                dict(scaling=1, factor=0.0), dict(scaling=1, factor=nan), dict(scaling=3, trained=0.0),
                dict(scaling=4, trained=nan), dict(scaling=3, fast=1.0), dict(scaling=4, slow=0.0),
                dict(scaling=4, fast=inf), dict(scaling=2, factor=1e-9)):
        assert L.llk_rotary_frequencies(_params(**bad), f, a) == -1, bad
    assert L.llk_rotary_frequencies(_params(scaling=2, rotary_dim=2), f, a) == -2
    t = (C.c_uint64 * 4)()
    good = (C.c_double * 4)(1, 2, 3, 4)
    assert L.llk_rotary_turns(good, 4, t) == 0
    assert L.llk_rotary_turns(None, 4, t) == -1 and L.llk_rotary_turns(good, 4, None) == -1
    assert L.llk_rotary_turns(good, 0, t) == -2 and L.llk_rotary_turns(good, 513, t) == -2
    assert L.llk_rotary_turns((C.c_double * 1)(inf), 1, t) == -1
    with pytest.raises(ValueError, match="scaling"):
        table(llk, 64, scaling="other")
    with pytest.raises(ValueError, match="trained"):
        table(llk, 64, scaling="yarn")
    with pytest.raises(llk.LLKError, match="rotary_dim"):
        table(llk, 63)
    with pytest.raises(llk.LLKError, match="pairs"):
        llk.RotaryTable.from_frequencies([], device="cpu")


def _x(T=3, H=2, D=128, s0=None, s1=None, data=FAKE, s2=1):
    from dslcompiler_amd._lib import Tensor3D
    return Tensor3D(data, T, H, D, H * D if s0 is None else s0, D if s1 is None else s1, s2)


def test_refusals(L):
    x = _x()

    def call(q=x, k=None, pos=FAKE, turns=FAKE, pairs=64, factor=1.0, dtype=0, flags=0, qo=x, ko=None):
        return L.llk_rotary(q, k, pos, turns, pairs, factor, dtype, flags, qo, ko, None)

    assert call(q=None) == -1 and call(qo=None) == -1
    assert call(k=x) == -1 and call(ko=x) == -1
    assert call(pos=None) == -1 and call(turns=None) == -1
    assert call(dtype=1) == -3 and call(dtype=9) == -3
    assert call(flags=4) == -1
    for pairs in (0, -1, 65):
        assert call(pairs=pairs) == -2, pairs
    assert call(factor=float("nan")) == -1 and call(factor=float("inf")) == -1
    assert call(q=_x(D=1025), qo=_x(D=1025)) == -2
    assert call(q=_x(H=4097), qo=_x(H=4097)) == -2
    assert call(q=_x(T=1 << 24), qo=_x(T=1 << 24)) == -2
    assert call(q=_x(T=-1), qo=_x(T=-1)) == -2
    for bad, code in ((dict(T=4), -2), (dict(H=3), -2), (dict(D=64), -2), (dict(data=None), -1),
                      (dict(data=FAKE + 1), -4), (dict(s2=2), -4), (dict(s0=-5), -4)):
        assert call(qo=_x(**bad)) == code, bad
        if not {"T", "H", "D"} & set(bad):
            assert call(q=_x(**bad)) == code, bad
        else:
            assert call(k=x, ko=_x(**bad)) == code, bad
    for bad in (dict(s0=128, s1=128), dict(s0=255), dict(s1=127), dict(s0=0)):
        assert call(qo=_x(**bad)) == -4, bad
    assert call(q=_x(data=FAKE + 2), qo=x, dtype=2) == -4
    assert call(k=_x(D=64), ko=_x(D=64)) == -2
    # nothing to do
    e = _x(T=0)
    assert call(q=e, qo=e, pos=None) == 0
    assert call(q=_x(H=0), qo=_x(H=0), pos=None) == 0


def test_python_refusals(llk):
    import torch
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        llk.rotary(x, x, torch.zeros(4, dtype=torch.int32), table(llk, 64))
