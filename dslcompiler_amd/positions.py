"""Rotary positions on torch tensors.

- :class:`RotaryTable`: the angles that pairs of a head turn by at each position,
  plain or scaled for contexts longer than those of the training;
- :func:`rotary`: queries and keys turned by them, in one launch.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import LLK_BF16, LLK_FP32, check, lib
from .decoder import _begin, _context, _kind
from .ops import _torch

_SCALINGS = {None: 0, "linear": 1, "base": 2, "yarn": 3, "bands": 4}
_FLOATS = _INT32 = None  # torch dtype -> llk_dtype (0 for positions)


class RotaryTable:
    """Frequencies (radians a position) of rotary_dim / 2 pairs, and their table
    on a device.

    Plain: base ** (-2 i / rotary_dim).  For contexts `factor` times as long:

    - "linear": all of them / factor;
    - "base": those of the base base * factor ** (rotary_dim / (rotary_dim - 2));
    - "yarn": / factor for pairs that turn less than `slow` (1) times over
      `trained` positions, as they are for those beyond `fast` (32) times, mixed
      by the pair's number between; the result is multiplied by
      attention_factor, 0.1 ln(factor) + 1 if none is given;
    - "bands": / factor below `slow` (1) turns, as they are above `fast` (4), mixed
      by the turns between.
    """

    def __init__(self, rotary_dim: int, *, base: float = 10000.0, scaling: str | None = None,
                 factor: float = 1.0, trained: float | None = None, fast: float | None = None,
                 slow: float = 1.0, attention_factor: float | None = None, device="cuda"):
        if scaling not in _SCALINGS:
            raise ValueError(f"unknown scaling {scaling!r}; expected one of {tuple(_SCALINGS)}")
        if scaling in ("yarn", "bands") and trained is None:
            raise ValueError(f"scaling {scaling!r} needs `trained`, the positions of the training")
        if fast is None:
            fast = 4.0 if scaling == "bands" else 32.0
        f, own = (C.c_double * max(rotary_dim // 2, 1))(), C.c_double()
        check(lib().llk_rotary_frequencies(
            _lib.RotaryParams(rotary_dim, base, _SCALINGS[scaling], factor, trained or 0.0, fast,
                              slow), f, own))
        self._fill(list(f), own.value if attention_factor is None else attention_factor, device)

    @classmethod
    def from_frequencies(cls, frequencies, *, attention_factor: float = 1.0,
                         device="cuda") -> "RotaryTable":
        """Any frequencies (radians a position), one a pair."""
        table = cls.__new__(cls)
        table._fill([float(f) for f in frequencies], attention_factor, device)
        return table

    def _fill(self, frequencies, attention_factor, device) -> None:
        n = len(frequencies)
        turns = (C.c_uint64 * max(n, 1))()
        check(lib().llk_rotary_turns((C.c_double * max(n, 1))(*frequencies), n, turns))
        self.frequencies, self.attention_factor = frequencies, float(attention_factor)
        self.rotary_dim = 2 * n
        torch = _torch()
        # turns a position, in units of 2^-64 (the bits of an unsigned number)
        self.turns = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns],
                                  dtype=torch.int64, device=device)
        self.turns_ptr, self.device_index = self.turns.data_ptr(), self.turns.get_device()


def _rows(t, name: str, dev: int, kinds):
    _kind(t, name, dev, kinds)
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim]")
    return _lib.Tensor3D(t.data_ptr(), *t.shape, *t.stride())


def _new(like, d):
    """A contiguous result of like's shape (descriptor d), and its descriptor."""
    t = like.new_empty(like.shape)
    return t, _lib.Tensor3D(t.data_ptr(), d.dim0, d.dim1, d.dim2, d.dim1 * d.dim2, d.dim2, 1)


def rotary(q, k, positions, table: RotaryTable, *, interleaved: bool = False,
           inverse: bool = False, q_out=None, k_out=None, stream=None):
    """(q, k) with the first table.rotary_dim values of every head turned; the
    others are copied.

    q and k (or None) are bf16 or fp32 [tokens, heads, head_dim], positions int32
    [tokens], any of them.  Pair i is (x[i], x[i + rotary_dim / 2]), or (x[2 i],
    x[2 i + 1]) with interleaved=True: a cos - b sin, b cos + a sin, times the
    table's attention_factor.  inverse=True turns back by the same angles (and
    multiplies by the same factor): the gradient of the call without it.  q_out
    and k_out may be q and k."""
    global _FLOATS, _INT32
    if _INT32 is None:  # the one that is set last: a second thread finds both of them, or none
        torch = _torch()
        _FLOATS = {torch.bfloat16: LLK_BF16, torch.float32: LLK_FP32}
        _INT32 = {torch.int32: 0}
    dev = _begin()
    qd = _rows(q, "q", dev, _FLOATS)
    kind = _FLOATS[q.dtype]
    kd = kod = None
    if k is not None:
        kd = _rows(k, "k", dev, _FLOATS)
        if k.dtype is not q.dtype:
            raise ValueError("q and k have different types")
    elif k_out is not None:
        raise ValueError("k_out without k")
    _kind(positions, "positions", dev, _INT32)
    if positions.dim() != 1 or positions.shape[0] != qd.dim0:
        raise ValueError("positions must be [tokens]")
    if qd.dim0 > 1 and positions.stride(0) != 1:
        raise ValueError("positions must be contiguous")
    if table.device_index != dev:
        raise ValueError("table is not on the current device")
    if q_out is None:
        q_out, qod = _new(q, qd)
    else:
        qod = _rows(q_out, "q_out", dev, _FLOATS)
    if k is not None:
        if k_out is None:
            k_out, kod = _new(k, kd)
        else:
            kod = _rows(k_out, "k_out", dev, _FLOATS)
    if q_out.dtype is not q.dtype or (k is not None and k_out.dtype is not q.dtype):
        raise ValueError("q_out and k_out must have q's type")
    check(lib().llk_rotary(qd, kd, positions.data_ptr(), table.turns_ptr, table.rotary_dim // 2,
                           table.attention_factor, kind,
                           (1 if interleaved else 0) | (2 if inverse else 0), qod, kod,
                           _context(dev, stream)))
    return q_out, k_out
