"""Attention over the 4-bit cache on each of its row tiles (16, 32 and 128
rows), whose kernels mask, join and round by themselves: every test names the
tile that its calls run on.  Definitions, cases and bounds are those of
test_gpu_kv4."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import Case, _bits, _dev, attend, check

pytestmark = pytest.mark.gpu

# row tile -> (new tokens of each sequence, query heads to a key head): one new
# token each (no starts) and more
LAYOUTS = [(16, [1, 1, 1, 1], 4), (16, [2, 3, 4, 3], 5), (32, [1, 1, 1, 1], 20),
           (32, [7, 20, 9, 12], 3), (128, [1, 1, 1, 1], 100), (128, [60, 130, 97, 101], 2)]
TILES = pytest.mark.parametrize("rows,news,group", LAYOUTS)


def planned(llk, c, q, rows, **kw):
    """The plan of a call, which has to be on the row tile."""
    pool, table, lens, starts = c.dev()
    plan = llk.describe_kv4_attention(_dev(c.torch, q, c.torch.bfloat16), pool, table, lens,
                                      starts=starts, **kw)
    assert plan["rows"] == rows
    return plan


# ---- lengths beyond the table -------------------------------------------------


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 0), (5, 0), (40, 7), (3, 20), (1000, 0)])
@TILES
def test_lengths_beyond_the_table(llk, gpu, rows, news, group, D, window, sinks):
    """A token keeps its position: what it would see past the table is absent,
    and its window ends where it does."""
    c = Case(gpu, [64 + n for n in news], news, 1, D, 16, seed=D + window)
    c.table = np.ascontiguousarray(c.table[:, :4])  # 64 positions
    c.lens = np.array([80, 64, 65 + news[2], 150], np.int32)
    q = c.queries(group)
    planned(llk, c, q, rows, window=window, sinks=sinks)
    got, want, mag = attend(llk, c, q, window=window, sinks=sinks)
    check(got, want, mag)
    c.lens = np.array([0x7fffffff, 70, 1 << 30, 103], np.int32)
    check(*attend(llk, c, q, window=window, sinks=sinks))


@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 0), (700, 100)])
@pytest.mark.parametrize("rows,news,group", [(16, [1, 1], 4), (32, [9, 8], 2), (128, [130, 110], 1)])
def test_long_lengths_beyond_the_table(llk, gpu, rows, news, group, window, sinks):
    """The same over keys that are split."""
    c = Case(gpu, [2560, 2560], news, 1, 128, 64, seed=rows)
    c.lens = np.array([2900, 2560 + news[1] // 2], np.int32)
    q = c.queries(group)
    assert planned(llk, c, q, rows, window=window, sinks=sinks)["splits"] > 1
    check(*attend(llk, c, q, window=window, sinks=sinks))


@TILES
def test_lengths_below_zero(llk, gpu, rows, news, group):
    """No position at all, however far below: zeros beside sequences that hold some."""
    c = Case(gpu, [40 + n for n in news], news, 2, 64, 16, seed=rows)
    c.lens = np.array([-1, c.lens[1], -0x80000000, 0], np.int32)
    q = c.queries(2 * group)
    planned(llk, c, q, rows)
    for window, sinks in ((0, 0), (9, 2)):
        got, want, mag = attend(llk, c, q, window=window, sinks=sinks)
        assert (want[:news[0]] == 0).all() and (want[-news[3]:] == 0).all()
        check(got, want, mag, (window, sinks))


# ---- rows whose every score is -infinity ----------------------------------------


@pytest.mark.parametrize("before", [20, 2500])
@pytest.mark.parametrize("rows,news,group", [(16, [1, 1], 4), (16, [2, 3], 5), (32, [9, 8], 3),
                                             (128, [65, 80], 2)])
def test_scores_of_minus_infinity(llk, gpu, rows, news, group, before):
    """Zeros, also where a value that the row sees is NaN; NaN for the other rows."""
    c = Case(gpu, [before + n for n in news], news, 1, 64, 16, seed=rows)
    codes, scales = ref._views(c.pool, 64)
    keys = codes[:, :, :, 0, 0, :, 0]
    keys[:] = keys & 0xf0 | 2  # the first element of every key: 1 times its scale
    scales[c.table[0, 0], 0, 0, 1, 1, 5] = 255  # a block of the value at position 5
    q = c.queries(group)
    q[:, 0, 0] = -np.inf
    assert (planned(llk, c, q, rows)["splits"] > 1) == (before > 1000)
    got, want, mag = attend(llk, c, q)
    assert (want[:, 0] == 0).all() and np.isnan(want[:news[0], 1:, 32:]).all()
    check(got, want, mag)
