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


# ---- what a row does not see ------------------------------------------------------


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("before", [100, 2500])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
@TILES
def test_unseen_keys_never_reach_a_row(llk, gpu, rows, news, group, before, window, sinks, D):
    """NaN keys and values before the window, among the first tokens, after a row's
    position and on pages given back: rows that see them are NaN, the others as
    without them; keys split and not."""
    c = Case(gpu, [before + 7 * i + n for i, n in enumerate(news)], news, 2, D, 16, seed=D + rows)
    codes, scales = ref._views(c.pool, D)

    def spoil(s, pos, head, part, block):
        scales[c.table[s, pos // 16], head, 0, part, block, pos % 16] = 255

    mid = [int(c.lens[s]) - 1 - n // 2 for s, n in enumerate(news)]  # among the new tokens
    spoil(0, mid[0], 0, 1, 1)
    spoil(0, mid[0] - 10, 1, 0, 0)
    spoil(1, 60, 0, 1, 0)  # before every window
    spoil(1, 41, 1, 0, D // 32 - 1)
    spoil(2, 1, 1, 1, D // 32 - 1)  # a first token
    for head in (0, 1):
        for part in (0, 1):
            spoil(3, 65, head, part, 0)
    c.table[3, 4] = -1  # positions 64 to 79: given back
    q = c.queries(2 * group)
    plan = planned(llk, c, q, rows, window=window, sinks=sinks)
    assert window or (plan["splits"] > 1) == (before > 1000)
    got, want, mag = attend(llk, c, q, window=window, sinks=sinks)
    nan = np.isnan(want)
    assert nan.any() and not nan.all(axis=(1, 2)).all()
    assert not nan[-news[3]:].any()
    check(got, want, mag)


# ---- numerics and strides -----------------------------------------------------------


@TILES
def test_large_scores(llk, gpu, rows, news, group):
    """Scores of hundreds: fp32 scores to 2^11 leave weights within 2^-7."""
    c = Case(gpu, [200 + 90 * i + n for i, n in enumerate(news)], news, 2, 128, 16, seed=rows,
             big=4.0)
    q = c.queries(2 * group, sigma=8.0)
    planned(llk, c, q, rows)
    got, want, mag = attend(llk, c, q, scale=1.0)
    bound = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -7) * mag + 1e-30
    assert (np.abs(_bits(got) - want) <= bound).all()


@TILES
def test_queries_that_are_not_finite(llk, gpu, rows, news, group):
    c = Case(gpu, [50 + n for n in news], news, 1, 64, 16, seed=rows)
    q = c.queries(group)
    bad = [(0, 0, np.nan), (c.tokens // 2, group - 1, np.inf), (c.tokens - 1, 1, np.nan)]
    keep = np.ones(q.shape[:2], bool)
    for t, h, v in bad:
        q[t, h, 5] = v
        keep[t, h] = False
    planned(llk, c, q, rows)
    got, want, mag = attend(llk, c, q)
    got = _bits(got)
    assert np.isnan(got[~keep]).all()
    assert (np.abs(got[keep] - want[keep]) <= 2.0 ** -8 * np.abs(want[keep]) +
            (2.0 ** -8 + 2.0 ** -12) * mag[keep]).all()


@TILES
def test_strides(llk, gpu, rows, news, group):
    """Queries inside a wider row at an odd element; results with heads outermost
    and in a wider buffer, whose other elements stay."""
    D, H = 128, 2 * group
    c = Case(gpu, [60 + n for n in news], news, 2, D, 32, seed=rows)
    q = c.queries(H)
    planned(llk, c, q, rows)
    want, mag = ref.attention(q, c.pool, c.table, c.lens, c.starts, D ** -0.5)
    pool, table, lens, starts = c.dev()
    wide = gpu.full((c.tokens, H * D + 5), float("nan"), dtype=gpu.bfloat16, device="cuda")
    qd = wide[:, 3:3 + H * D].unflatten(1, (H, D))
    qd.copy_(_dev(gpu, q))
    out = gpu.empty((H, c.tokens, D), dtype=gpu.bfloat16, device="cuda").transpose(0, 1)
    llk.kv4_attention(qd, pool, table, lens, starts=starts, out=out)
    check(out, want, mag)
    buf = gpu.full((c.tokens, H, D + 3), 8.0, dtype=gpu.bfloat16, device="cuda")
    llk.kv4_attention(qd, pool, table, lens, starts=starts, out=buf[:, :, 1:D + 1])
    check(buf[:, :, 1:D + 1], want, mag)
    assert bool((buf[:, :, 0] == 8).all()) and bool((buf[:, :, D + 1:] == 8).all())


# ---- prompts and single tokens in one call --------------------------------------------


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows,news,group", [(16, [9, 1, 1, 1, 2, 1], 4),
                                             (32, [100, 1, 1, 1, 1, 30], 4),
                                             (128, [400, 1, 1, 1, 1], 4),
                                             (128, [1, 1, 250, 0, 1, 180], 3)])
def test_prompts_and_single_tokens(llk, gpu, rows, news, group, D):
    before = [0, 700, 31, 2000, 64, 5]
    c = Case(gpu, [before[i] + n if n else 0 for i, n in enumerate(news)], news, 1, D, 32,
             seed=D + rows)
    q = c.queries(group)
    planned(llk, c, q, rows)
    check(*attend(llk, c, q))
    check(*attend(llk, c, q, window=90, sinks=4))
    # the same rows as from a call of their own
    pool, table, lens, _ = c.dev()
    one = [s for s, n in enumerate(news) if n == 1]
    first = [int(c.starts[s]) for s in one]
    got = llk.kv4_attention(_dev(gpu, q[first], gpu.bfloat16), pool, table[one], lens[one])
    want, mag = ref.attention(q[first], c.pool, c.table[one], c.lens[one], None, D ** -0.5)
    check(got, want, mag)
