"""The 4-bit paged cache and the attention over it, against their definitions
in 64 bits (kv4_ref): quantisation bit by bit, reading back exactly, attention
over lengths from 0, all head sizes, groups, pages, windows and first tokens,
masked and absent keys that hold NaN, strides, streams and graphs.

Bound of the attention: weights and result are each rounded to bf16, by at most
2^-8 of the value, and fp32 scores, exponentials and sums add less than 2^-12 of
the weights: |error| <= 2^-8 |out| + (2^-8 + 2^-12) sum(weight |v|)."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu


def _bits(t):
    """bf16 tensor -> float64 values."""
    return t.double().cpu().numpy()


def _dev(torch, x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    return t.to(dtype) if dtype is not None else t


class Case:
    """Sequences in a cache with pages in any order; garbage where nothing is held."""

    def __init__(self, torch, lens, news, heads, D, page, seed=0, spare=3, big=1.0):
        rng = np.random.default_rng(seed)
        self.torch, self.D, self.page, self.heads = torch, D, page, heads
        self.lens = np.array(lens, np.int32)
        self.news = list(news)
        self.starts = None if all(n == 1 for n in news) else \
            np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.tokens = int(sum(news))
        need = [-(-n // page) for n in lens]
        total = sum(need) + spare
        order = rng.permutation(total)
        self.table = np.full((len(lens), max(max(need), 1)), -1, np.int32)
        # bytes of 255 everywhere: NaN scales where nothing was written
        self.pool = np.full((total, heads, page // 16 * 17 * D), 255, np.uint8)
        self.free = order[sum(need):]
        at = 0
        codes, scales = ref._views(self.pool, D)
        for s, n in enumerate(lens):
            self.table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            if n <= 0:
                continue
            for part in (0, 1):
                x = ref.bf16_round(rng.standard_normal((n, heads, D)).astype(np.float32) * big)
                c, e = ref.quantise(x)
                packed = c[..., 0::2] | (c[..., 1::2] << 4)
                pos = np.arange(n)
                pg, off = self.table[s, pos // page], pos % page
                codes[pg, :, off // 16, part, :, off % 16] = packed
                scales[pg, :, off // 16, part, :, off % 16] = e
        self.rng = rng

    def queries(self, H, sigma=1.0):
        return ref.bf16_round(
            self.rng.standard_normal((self.tokens, H, self.D)).astype(np.float32) * sigma)

    def dev(self):
        t = self.torch
        return (_dev(t, self.pool), _dev(t, self.table), _dev(t, self.lens),
                None if self.starts is None else _dev(t, self.starts))


def check(got, want, mag, what=""):
    got = _bits(got)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), (what, "NaN", int((np.isnan(got) != nan).sum()))
    bound = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -12) * mag + 1e-30
    bad = ~nan & ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4])


def attend(llk, c, q, **kw):
    pool, table, lens, starts = c.dev()
    scale = kw.pop("scale", c.D ** -0.5)
    got = llk.kv4_attention(_dev(c.torch, q, c.torch.bfloat16), pool, table, lens, starts=starts,
                            scale=scale, **kw)
    kw.pop("max_len", None)
    want, mag = ref.attention(q, c.pool, c.table, c.lens, c.starts, scale, **kw)
    return got, want, mag


# ---- write and read ---------------------------------------------------------


@pytest.mark.parametrize("D,heads,page", [(64, 1, 16), (64, 8, 64), (128, 8, 64), (128, 5, 32),
                                          (128, 32, 256), (256, 2, 16), (256, 3, 128)])
def test_write_and_read(llk, gpu, D, heads, page):
    lens, news = [1, 40, 0, 129, 16, 77], [1, 17, 0, 128, 16, 3]
    c = Case(gpu, lens, news, heads, D, page, seed=D + heads)
    kv = [ref.bf16_round(c.rng.standard_normal((c.tokens, heads, D)).astype(np.float32) * 3)
          for _ in range(2)]
    pool, table, lens_d, starts = c.dev()
    llk.kv4_write(_dev(gpu, kv[0], gpu.bfloat16), _dev(gpu, kv[1], gpu.bfloat16), pool, table,
                  lens_d, starts=starts)
    want = c.pool.copy()
    for s in range(len(lens)):
        for i, (p, page_id) in enumerate(ref.places(len(want), page, c.table, c.lens, c.starts, s)):
            t = int(c.starts[s]) + i
            ref.put(want, page_id, p % page, kv[0][t], kv[1][t])
    # every byte: what was written, and all that was not
    assert np.array_equal(pool.cpu().numpy(), want)
    k, v = llk.kv4_read(pool, table, lens_d, head_dim=D, starts=starts, tokens=c.tokens)
    for got, x in zip((k, v), kv):
        assert np.array_equal(_bits(got), ref.values(*ref.quantise(x)))
    # whole sequences
    all_starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    k, v = llk.kv4_read(pool, table, lens_d, head_dim=D, starts=_dev(gpu, all_starts),
                        tokens=int(all_starts[-1]))
    t = 0
    for s, n in enumerate(lens):
        for p in range(n):
            wk, wv = ref.get(want, int(c.table[s, p // page]), p % page, D)
            assert np.array_equal(_bits(k[t]), wk) and np.array_equal(_bits(v[t]), wv), (s, p)
            t += 1


def test_quantisation_of_every_bf16(llk, gpu):
    """Blocks that begin with each positive bf16 as their largest magnitude,
    infinities and NaN among them, and values at and beside the codes' ties."""
    D = 64
    tops = np.arange(0x8000, dtype=np.uint32)  # bits of the largest magnitude
    x = np.zeros((tops.size, 1, D), np.float32)
    top = (tops << 16).astype(np.uint32).view(np.float32)
    frac = np.array([1, 0.9, 0.75, 5 / 7, 0.5, 3.5 / 7, 2.5 / 7, 0.25, 1.75 / 7, 1.25 / 7, 0.75 / 7,
                     0.25 / 7, 0.1, 0.03, 0.01, 0], np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        part = ref.bf16_round(top[:, None] * frac)
    part[np.isinf(top)[:, None] & (frac == 0)] = 0
    x[:, 0, :16], x[:, 0, 16:32] = part, -part
    x[:, 0, 32:] = 1.0  # another block: nothing of the first one may reach it
    T = tops.size
    page = 4096
    table = np.arange(T // page, dtype=np.int32)[None]
    lens, starts = np.array([T], np.int32), np.array([0, T], np.int32)
    pool = llk.kv4_cache(T // page, 1, page, D)
    xd = _dev(gpu, x.view(np.int32) >> 16).to(gpu.int16).view(gpu.bfloat16)
    args = (_dev(gpu, table), _dev(gpu, lens))
    llk.kv4_write(xd, xd, pool, *args, starts=_dev(gpu, starts))
    codes, scales = ref._views(pool.cpu().numpy(), D)
    want_c, want_s = ref.quantise(x[:, 0])
    got = codes[:, 0, :, 0].transpose(0, 1, 3, 2, 4).reshape(T, 2, 16)  # [token, block, bytes]
    assert np.array_equal(scales[:, 0, :, 0].transpose(0, 1, 3, 2).reshape(T, 2), want_s)
    assert np.array_equal(got, want_c[..., 0::2] | (want_c[..., 1::2] << 4))
    assert np.array_equal(codes[:, :, :, 0], codes[:, :, :, 1])
    k, v = llk.kv4_read(pool, *args, head_dim=D, starts=_dev(gpu, starts), tokens=T)
    want = ref.values(want_c, want_s)
    assert np.array_equal(_bits(k[:, 0]), want, equal_nan=True)
    assert np.array_equal(_bits(v[:, 0]), want, equal_nan=True)


def test_tokens_without_a_place(llk, gpu):
    """Before position 0, past the table, on absent pages, outside every
    sequence: not written, and read as zeros."""
    D, page, heads = 64, 16, 2
    pool = llk.kv4_cache(3, heads, page, D)
    pool.fill_(7)
    table = np.array([[0, -1], [1, 99], [2, 2], [0, 0]], np.int32)
    lens = np.array([20, 18, 2, 40], np.int32)  # the last one is longer than the table
    starts = np.array([1, 7, 11, 15, 21], np.int32)  # row 0 and rows 21, 22 in no sequence
    T = 23
    x = _dev(gpu, np.ones((T, heads, D), np.float32), gpu.bfloat16)
    args = (_dev(gpu, table), _dev(gpu, lens))
    llk.kv4_write(x, x, pool, *args, starts=_dev(gpu, starts))
    want = np.full((3, heads, page // 16 * 17 * D), 7, np.uint8)
    held = np.zeros(T, bool)
    one = np.ones((heads, D))
    for s in range(4):
        for i, (p, pg) in enumerate(ref.places(3, page, table, lens, starts, s)):
            if pg >= 0:
                ref.put(want, pg, p % page, one, one)
                held[int(starts[s]) + i] = True
    assert 0 < held.sum() < T - 3
    assert np.array_equal(pool.cpu().numpy(), want)
    k, v = llk.kv4_read(pool, *args, head_dim=D, starts=_dev(gpu, starts), tokens=T)
    for got in (k, v):
        got = _bits(got)
        assert (got[held] == 1).all() and (got[~held] == 0).all()


def test_no_sequences(llk, gpu):
    """Rows that belong to no sequence at all: nothing written, zeros read."""
    pool = llk.kv4_cache(2, 2, 16, 64)
    pool.fill_(7)
    table = gpu.zeros((0, 3), dtype=gpu.int32, device="cuda")
    lens = gpu.zeros(0, dtype=gpu.int32, device="cuda")
    starts = gpu.zeros(1, dtype=gpu.int32, device="cuda")
    x = gpu.ones((5, 2, 64), dtype=gpu.bfloat16, device="cuda")
    llk.kv4_write(x, x, pool, table, lens, starts=starts)
    assert bool((pool == 7).all())
    k, v = x.clone(), x.clone()
    llk.kv4_read(pool, table, lens, head_dim=64, starts=starts, k=k, v=v)
    assert bool((k == 0).all()) and bool((v == 0).all())
    out = llk.kv4_attention(x, pool, table, lens, starts=starts)
    assert out.shape == x.shape


def test_write_read_strides(llk, gpu):
    """Keys and values as slices at odd elements and with heads outermost; a
    cache that is one layer of a larger pool; results into a wider buffer."""
    D, page, heads, T = 128, 32, 3, 50
    rng = np.random.default_rng(3)
    big = _dev(gpu, rng.standard_normal((T, 2 * heads * D + 9)).astype(np.float32), gpu.bfloat16)
    k = big[:, 1:1 + heads * D].unflatten(1, (heads, D))
    v = _dev(gpu, rng.standard_normal((heads, T, D)).astype(np.float32),
             gpu.bfloat16).transpose(0, 1)
    layers = gpu.full((4, 5, heads, page // 16 * 17 * D), 9, dtype=gpu.uint8, device="cuda")
    cache = layers[:, 2]
    table = _dev(gpu, np.array([[3, 1, 77, 77]], np.int32))[:, :2]
    lens, starts = _dev(gpu, np.array([T], np.int32)), _dev(gpu, np.array([0, T], np.int32))
    llk.kv4_write(k, v, cache, table, lens, starts=starts)
    out = gpu.full((T, heads, 2 * D + 1), 4.0, dtype=gpu.bfloat16, device="cuda")
    rk = out[:, :, 1:D + 1]
    rv = gpu.empty((heads, T, D), dtype=gpu.bfloat16, device="cuda").transpose(0, 1)
    llk.kv4_read(cache, table, lens, head_dim=D, starts=starts, k=rk, v=rv)
    for got, x in ((rk, k), (rv, v)):
        assert np.array_equal(_bits(got), ref.values(*ref.quantise(_bits(x))))
    assert bool((out[:, :, 0] == 4).all()) and bool((out[:, :, D + 1:] == 4).all())
    assert bool((layers[:, [0, 1, 3, 4]] == 9).all())


# ---- attention --------------------------------------------------------------


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 4, 8, 16, 17, 40])
def test_single_tokens(llk, gpu, D, group):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 130, 259, 0]
    c = Case(gpu, lens, [1] * len(lens), 2, D, 16, seed=D + group)
    check(*attend(llk, c, c.queries(2 * group)))


@pytest.mark.parametrize("page", [16, 32, 64, 512])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (7, 4), (33, 0), (64, 40),
                                          (200, 64), (5000, 3), (16, 5000)])
def test_window_and_first_tokens(llk, gpu, page, window, sinks):
    c = Case(gpu, [1, 40, 300, 129, 511], [1] * 5, 2, 64, page, seed=window + sinks)
    check(*attend(llk, c, c.queries(8), window=window, sinks=sinks))
    c = Case(gpu, [5, 300, 64, 200, 1], [5, 70, 64, 1, 1], 2, 64, page, seed=window)
    check(*attend(llk, c, c.queries(6), window=window, sinks=sinks))


@pytest.mark.parametrize("D,heads,group,news,before", [
    (128, 2, 1, [100], 0), (128, 2, 4, [33, 1, 64], 50), (128, 1, 8, [2, 3, 4, 5], 100),
    (64, 3, 1, [257], 0), (64, 2, 5, [31, 130], 7), (256, 1, 2, [40, 17], 20),
    (128, 1, 1, [1, 0, 300, 0, 2], 0), (128, 1, 40, [9], 33),
])
def test_prompts(llk, gpu, D, heads, group, news, before):
    lens = [n + before * (i + 1) if n else 0 for i, n in enumerate(news)]
    c = Case(gpu, lens, news, heads, D, 32, seed=D + group)
    check(*attend(llk, c, c.queries(heads * group)))
    check(*attend(llk, c, c.queries(heads * group), window=37, sinks=5))


def test_long_sequences_are_split(llk, gpu):
    c = Case(gpu, [5000, 4097, 1, 3333], [1] * 4, 1, 128, 64, seed=8)
    q = c.queries(4)
    pool, table, lens, _ = c.dev()
    plan = llk.describe_kv4_attention(_dev(gpu, q, gpu.bfloat16), pool, table, lens)
    assert plan["splits"] > 1 and plan["workspace_bytes"] > 0
    got, want, mag = attend(llk, c, q)
    check(got, want, mag)
    # other hints at the length, too small ones among them: other splits
    for max_len in (1, 300, 4000, 5000):
        check(attend(llk, c, q, max_len=max_len)[0], want, mag, max_len)
    check(*attend(llk, c, q, window=2000, sinks=4))
    # a prompt's last rows over a long context
    c = Case(gpu, [4100, 2500], [9, 3], 1, 128, 64, seed=9)
    check(*attend(llk, c, c.queries(4)))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64, 512])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 1), (33, 0), (64, 40), (200, 64), (16, 5000)])
def test_full_row_tiles(llk, gpu, D, page, window, sinks):
    """Rows enough for the tiles of 128, of which each sequence's last is part."""
    c = Case(gpu, [300, 130, 511, 1], [130, 130, 1, 1], 1, D, page, seed=D + window)
    q = c.queries(3)
    pool, table, lens, starts = c.dev()
    plan = llk.describe_kv4_attention(_dev(gpu, q, gpu.bfloat16), pool, table, lens, starts=starts)
    assert plan["rows"] == 128
    check(*attend(llk, c, q, window=window, sinks=sinks))
    # tiles by the rows of a sequence on average, the same rows in both
    for new, rows in ((96, 32), (97, 128)):
        c = Case(gpu, [200, 100], [new, new], 1, D, page, seed=new)
        q = c.queries(1)
        pool, table, lens, starts = c.dev()
        plan = llk.describe_kv4_attention(_dev(gpu, q, gpu.bfloat16), pool, table, lens,
                                          starts=starts)
        assert plan["rows"] == rows
        check(*attend(llk, c, q, window=window, sinks=sinks))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_prompt_over_a_long_context_is_split(llk, gpu, D):
    c = Case(gpu, [3000, 1700, 140], [130, 100, 120], 1, D, 64, seed=D)
    c.table[0, 20] = -1  # a page given back
    q = c.queries(1)
    pool, table, lens, starts = c.dev()
    plan = llk.describe_kv4_attention(_dev(gpu, q, gpu.bfloat16), pool, table, lens, starts=starts)
    assert plan["rows"] == 128 and plan["splits"] > 1 and plan["launches"] == 2
    got, want, mag = attend(llk, c, q)
    check(got, want, mag)
    for max_len in (1, 300, 1500):
        check(attend(llk, c, q, max_len=max_len)[0], want, mag, max_len)
    check(*attend(llk, c, q, window=1100, sinks=70))


def test_large_scores(llk, gpu):
    """Scores of hundreds, where the running maximum moves late and far."""
    c = Case(gpu, [700, 64], [1, 30], 2, 128, 16, seed=4, big=4.0)
    q = c.queries(4, sigma=8.0)
    got, want, mag = attend(llk, c, q, scale=1.0)
    # scores to 2^11, so weights within 2^-24 * 2^11 * a few of theirs; below
    # 1e-30 (weights of e^-100 are no fp32 numbers) nothing is asked
    got = _bits(got)
    bound = 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -7) * mag + 1e-30
    assert (np.abs(got - want) <= bound).all()


def test_rows_that_see_nothing(llk, gpu):
    """Lengths of 0 and fewer positions than new tokens: zeros, nothing else."""
    c = Case(gpu, [0, 3, 40], [4, 5, 2], 2, 64, 16, seed=5)
    got, want, mag = attend(llk, c, c.queries(4))
    assert (want[:6] == 0).all() and (_bits(got)[:6] == 0).all()
    check(got, want, mag)
    c = Case(gpu, [0, 0], [1, 1], 2, 128, 16)
    got, _, _ = attend(llk, c, c.queries(2))
    assert (_bits(got) == 0).all()


@pytest.mark.parametrize("news", [[1, 3, 2], [20, 0, 30], [130, 140]])
def test_rows_outside_every_sequence_are_not_written(llk, gpu, news):
    c = Case(gpu, [n + 40 for n in news], news, 2, 64, 16, seed=sum(news))
    q = c.queries(2)
    want, mag = ref.attention(q, c.pool, c.table, c.lens, c.starts, 64 ** -0.5)
    pool, table, lens, starts = c.dev()
    padded = gpu.full((c.tokens + 3, 2, 64), float("nan"), dtype=gpu.bfloat16, device="cuda")
    padded[1:-2] = _dev(gpu, q)
    out = gpu.full_like(padded, 5.0)
    llk.kv4_attention(padded, pool, table, lens, starts=starts + 1, out=out)
    check(out[1:-2], want, mag)
    assert bool((out[:1] == 5).all()) and bool((out[-2:] == 5).all())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_unseen_keys_never_reach_a_row(llk, gpu, D):
    """NaN keys and values past the end, after a row's position, outside its
    window and on pages given back: rows that do not see them are as without
    them, rows that do are NaN."""
    lens, news = [70, 200], [60, 30]
    for window, sinks in ((0, 0), (20, 3)):
        c = Case(gpu, lens, news, 2, D, 16, seed=D)
        codes, scales = ref._views(c.pool, D)
        # one block of a value of head 0, and a key of head 1, in the middle of
        # the new tokens; blocks outside the window of the second sequence
        for s, pos, head, part, block in ((0, 30, 0, 1, 1), (0, 47, 1, 0, 0), (1, 185, 0, 1, 0),
                                          (1, 185, 1, 1, D // 32 - 1), (1, 100, 0, 1, 0)):
            scales[c.table[s, pos // 16], head, pos % 16 // 16, part, block, pos % 16] = 255
        if window:
            c.table[1, 2] = -1  # positions 32 to 47: given back
        q = c.queries(6)
        got, want, mag = attend(llk, c, q, window=window, sinks=sinks)
        nan = np.isnan(want)
        assert nan.any() and not nan.all(axis=(1, 2)).all()
        check(got, want, mag, (window, sinks))


def test_absent_pages(llk, gpu):
    c = Case(gpu, [100, 64, 40], [1, 20, 1], 2, 128, 16, seed=6)
    c.table[0, 2] = -1
    c.table[0, 5] = c.pool.shape[0]
    c.table[1, 0] = -2147483648
    c.table[2, :] = 2147483647
    got, want, mag = attend(llk, c, c.queries(4))
    assert (want[-1] == 0).all()
    check(got, want, mag)


def test_queries_that_are_not_finite(llk, gpu):
    c = Case(gpu, [50, 50], [3, 1], 1, 64, 16, seed=7)
    q = c.queries(2)
    q[1, 0, 5] = np.nan
    q[2, 1, 6] = np.inf
    got, want, mag = attend(llk, c, q)
    assert np.isnan(_bits(got)[1, 0]).all() and np.isnan(_bits(got)[2, 1]).all()
    keep = np.ones((4, 2), bool)
    keep[1, 0] = keep[2, 1] = False
    g = _bits(got)[keep]
    assert (np.abs(g - want[keep]) <= 2.0 ** -8 * np.abs(want[keep]) +
            (2.0 ** -8 + 2.0 ** -12) * mag[keep]).all()


def test_attention_strides(llk, gpu):
    """Queries as a slice of a fused product at an odd element, results with
    heads outermost or in a wider buffer, a table that is part of a wider one."""
    c = Case(gpu, [100, 37], [20, 5], 2, 128, 32, seed=11)
    H, T, D = 6, c.tokens, 128
    q = c.queries(H)
    want, mag = ref.attention(q, c.pool, c.table, c.lens, c.starts, D ** -0.5)
    pool, table, lens, starts = c.dev()
    layers = gpu.zeros((pool.shape[0], 3, *pool.shape[1:]), dtype=gpu.uint8, device="cuda")
    layers[:, 1] = pool
    wide = gpu.full((T, 2 * H * D + 5), float("nan"), dtype=gpu.bfloat16, device="cuda")
    qd = wide[:, 3:3 + H * D].unflatten(1, (H, D))
    qd.copy_(_dev(gpu, q))
    more = gpu.full((2, table.shape[1] + 3), -1, dtype=gpu.int32, device="cuda")
    more[:, :table.shape[1]] = table
    out = gpu.empty((H, T, D), dtype=gpu.bfloat16, device="cuda").transpose(0, 1)
    got = llk.kv4_attention(qd, layers[:, 1], more[:, :table.shape[1]], lens, starts=starts, out=out)
    assert got is out
    check(out, want, mag)
    buf = gpu.full((T, H, D + 3), 8.0, dtype=gpu.bfloat16, device="cuda")
    llk.kv4_attention(qd, layers[:, 1], more, lens, starts=starts, out=buf[:, :, 1:D + 1])
    check(buf[:, :, 1:D + 1], want, mag)
    assert bool((buf[:, :, 0] == 8).all()) and bool((buf[:, :, D + 1:] == 8).all())


def test_cache_beyond_32_bit_offsets(llk, gpu):
    """Pages at byte offsets above 2^32: written, read and attended."""
    D, heads, page = 128, 8, 256
    per = heads * page // 16 * 17 * D
    pages = (1 << 32) // per + 40
    pool = llk.kv4_cache(pages, heads, page, D)
    c = Case(gpu, [600, 300], [600, 300], heads, D, page, seed=12)
    table = np.array([[pages - 1, 3, pages - 7], [pages - 20, pages - 2, 0]], np.int32)
    td, ld, sd = _dev(gpu, table), _dev(gpu, c.lens), _dev(gpu, c.starts)
    x = [ref.bf16_round(c.rng.standard_normal((900, heads, D)).astype(np.float32))
         for _ in range(2)]
    llk.kv4_write(*(_dev(gpu, t, gpu.bfloat16) for t in x), pool, td, ld, starts=sd)
    k, v = llk.kv4_read(pool, td, ld, head_dim=D, starts=sd, tokens=900)
    kq, vq = (ref.values(*ref.quantise(t)) for t in x)
    assert np.array_equal(_bits(k), kq) and np.array_equal(_bits(v), vq)
    q = ref.bf16_round(c.rng.standard_normal((2, heads, D)).astype(np.float32))
    got = _bits(llk.kv4_attention(_dev(gpu, q, gpu.bfloat16), pool, td, ld))
    for s, (a, b) in enumerate(((0, 600), (600, 900))):
        for h in range(heads):
            w = kq[a:b, h] @ q[s, h].astype(np.float64) * D ** -0.5
            w = np.exp(w - w.max())
            w /= w.sum()
            want, mag = w @ vq[a:b, h], w @ np.abs(vq[a:b, h])
            assert (np.abs(got[s, h] - want) <= 2.0 ** -8 * np.abs(want) +
                    (2.0 ** -8 + 2.0 ** -12) * mag).all(), (s, h)


def test_streams_scratch_and_repeats(llk, gpu):
    """The same bits from run to run, on another stream, and with a workspace
    of the caller's; one that is too small is refused."""
    c = Case(gpu, [3000, 900], [1, 1], 2, 128, 64, seed=13)
    pool, table, lens, _ = c.dev()
    q = _dev(gpu, c.queries(8), gpu.bfloat16)
    want = llk.kv4_attention(q, pool, table, lens)
    need = llk.describe_kv4_attention(q, pool, table, lens)["workspace_bytes"]
    assert need > 0
    for _ in range(3):
        assert gpu.equal(llk.kv4_attention(q, pool, table, lens), want)
    scratch = gpu.full((need,), 255, dtype=gpu.uint8, device="cuda")  # NaN in fp32
    assert gpu.equal(llk.kv4_attention(q, pool, table, lens, scratch=scratch), want)
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        got = llk.kv4_attention(q, pool, table, lens)
    gpu.cuda.synchronize()
    assert gpu.equal(got, want)
    with pytest.raises(llk.LLKError, match="scratch"):
        llk.kv4_attention(q, pool, table, lens, scratch=scratch[:need - 256])


def test_graph_replays(llk, gpu):
    """A decode step (write, then attend) captured once: lengths, tables, keys
    and queries are read at each replay."""
    c = Case(gpu, [700, 40, 300], [1, 1, 1], 2, 128, 64, seed=14)
    pool, table, lens, _ = c.dev()
    k, v = (_dev(gpu, c.queries(2), gpu.bfloat16) for _ in range(2))
    q = _dev(gpu, c.queries(8), gpu.bfloat16)

    def step():
        llk.kv4_write(k, v, pool, table, lens)
        return llk.kv4_attention(q, pool, table, lens)

    # the library's workspace of the capturing stream exists before the capture
    side = gpu.cuda.Stream()
    with gpu.cuda.stream(side):
        step()
    gpu.cuda.synchronize()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        out = step()
    for n in range(4):
        lens += 1
        q.mul_(1.25)
        k.add_(0.5)
        if n == 2:
            lens.fill_(17)
        before = pool.clone()
        want = step().clone()
        after = pool.clone()
        pool.copy_(before)
        out.zero_()
        graph.replay()
        gpu.cuda.synchronize()
        assert gpu.equal(out, want), n
        assert gpu.equal(pool, after), n
