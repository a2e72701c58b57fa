"""Attention that adds its weights up, against the definition in 64 bits.

Bound.  A score has D products and is rounded with each, by 2^-24 of what S = scale
sum |q| |k| bounds, and its exponent once more; a weight carries the errors of its
own score and of the sum's: |error| <= w ((D + 16) 2^-22 S + 2^-18) with the largest
S of the row, and as much for the sums over rows."""
from __future__ import annotations

import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import Case, _dev

pytestmark = pytest.mark.gpu


def garbage(c, seed=7):
    """Marks of a pool that hold something everywhere."""
    shape = (c.pool.shape[0], c.heads, c.page)
    return np.random.default_rng(seed).uniform(0.5, 2.0, shape).astype(np.float32)


def expected(c, q, before, decay, scale, window=0, sinks=0):
    """(weights, bound) of the pool in float64; NaN where nothing is asked."""
    want, near = before.astype(np.float64), np.zeros(before.shape)
    group = q.shape[1] // c.heads
    for s, length in enumerate(c.lens):
        first = s if c.starts is None else int(c.starts[s])
        new = 1 if c.starts is None else int(c.starts[s + 1]) - first
        n = min(max(int(length), 0), c.table.shape[1] * c.page)
        if new == 0 or n == 0:
            continue
        j = np.arange(n)
        pages, off = c.table[s, j // c.page], j % c.page
        here = (pages >= 0) & (pages < c.pool.shape[0])
        keys = np.zeros((n, c.heads, c.D))
        for i in np.flatnonzero(here):
            keys[i] = ref.get(c.pool, int(pages[i]), int(off[i]), c.D)[0]
        got, most = np.zeros((n, c.heads)), np.zeros((n, c.heads))
        for i in range(new):
            p = int(length) - new + i
            seen = here & (j <= p)
            if window:
                seen &= (j > p - window) | (j < sinks)
            if not seen.any():
                continue
            for h in range(q.shape[1]):
                k, x = keys[seen, h // group], q[first + i, h].astype(np.float64)
                with np.errstate(invalid="ignore"):
                    w = k @ x * scale
                    if (w == -np.inf).all():
                        continue
                    w = np.exp(w - w.max())
                    w /= w.sum()
                    size = (np.abs(k) @ np.abs(x)).max() * scale
                got[seen, h // group] += w
                most[seen, h // group] += w * ((c.D + 16) * 2.0 ** -22 * size + 2.0 ** -18)
        at = (pages[here], slice(None), off[here])
        old = want[at] * decay if decay else 0.0
        want[at] = old + got[here]
        near[at] = most[here] + 2.0 ** -23 * np.abs(want[at])
    return want, near


def run(llk, c, q, decay=1.0, **kw):
    pool, table, lens, starts = c.dev()
    scale = c.D ** -0.5
    before = garbage(c)
    weights = _dev(c.torch, before)
    qd = _dev(c.torch, q, c.torch.bfloat16)
    max_len = kw.pop("max_len", None)
    out = llk.kv4_attention(qd, pool, table, lens, starts=starts, scale=scale, weights=weights,
                            decay=decay, max_len=max_len, **kw)
    plain = llk.kv4_attention(qd, pool, table, lens, starts=starts, scale=scale, max_len=max_len, **kw)
    assert c.torch.equal(out.view(c.torch.int16), plain.view(c.torch.int16))
    want, near = expected(c, q, before, decay, scale, **kw)
    got = weights.double().cpu().numpy()
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    bad = ~nan & ~(np.abs(got - want) <= near)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4], near[bad][:4])
    return got


@pytest.mark.parametrize("D,heads,group,page", [(64, 2, 4, 16), (128, 2, 4, 64), (128, 1, 1, 32),
                                                (256, 2, 5, 16), (128, 2, 20, 32), (64, 3, 16, 128)])
def test_single_tokens(llk, gpu, D, heads, group, page):
    lens = [1, 16, 17, 31, 33, 130, 700, 0]
    c = Case(gpu, lens, [1] * len(lens), heads, D, page, seed=D)
    q = c.queries(heads * group)
    for decay in (0.0, 0.5, 1.0):
        run(llk, c, q, decay, max_len=700 if decay else None)


@pytest.mark.parametrize("D,heads,group,page", [(64, 2, 1, 16), (128, 2, 4, 64), (256, 1, 2, 32)])
@pytest.mark.parametrize("news", [[3, 1, 0, 2, 5], [40, 7, 0, 1, 90], [150, 300, 0, 1, 1]])
def test_prompts_and_chunks(llk, gpu, D, heads, group, page, news):
    lens = [max(n + extra, 0) for n, extra in zip(news, (0, 37, 20, 129, 300))]
    c = Case(gpu, lens, news, heads, D, page, seed=D + news[0])
    q = c.queries(heads * group)
    run(llk, c, q, 1.0)
    run(llk, c, q, 0.0, max_len=max(lens))


@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 0), (33, 4), (100, 40)])
@pytest.mark.parametrize("news", [[1, 1, 1], [9, 1, 30], [130, 140, 200]])
def test_windows(llk, gpu, window, sinks, news):
    lens = [n + extra for n, extra in zip(news, (0, 60, 300))]
    c = Case(gpu, lens, news, 2, 64, 16, seed=window)
    q = c.queries(4)
    run(llk, c, q, 0.5, window=window, sinks=sinks)


@pytest.mark.parametrize("news", [[1, 1, 1], [20, 30, 5], [140, 200, 129]])
def test_absent_pages_and_lengths_beyond_the_table(llk, gpu, news):
    lens = [max(n, 90) for n in news]
    c = Case(gpu, lens, news, 2, 128, 32, seed=3)
    c.table[0, 1], c.table[1, 0] = -1, 10 ** 6
    q = c.queries(4)
    run(llk, c, q, 0.5)
    c.lens = c.lens + np.array([0, 0, 4000], np.int32)  # past what the table holds
    run(llk, c, q, 0.5)
    c.lens[0] = news[0] - 1 if news[0] > 1 else 0  # fewer than the call's tokens
    run(llk, c, q, 0.0)


@pytest.mark.parametrize("news", [[1, 1], [24, 3], [150, 131]])
def test_values_that_are_not_finite(llk, gpu, news):
    """NaN keys make the rows that see them NaN, and with them the slots that those
    see; keys that no row sees, and slots past the lengths, change nothing."""
    lens = [n + 40 for n in news]
    c = Case(gpu, lens, news, 2, 64, 16, seed=5)
    q = c.queries(2)
    _, scales = ref._views(c.pool, 64)
    last = lens[1] - 1  # seen by the last row of sequence 1 only
    scales[c.table[1, last // 16], 1, last % 16 // 16, 0, 0, last % 16] = 255
    with np.errstate(invalid="ignore"):
        run(llk, c, q, 1.0)
    q[0, 0, 0] = np.inf
    c2 = Case(gpu, lens, news, 2, 64, 16, seed=6)
    with np.errstate(invalid="ignore"):
        run(llk, c2, q, 0.0)


def test_extreme_scores(llk, gpu):
    """Scores to +-2000: weights of nothing and of one, without overflow."""
    c = Case(gpu, [300, 40], [1, 20], 1, 128, 64, seed=8, big=16.0)
    run(llk, c, c.queries(2, sigma=16.0), 1.0)


def test_the_same_every_time_and_in_a_graph(llk, gpu):
    c = Case(gpu, [500, 90, 130], [1, 1, 1], 4, 128, 32, seed=9)
    q = _dev(gpu, c.queries(16), gpu.bfloat16)
    pool, table, lens, _ = c.dev()
    first = None
    for _ in range(3):
        w = gpu.zeros(pool.shape[0], 4, 32, device="cuda")
        llk.kv4_attention(q, pool, table, lens, weights=w)
        first = w if first is None else first
        assert gpu.equal(w, first)
    side = gpu.cuda.Stream()
    scratch = gpu.empty(llk.describe_kv4_attention(q, pool, table, lens, weigh=True)["workspace_bytes"],
                        dtype=gpu.uint8, device="cuda")
    gpu.cuda.synchronize()
    w = gpu.zeros_like(first)
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        out = llk.kv4_attention(q, pool, table, lens, weights=w, scratch=scratch)
    want = gpu.zeros_like(first)
    for _ in range(4):
        lens -= 3
        q.copy_(gpu.randn(*q.shape, device="cuda"))
        graph.replay()
        got = llk.kv4_attention(q, pool, table, lens, weights=want)
        assert gpu.equal(out, got) and gpu.equal(w, want)


def test_weights_in_a_larger_pool(llk, gpu):
    """A layer's marks as a slice of [pages, layers, heads, page_size]: the other
    layers' stay."""
    c = Case(gpu, [100, 33], [1, 1], 2, 64, 32, seed=10)
    q = _dev(gpu, c.queries(4), gpu.bfloat16)
    pool, table, lens, _ = c.dev()
    every = gpu.full((pool.shape[0], 3, 2, 32), 7.0, device="cuda")
    alone = gpu.full((pool.shape[0], 2, 32), 7.0, device="cuda")
    llk.kv4_attention(q, pool, table, lens, weights=every[:, 1], decay=0.25)
    llk.kv4_attention(q, pool, table, lens, weights=alone, decay=0.25)
    assert gpu.equal(every[:, 1], alone)
    assert (every[:, 0] == 7).all() and (every[:, 2] == 7).all()
    with pytest.raises(ValueError, match="page_size"):
        llk.kv4_attention(q, pool, table, lens, weights=gpu.zeros(pool.shape[0], 2, 16, device="cuda"))
    with pytest.raises(ValueError, match="contiguous"):
        llk.kv4_attention(q, pool, table, lens, weights=gpu.zeros(pool.shape[0], 4, 32, device="cuda")[:, ::2])


@pytest.mark.parametrize("heads,page", [(1, 16), (5, 64), (40, 32)])
def test_written_marks(llk, gpu, heads, page):
    lens, news = [1, 40, 0, 129, 16, 77], [1, 17, 0, 128, 16, 3]
    c = Case(gpu, lens, news, heads, 64, page, seed=heads)
    c.table[1, 0] = -1  # some of the tokens have no place
    pool, table, lens_d, starts = c.dev()
    shape = (pool.shape[0], heads, page)
    kv = gpu.randn(c.tokens, heads, 64, device="cuda").bfloat16()
    at = gpu.randint(-1000, 1000, (c.tokens,), device="cuda").int()
    for positions in (None, at):
        w, p = gpu.full(shape, 5.0, device="cuda"), gpu.full(shape, -7, dtype=gpu.int32, device="cuda")
        ww, wp = w.cpu().numpy().copy(), p.cpu().numpy().copy()
        same = pool.clone()
        llk.kv4_write(kv, kv, pool, table, lens_d, starts=starts, weights=w, positions=p, at=positions)
        llk.kv4_write(kv, kv, same, table, lens_d, starts=starts)
        assert gpu.equal(pool, same)
        for s in range(len(lens)):
            for i, (pos, page_id) in enumerate(ref.places(shape[0], page, c.table, c.lens, c.starts, s)):
                if page_id < 0:
                    continue
                ww[page_id, :, pos % page] = 0
                wp[page_id, :, pos % page] = pos if positions is None else int(at[int(c.starts[s]) + i])
        assert np.array_equal(w.cpu().numpy(), ww) and np.array_equal(p.cpu().numpy(), wp)
    # either alone
    w = gpu.full(shape, 5.0, device="cuda")
    llk.kv4_write(kv, kv, pool, table, lens_d, starts=starts, weights=w)
    assert np.array_equal(w.cpu().numpy(), ww)
    p = gpu.full(shape, -7, dtype=gpu.int32, device="cuda")
    llk.kv4_write(kv, kv, pool, table, lens_d, starts=starts, positions=p, at=at)
    assert np.array_equal(p.cpu().numpy(), wp)
    with pytest.raises(ValueError, match="at"):
        llk.kv4_write(kv, kv, pool, table, lens_d, starts=starts, at=at)


@pytest.mark.parametrize("news,group", [([1, 1, 1], 4), ([1, 1, 1], 20), ([3, 2, 1], 2), ([140, 200, 129], 2)])
def test_a_hint_below_the_lengths(llk, gpu, news, group):
    """Any max_len gives right sums: scores are kept of the first keys only, or fewer
    workgroups go round."""
    lens = [n + extra for n, extra in zip(news, (700, 30, 1500))]
    c = Case(gpu, lens, news, 2, 64, 32, seed=group)
    q = c.queries(2 * group)
    for hint in (1, 256, 300, 1024):
        run(llk, c, q, 0.5, max_len=hint)
        run(llk, c, q, 1.0, max_len=hint, window=400, sinks=10)


def test_single_tokens_given_by_starts(llk, gpu):
    """With `starts` no scores are kept; the sums are the same."""
    c = Case(gpu, [300, 41, 513], [1, 1, 1], 2, 128, 16, seed=2)
    pool, table, lens, _ = c.dev()
    q = _dev(gpu, c.queries(8), gpu.bfloat16)
    got = []
    for starts in (None, gpu.arange(4, device="cuda").int()):
        w = gpu.zeros(pool.shape[0], 2, 16, device="cuda")
        llk.kv4_attention(q, pool, table, lens, starts=starts, weights=w)
        got.append(w)
    # each within this file's bound, its keys being below 6
    near = 144 * 2.0 ** -22 * 128 ** -0.5 * 6 * float(q.float().abs().sum(-1).max()) + 2.0 ** -18
    assert ((got[0] - got[1]).abs() <= 2 * near * gpu.maximum(*got)).all()
    rows = gpu.stack(got).double().sum((1, 3))
    assert ((rows - 3 * 4).abs() <= 12 * near).all()  # 3 tokens, 4 query heads, a sum of 1 each


def test_weights_beyond_32_bits(llk, gpu):
    """Pages of the cache and of the marks at offsets beyond 2^32 bytes."""
    D, size = 64, 16
    c = Case(gpu, [40, 20], [1, 1], 2, D, size, seed=4)
    q = _dev(gpu, c.queries(4), gpu.bfloat16)
    pool, table, lens, _ = c.dev()
    pages = pool.shape[0]
    step = ((1 << 32) + 4096) // (pages - 1) // 16 * 16 + 16
    far = gpu.empty(pages * step, dtype=gpu.uint8, device="cuda").as_strided(
        pool.shape, (step, pool.shape[2], 1))
    far.copy_(pool)
    marks = gpu.empty(pages * step // 4, dtype=gpu.float32, device="cuda").as_strided(
        (pages, 2, size), (step // 4, size, 1))
    marks.fill_(1.0)
    near = gpu.ones(pages, 2, size, device="cuda")
    a = llk.kv4_attention(q, pool, table, lens, weights=near)
    b = llk.kv4_attention(q, far, table, lens, weights=marks)
    assert gpu.equal(a, b) and gpu.equal(near, marks)
    k = gpu.randn(2, 2, D, device="cuda").bfloat16()
    llk.kv4_write(k, k, pool, table, lens, weights=near)
    llk.kv4_write(k, k, far, table, lens, weights=marks)
    assert gpu.equal(pool, far) and gpu.equal(near, marks)
    for x, w in ((pool, near), (far, marks)):
        _, source = llk.kv4_evict_plan(w, table, lens, 17)
        llk.kv4_evict(x, table, source, head_dim=D, weights=w)
    assert gpu.equal(pool, far) and gpu.equal(near, marks)


@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 0), (33, 4), (256, 40)])
def test_scores_that_a_window_leaves_unwritten(llk, gpu, window, sinks):
    """A workspace of NaN: what the attention did not write of it has no part in the
    weights, or in the result."""
    D, group = 64, 4
    c = Case(gpu, [1, 700, 1500, 33], [1, 1, 1, 1], 2, D, 16, seed=window)
    q = _dev(gpu, c.queries(2 * group), gpu.bfloat16)
    pool, table, lens, _ = c.dev()
    kw = dict(window=window, sinks=sinks, max_len=1500)
    need = llk.describe_kv4_attention(q, pool, table, lens, weigh=True, **kw)["workspace_bytes"]
    got = []
    for fill in (0xff, 0x00):
        scratch = gpu.full((need,), fill, dtype=gpu.uint8, device="cuda")
        weights = gpu.zeros(pool.shape[0], 2, 16, device="cuda")
        out = llk.kv4_attention(q, pool, table, lens, weights=weights, scratch=scratch, **kw)
        got.append((out, weights))
    assert gpu.equal(got[0][0], got[1][0]) and gpu.equal(got[0][1], got[1][1])
    assert got[0][1].isfinite().all()
    run(llk, c, c.queries(2 * group), 0.5, window=window, sinks=sinks, max_len=1500)
