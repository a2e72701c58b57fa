"""Which slots of the cache stay, and the cache moved together: whole numbers and
bytes, equal to a plain implementation's."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def plan(weights, positions, table, lens, keep, recent, first):
    """(new lens, source) by sorting."""
    pages, heads, size = weights.shape
    source = np.tile(np.arange(keep, dtype=np.int32), (len(lens), heads, 1))
    for s, length in enumerate(lens):
        n = min(max(int(length), 0), table.shape[1] * size)
        if n <= keep:
            continue
        j = np.arange(n)
        page, off = table[s, j // size], j % size
        here = (page >= 0) & (page < pages)
        for h in range(heads):
            w = np.where(here, weights[np.where(here, page, 0), h, off], 0).astype(np.float64)
            rank = np.where(np.isnan(w), -2, 0)  # below -infinity
            w = np.where(np.isnan(w), 0, w)
            if recent or first:
                pos = positions[np.where(here, page, 0), h, off].astype(np.int64)
                last = pos[here].max() if here.any() else -2 ** 31
                rank = np.where((pos > last - recent) | (pos < first), 1, rank)
                w = np.where(rank == 1, 0, w)
            rank = np.where(here, rank, -3)
            w = np.where(here, w, 0)
            stay = np.sort(np.lexsort((j, -w, -rank))[:keep])
            source[s, h, np.setdiff1d(np.arange(keep), stay)] = stay[stay >= keep]
    return np.minimum(lens, keep), source


class Pool:
    def __init__(self, torch, lens, heads, page, seed, spare=2, ties=False, wide=0):
        rng = np.random.default_rng(seed)
        need = [-(-max(n, 0) // page) for n in lens]
        total = sum(need) + spare
        order = rng.permutation(total)
        self.table = np.full((len(lens), max(max(need), 1) + wide), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (total, heads, page)
        self.weights = rng.integers(0, 5, shape).astype(np.float32) if ties else \
            np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
        self.positions = rng.integers(0, 1 << 20, shape).astype(np.int32)
        self.lens, self.torch, self.rng = np.array(lens, np.int32), torch, rng

    def dev(self):
        return tuple(self.torch.from_numpy(x).cuda()
                     for x in (self.weights, self.positions, self.table, self.lens))

    def check(self, llk, keep, recent=0, first=0, with_positions=True, **kw):
        w, p, t, n = self.dev()
        before = n.clone()
        lens, source = llk.kv4_evict_plan(w, t, n, keep, positions=p if with_positions else None,
                                          recent=recent, first=first, **kw)
        want = plan(self.weights, self.positions, self.table, self.lens, keep, recent, first)
        assert np.array_equal(lens.cpu().numpy(), want[0])
        assert np.array_equal(source.cpu().numpy(), want[1])
        assert self.torch.equal(n, before)
        return source


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("keep", [1, 2, 15, 64, 100, 1000, 1023, 1025])
def test_plan(llk, gpu, keep, page, ties):
    lens = [0, 1, keep - 1, keep, keep + 1, keep + 70, 2 * keep + 5, 3000, -4]
    pool = Pool(gpu, lens, 3, page, keep, ties=ties)
    pool.check(llk, keep, with_positions=False)
    pool.check(llk, keep, max_len=3000)
    if keep > 2:
        pool.check(llk, keep, recent=keep // 2, first=1)
        pool.check(llk, keep, recent=keep, first=0)
        pool.check(llk, keep, recent=0, first=keep, max_len=3000)


@pytest.mark.parametrize("n,keep", [(20000, 700), (20000, 19990), (70001, 33000), (9000, 4096),
                                    (16384, 1024), (16385, 1), (140000, 70000)])
def test_long_sequences(llk, gpu, n, keep):
    for ties in (False, True):
        pool = Pool(gpu, [n, n // 3], 2, 256, n + keep, ties=ties)
        pool.check(llk, keep, recent=min(keep, 128) - keep // 64 % 2, first=0, max_len=n)
        pool.check(llk, keep, with_positions=False)


def test_weights_that_are_not_finite_and_zeros(llk, gpu):
    pool = Pool(gpu, [300, 200], 2, 32, 5)
    flat = pool.weights.reshape(-1)
    flat[pool.rng.permutation(flat.size)[:flat.size // 2]] = \
        pool.rng.choice([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0, 1e-45, -1e-45, 3e38],
                        flat.size // 2).astype(np.float32)
    for keep in (1, 50, 120, 199, 299):
        pool.check(llk, keep)
        pool.check(llk, keep, recent=min(keep, 9))


def test_equal_weights_keep_the_lowest_slots(llk, gpu):
    pool = Pool(gpu, [5000], 2, 64, 6)
    pool.weights[:] = 1.0
    source = pool.check(llk, 3000)
    assert gpu.equal(source[0, 0], gpu.arange(3000, device="cuda").int())


def test_absent_pages_and_lengths_beyond_the_table(llk, gpu):
    pool = Pool(gpu, [300, 300, 300], 2, 32, 7)
    pool.table[0, 2], pool.table[1, 0], pool.table[1, 9] = -1, 1 << 20, -5
    pool.table[2] = -1  # no page at all
    pool.lens[0] = 100000  # whole table
    for keep in (10, 150, 250, 280, 319):
        pool.check(llk, keep)
        pool.check(llk, keep, recent=7, first=3)
    pool.check(llk, 5000)  # more than there are


def test_extreme_positions(llk, gpu):
    pool = Pool(gpu, [200], 2, 16, 8)
    pool.positions[:] = pool.rng.choice([-2 ** 31, 2 ** 31 - 1, 0, 5, 2 ** 31 - 2, -1], pool.positions.shape)
    for recent, first in ((1, 0), (2, 0), (0, 3), (50, 50)):
        pool.check(llk, 100, recent=recent, first=first)


def moved(pool, table, source, keep, size, D, marks):
    """The pool (and marks) after the moves, in numpy."""
    pool = pool.copy()
    marks = [m.copy() for m in marks]
    tiles = pool.reshape(*pool.shape[:2], -1, 17 * D)
    old, old_marks = tiles.copy(), [m.copy() for m in marks]
    for s in range(table.shape[0]):
        for h in range(pool.shape[1]):
            for to in range(keep):
                of = int(source[s, h, to])
                if of == to or of < keep or max(of, to) >= table.shape[1] * size:
                    continue
                a, b = int(table[s, to // size]), int(table[s, of // size])
                if not (0 <= a < pool.shape[0] and 0 <= b < pool.shape[0]):
                    continue
                x, y = to % size, of % size
                for block in range(D // 16):
                    tiles[a, h, x // 16, block * 256 + x % 16 * 16:][:16] = \
                        old[b, h, y // 16, block * 256 + y % 16 * 16:][:16]
                    tiles[a, h, x // 16, 16 * D + block * 16 + x % 16] = \
                        old[b, h, y // 16, 16 * D + block * 16 + y % 16]
                for m, o in zip(marks, old_marks):
                    m[a, h, x] = o[b, h, y]
    return pool, marks


@pytest.mark.parametrize("D,heads,size", [(64, 3, 16), (128, 2, 64), (256, 1, 32)])
def test_moves(llk, gpu, D, heads, size):
    p = Pool(gpu, [300, 70, 129, 1000], heads, size, D)
    w, pos, table, lens = p.dev()
    data = p.rng.integers(0, 256, (w.shape[0], heads, size // 16 * 17 * D)).astype(np.uint8)
    for keep in (65, 128, 260):
        _, source = llk.kv4_evict_plan(w, table, lens, keep, positions=pos, recent=30, first=2)
        for given in ((None, None), (w, None), (w, pos)):
            cache = gpu.from_numpy(data.copy()).cuda()
            marks = [None if m is None else m.clone() for m in given]
            cut = lens.clone()
            llk.kv4_evict(cache, table, source, head_dim=D, weights=marks[0], positions=marks[1],
                          lens=cut)
            assert gpu.equal(cut, lens.clamp(max=keep))
            want, wm = moved(data, p.table, source.cpu().numpy(), keep, size, D,
                             [m.cpu().numpy() for m in given if m is not None])
            assert np.array_equal(cache.cpu().numpy(), want)
            for m, x in zip([m for m in marks if m is not None], wm):
                assert np.array_equal(m.cpu().numpy(), x)


def test_maps_that_are_no_plan(llk, gpu):
    """Sources out of range, on absent pages or below keep move nothing."""
    D, size, keep = 64, 16, 40
    p = Pool(gpu, [200], 2, size, 9)
    p.table[0, 5], p.table[0, 1] = -1, 1 << 30
    w, pos, table, lens = p.dev()
    data = p.rng.integers(0, 256, (w.shape[0], 2, 17 * D)).astype(np.uint8)
    source = np.tile(np.arange(keep, dtype=np.int32), (1, 2, 1))
    source[0, 0, :8] = [-1, 5, 2 ** 31 - 1, 100000, 85, 100, 207, 208]
    source[0, 1, 14:20] = [150, 151, 152, 153, -2 ** 31, 39]
    cache = gpu.from_numpy(data.copy()).cuda()
    llk.kv4_evict(cache, table, gpu.from_numpy(source).cuda(), head_dim=D, weights=w, positions=pos)
    want, (ww, wp) = moved(data, p.table, source, keep, size, D, [p.weights, p.positions])
    assert np.array_equal(cache.cpu().numpy(), want)
    assert np.array_equal(w.cpu().numpy(), ww) and np.array_equal(pos.cpu().numpy(), wp)


def test_layers_of_one_pool_streams_and_graph(llk, gpu):
    """Cache and marks as slices of a pool of layers; a captured plan and move
    replays with new weights, lengths and pages."""
    D, size, keep, layers = 64, 16, 50, 3
    p = Pool(gpu, [120, 49, 90], 2, size, 10)
    w, pos, table, lens = p.dev()
    pages = w.shape[0]
    every = gpu.randint(0, 256, (pages, layers, 2, 17 * D), device="cuda").to(gpu.uint8)
    ew = gpu.rand(pages, layers, 2, size, device="cuda")
    ep = gpu.randint(0, 999, (pages, layers, 2, size), device="cuda").int()
    side = gpu.cuda.Stream()
    gpu.cuda.synchronize()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        new, source = llk.kv4_evict_plan(ew[:, 1], table, lens, keep, positions=ep[:, 1], recent=9)
        llk.kv4_evict(every[:, 1], table, source, head_dim=D, weights=ew[:, 1], positions=ep[:, 1],
                      lens=lens)
    for n in range(4):
        lens.copy_(gpu.tensor([120 - n, 49, 90 + n], device="cuda"))
        ew.copy_(gpu.rand(*ew.shape, device="cuda"))
        table.copy_(table.flip(0) if n == 2 else table)
        before = every.cpu().numpy(), ew.cpu().numpy(), ep.cpu().numpy()
        old = lens.cpu().numpy()
        graph.replay()
        t = table.cpu().numpy()
        want_len, want = plan(before[1][:, 1], before[2][:, 1], t, old, keep, 9, 0)
        assert np.array_equal(new.cpu().numpy(), want_len) and gpu.equal(lens, new)
        assert np.array_equal(source.cpu().numpy(), want)
        data, (mw, mp) = moved(before[0][:, 1], t, want, keep, size, D,
                               [before[1][:, 1], before[2][:, 1]])
        for got, old_all, one in ((every, before[0], data), (ew, before[1], mw), (ep, before[2], mp)):
            expect = old_all.copy()
            expect[:, 1] = one
            assert np.array_equal(got.cpu().numpy(), expect)
    # on a stream of the caller's
    a = llk.kv4_evict_plan(ew[:, 1], table, gpu.full_like(lens, 100), keep)
    gpu.cuda.synchronize()
    b = llk.kv4_evict_plan(ew[:, 1], table, gpu.full_like(lens, 100), keep, stream=gpu.cuda.current_stream())
    assert gpu.equal(a[1], b[1])


def test_no_sequences(llk, gpu):
    p = Pool(gpu, [10], 2, 16, 11)
    w, pos, table, lens = p.dev()
    new, source = llk.kv4_evict_plan(w, table[:0], lens[:0], 4)
    assert new.shape == (0,) and source.shape == (0, 2, 4)
    cache = gpu.zeros(w.shape[0], 2, 17 * 64, dtype=gpu.uint8, device="cuda")
    llk.kv4_evict(cache, table[:0], source, head_dim=64)
    llk.kv4_evict(cache, table[:, :0], gpu.zeros(1, 2, 4, dtype=gpu.int32, device="cuda"), head_dim=64)


def test_refusals(llk, gpu):
    p = Pool(gpu, [40], 2, 16, 12)
    w, pos, table, lens = p.dev()
    for kw in (dict(keep=0), dict(keep=-1), dict(keep=4, recent=5), dict(keep=4, recent=3, first=2),
               dict(keep=4, recent=-1), dict(keep=1 << 31)):
        with pytest.raises((llk.LLKError, RuntimeError)):
            llk.kv4_evict_plan(w, table, lens, positions=pos, **kw)
    with pytest.raises(llk.LLKError, match="positions"):
        llk.kv4_evict_plan(w, table, lens, 4, recent=1)
    with pytest.raises(llk.LLKError, match="replace"):
        llk.kv4_evict_plan(w, table, lens, 4, lens_out=lens)
    with pytest.raises(ValueError, match="positions"):
        llk.kv4_evict_plan(w, table, lens, 4, positions=pos[:, :1])
    cache = gpu.zeros(w.shape[0], 2, 17 * 64, dtype=gpu.uint8, device="cuda")
    with pytest.raises(ValueError, match="source"):
        llk.kv4_evict(cache, table, gpu.zeros(1, 3, 4, dtype=gpu.int32, device="cuda"), head_dim=64)


@pytest.mark.parametrize("hint", [1, 100, 2048, 3000, 9000])
def test_a_hint_below_the_lengths(llk, gpu, hint):
    """Any max_len gives the same plan."""
    pool = Pool(gpu, [2000, 5000, 2049, 8193, 100], 2, 64, hint, ties=hint > 1000)
    for keep in (60, 2000, 4000):
        pool.check(llk, keep, recent=20, first=4, max_len=hint)
        pool.check(llk, keep, with_positions=False, max_len=hint)


def test_lengths_are_cut_without_pages(llk, gpu):
    cache = gpu.zeros(3, 2, 17 * 64, dtype=gpu.uint8, device="cuda")
    table, source = gpu.zeros(2, 0, dtype=gpu.int32, device="cuda"), \
        gpu.zeros(2, 2, 5, dtype=gpu.int32, device="cuda")
    lens = gpu.tensor([9, 3], dtype=gpu.int32, device="cuda")
    new, plan_source = llk.kv4_evict_plan(gpu.zeros(3, 2, 16, device="cuda"), table, lens, 5)
    assert new.tolist() == [5, 3]
    assert gpu.equal(plan_source, gpu.arange(5, device="cuda").int().expand(2, 2, 5))
    llk.kv4_evict(cache, table, source, head_dim=64, lens=lens)
    assert lens.tolist() == [5, 3] and (cache == 0).all()


def test_new_lengths_in_a_shifted_view(llk, gpu):
    """Lengths and new lengths in one buffer: refused where they overlap."""
    p = Pool(gpu, [40, 30, 20], 2, 16, 13)
    w, pos, table, lens = p.dev()
    both = gpu.zeros(7, dtype=gpu.int32, device="cuda")
    old = both[2:5]
    old.copy_(lens)
    for at in (0, 1, 2, 3, 4):
        with pytest.raises(llk.LLKError, match="replace"):
            llk.kv4_evict_plan(w, table, old, 25, lens_out=both[at:at + 3])
    assert both.tolist() == [0, 0, 40, 30, 20, 0, 0]
    six = gpu.cat([lens, lens])
    new, source = llk.kv4_evict_plan(w, table, six[:3], 25, lens_out=six[3:])
    assert new.tolist() == [25, 25, 20] and six[:3].tolist() == [40, 30, 20]
    assert gpu.equal(source, llk.kv4_evict_plan(w, table, lens, 25)[1])


def test_a_stream_of_the_callers(llk, gpu):
    """Plan and move on another stream, which is behind, while the current one goes on;
    a captured step whose two calls are given the capturing stream."""
    D, size, keep = 64, 16, 50
    p = Pool(gpu, [120, 49, 90], 2, size, 14)
    w, pos, table, lens = p.dev()
    data = p.rng.integers(0, 256, (w.shape[0], 2, 17 * D)).astype(np.uint8)
    cache = gpu.from_numpy(data.copy()).cuda()
    want_len, want = plan(p.weights, p.positions, p.table, p.lens, keep, 9, 2)
    want_cache, (want_w, want_pos) = moved(data, p.table, want, keep, size, D, [p.weights, p.positions])
    big = [gpu.zeros(1 << 28, dtype=gpu.uint8, device="cuda") for _ in range(2)]
    side = gpu.cuda.Stream()
    held = [t.clone() for t in (cache, w, pos, lens)]
    new = gpu.full_like(lens, -1)

    def step():
        _, source = llk.kv4_evict_plan(w, table, lens, keep, positions=pos, recent=9, first=2,
                                       lens_out=new, stream=side)
        llk.kv4_evict(cache, table, source, head_dim=D, weights=w, positions=pos, lens=lens, stream=side)
        return source

    def check(source):
        assert np.array_equal(source.cpu().numpy(), want)
        assert np.array_equal(new.cpu().numpy(), want_len) and gpu.equal(new, lens)
        for got, expect in ((cache, want_cache), (w, want_w), (pos, want_pos)):
            assert np.array_equal(got.cpu().numpy(), expect)

    gpu.cuda.synchronize()
    with gpu.cuda.stream(side):
        for n in range(100):  # about 10 ms of copies
            big[n % 2].copy_(big[1 - n % 2])
        copied = gpu.cuda.Event()
        copied.record()
    source = step()
    same = bool((new == -1).all())
    if not copied.query():  # nothing of it ran on the current stream
        assert same
    gpu.cuda.synchronize()
    check(source)
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        source = step()
    for _ in range(3):
        for t, was in zip((cache, w, pos, lens), held):
            t.copy_(was)
        new.fill_(-1)
        graph.replay()
        check(source)
