"""What the marks of a cache's slots, the attention that adds its weights up and the
eviction refuse, before any device work, and the launches they plan."""
from __future__ import annotations

import pytest

from test_decoder_cpu import BAD_CACHES, FAKE, _batch, _cache, _kv, _par


@pytest.fixture()
def L(llk):
    return llk.lib()


def _marks(**kw):
    from dslcompiler_amd._lib import Kv4Marks
    d = dict(weights=FAKE, positions=FAKE, weights_stride=2 * 64, positions_stride=2 * 64)
    d.update(kw)
    return Kv4Marks(**d)


def _params(keep=100, recent=0, first=0):
    from dslcompiler_amd._lib import EvictParams
    return EvictParams(keep, recent, first)


BAD_MARKS = [(dict(weights=FAKE + 2), -4), (dict(positions=FAKE + 1), -4),
             (dict(weights_stride=127), -4), (dict(positions_stride=0), -4),
             (dict(weights_stride=-128), -4)]


def test_write_refusals(L):
    k = _kv()

    def call(cache=None, batch=None, marks=None, at=None):
        return L.llk_kv4_write_marked(k, k, cache or _cache(), batch or _batch(), marks, at, None)

    assert call() == -1 and b"marks" in L.llk_last_error()
    for bad, code in BAD_MARKS:
        assert call(marks=_marks(**bad)) == code, bad
    for bad, code in BAD_CACHES:
        assert call(cache=_cache(**bad), marks=_marks()) == code, bad
    assert L.llk_kv4_write_marked(None, k, _cache(), _batch(), _marks(), None, None) == -1
    # no tokens: nothing to do, with either mark alone or none
    e = _kv(T=0)
    b = _batch(tokens=0, sequences=0)
    for m in (_marks(), _marks(weights=None), _marks(positions=None),
              _marks(weights=None, positions=None)):
        assert L.llk_kv4_write_marked(e, e, _cache(), b, m, FAKE, None) == 0


def test_attention_refusals(L):
    q = _kv(H=8)

    def call(marks=None, decay=1.0, cache=None, q_=q, par=None, **b):
        return L.llk_kv4_attention_weigh(q_, cache or _cache(), _batch(**b), par or _par(), marks,
                                         decay, q, None)

    assert call() == -1 and b"marks" in L.llk_last_error()
    assert call(_marks(weights=None)) == -1 and b"weights" in L.llk_last_error()
    for bad, code in BAD_MARKS:
        assert call(_marks(**bad)) == code, bad
    for bad, code in BAD_CACHES:
        assert call(_marks(), cache=_cache(**bad)) == code, bad
    for decay in (-0.5, float("nan"), float("inf")):
        assert call(_marks(), decay) == -1 and b"decay" in L.llk_last_error()
    assert call(_marks(), q_=_kv(H=7)) == -2
    assert call(_marks(), par=_par(scale=0.0)) == -1
    assert call(_marks(), max_len=-1) == -1
    assert call(_marks(), lens=None) == -1
    n = 1 << 21  # sequences of 2 heads
    many = _kv(T=n, H=8)
    assert L.llk_kv4_attention_weigh(many, _cache(), _batch(sequences=n, tokens=n), _par(), _marks(),
                                     1.0, many, None) == -2
    assert b"too many" in L.llk_last_error()
    e = _kv(T=0, H=8)
    assert L.llk_kv4_attention_weigh(e, _cache(), _batch(tokens=0, sequences=0), _par(), _marks(), 1.0,
                                     e, None) == 0


def test_a_result_over_the_queries(L):
    """The weights are computed from q once more, after the result is there."""
    q = _kv(H=8)

    def call(out, **b):
        return L.llk_kv4_attention_weigh(q, _cache(), _batch(**b), _par(), _marks(), 1.0, out, None)

    assert call(q) == -1 and b"out" in L.llk_last_error()
    assert call(_kv(H=8, s0=4096)) == -1  # the same memory at other strides
    assert call(_kv(H=8, data=2 * FAKE)) != -1  # (no device here)


def test_attention_plans(L):
    """The rows' statistics, and of single tokens the scores up to 512 MiB, come on
    top of the attention's own workspace."""
    from dslcompiler_amd._lib import AttentionPlan

    def plans(T, H, **b):
        plain, weigh = AttentionPlan(), AttentionPlan()
        args = (_kv(T=T, H=H), _cache(), _batch(**b), _par())
        assert L.llk_kv4_attention_describe(*args, plain) == 0
        assert L.llk_kv4_attention_weigh_describe(*args, weigh) == 0
        assert weigh.launches == plain.launches + 1 and weigh.splits == plain.splits
        up = lambda n: -(-n // 256) * 256
        return weigh.workspace_bytes - up(plain.workspace_bytes) - up(T * H * 8)

    one = dict(sequences=1, tokens=1, table_pages=2048, table_stride=2048)
    assert plans(1, 8, **one) == 8 * 2048 * 64 * 4
    assert plans(1, 8, max_len=100, **one) == 8 * 256 * 4
    assert plans(1, 40, **one) == 0  # 20 query heads of a key head
    many = dict(sequences=200, tokens=200, table_pages=2048, table_stride=2048)
    assert plans(200, 32, **many) == 0  # 3.4 GB
    assert plans(200, 32, max_len=5000, **many) == 200 * 32 * 5120 * 4
    assert plans(200, 32, starts=FAKE, **many) == 0
    plan = AttentionPlan()
    e = _kv(T=0, H=8)
    assert L.llk_kv4_attention_weigh_describe(e, _cache(), _batch(tokens=0, sequences=0), _par(),
                                              plan) == 0
    assert plan.workspace_bytes == 0 and plan.launches == 0
    assert L.llk_kv4_attention_weigh_describe(_kv(H=7), _cache(), _batch(), _par(), plan) == -2


def test_plan_refusals(L):
    def call(marks=None, pages=10, heads=2, size=64, params=None, lens=2 * FAKE, source=FAKE, **b):
        return L.llk_kv4_evict_plan(marks or _marks(), pages, heads, size, _batch(**b),
                                    params or _params(), lens, source, None)

    assert L.llk_kv4_evict_plan(None, 10, 2, 64, _batch(), _params(), FAKE, FAKE, None) == -1
    assert L.llk_kv4_evict_plan(_marks(), 10, 2, 64, None, _params(), FAKE, FAKE, None) == -1
    assert L.llk_kv4_evict_plan(_marks(), 10, 2, 64, _batch(), None, FAKE, FAKE, None) == -1
    assert call(lens=None) == -1 and call(source=None) == -1
    assert call(lens=FAKE) == -1 and b"replace" in L.llk_last_error()
    for bad, code in BAD_MARKS:
        assert call(_marks(**bad)) == code, bad
    for kw in (dict(pages=0), dict(pages=1 << 31), dict(heads=0), dict(heads=70000), dict(size=8),
               dict(size=48), dict(size=8192), dict(tokens=4), dict(sequences=-1, tokens=-1)):
        assert call(**kw) == -2, kw
    assert call(table=None) == -1 and call(**{"table_stride": -1}) == -4
    for p in (dict(keep=0), dict(keep=-1), dict(keep=(1 << 30) + 1)):
        assert call(params=_params(**p)) == -2, p
    top = (1 << 63) - 1
    for p in (dict(recent=-1), dict(first=-1), dict(recent=101), dict(first=101),
              dict(recent=50, first=51), dict(recent=top, first=top), dict(recent=100, first=top)):
        assert call(params=_params(**p)) == -1, p
    assert call(_marks(positions=None), params=_params(recent=1)) == -1
    assert b"positions" in L.llk_last_error()
    assert call(_marks(weights=None)) == -1
    assert call(sequences=1 << 21, tokens=1 << 21) == -2 and b"too many" in L.llk_last_error()
    assert call(sequences=0, tokens=0) == 0


@pytest.mark.parametrize("sequences", [1, 2, 7])
def test_new_lengths_apart_from_the_old_ones(L, sequences):
    """Every head's workgroup reads batch.lens while the new lengths are written:
    a shifted view of them is refused as they themselves are."""
    def call(lens):
        return L.llk_kv4_evict_plan(_marks(), 10, 2, 64, _batch(sequences=sequences, tokens=sequences),
                                    _params(), lens, 2 * FAKE, None)

    for shift in range(1 - sequences, sequences):
        assert call(FAKE + 4 * shift) == -1 and b"replace" in L.llk_last_error(), shift
    for shift in (-sequences, sequences):  # right beside them
        assert call(FAKE + 4 * shift) != -1, shift


def test_move_refusals(L):
    def call(cache=None, marks=None, keep=10, source=FAKE, lens=None, **b):
        return L.llk_kv4_evict(cache or _cache(), _batch(**b), source, keep, marks, lens, None)

    for bad, code in BAD_CACHES:
        assert call(_cache(**bad)) == code, bad
    for bad, code in BAD_MARKS:
        assert call(marks=_marks(**bad)) == code, bad
    assert L.llk_kv4_evict(_cache(), None, FAKE, 10, None, None, None) == -1
    assert L.llk_kv4_evict(None, _batch(), FAKE, 10, None, None, None) == -1
    assert call(source=None) == -1 and b"source" in L.llk_last_error()
    assert call(table=None) == -1
    for keep in (0, -1, (1 << 30) + 1):
        assert call(keep=keep) == -2, keep
    assert call(sequences=-1, tokens=-1) == -2
    assert call(sequences=1 << 21, tokens=1 << 21) == -2 and b"too many" in L.llk_last_error()
    assert call(sequences=0, tokens=0, source=None) == 0


def test_python_refusals(llk):
    """The Python layer wants device tensors of the right type and shape."""
    import torch
    w, p = llk.kv4_marks(4, 2, 64, device="cpu")
    assert w.shape == p.shape == (4, 2, 64) and w.dtype == torch.float32 and p.dtype == torch.int32
    cache = llk.kv4_cache(4, 2, 64, 128, device="cpu")
    t, n = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    for call in (lambda: llk.kv4_write(x, x, cache, t, n, weights=w),
                 lambda: llk.kv4_attention(x, cache, t, n, weights=w),
                 lambda: llk.kv4_evict_plan(w, t, n, 4),
                 lambda: llk.kv4_evict(cache, t, torch.zeros(1, 2, 4, dtype=torch.int32), head_dim=128)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
