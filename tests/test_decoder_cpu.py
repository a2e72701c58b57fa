"""What the decoder block's operators refuse, before any device work, and the
launches they plan (host only: the C ABI with pointers that are never read)."""
from __future__ import annotations

import ctypes as C

import pytest

FAKE = 1 << 20  # an aligned address


@pytest.fixture()
def L(llk):
    return llk.lib()


def _t2(rows, cols, stride=None, data=FAKE, one=1):
    from dslcompiler_amd._lib import Tensor2D
    return Tensor2D(data, rows, cols, cols if stride is None else stride, one)


def _norm(L, y, h, ho, o, **kw):
    from dslcompiler_amd._lib import BlockNormParams
    p = dict(y_dtype=0, residual_dtype=0, out_dtype=0, weight_dtype=0, post_weight=None,
             pre_weight=FAKE, gate=_t2(0, 0, data=None), residual_scale=1.0, eps=1e-6,
             weight_offset=0.0)
    p.update(kw)
    return L.llk_block_norm(y, h, ho, o, BlockNormParams(**p), None)


def test_block_norm_refusals(L):
    t = _t2(4, 64)
    assert _norm(L, t, None, t, t) == -1
    assert _norm(L, t, t, t, None) == -1
    assert L.llk_block_norm(t, t, t, t, None, None) == -1
    assert _norm(L, t, t, None, t) == -1                      # y without residual_out
    assert _norm(L, None, t, None, t, post_weight=FAKE) == -1  # a norm of no y
    assert _norm(L, None, t, None, t, gate=t) == -1
    assert _norm(L, t, t, t, t, pre_weight=None) == -1
    assert _norm(L, t, t, t, t, eps=-1.0) == -1
    assert _norm(L, t, t, t, t, eps=float("nan")) == -1
    assert _norm(L, _t2(4, 65), t, t, t) == -2
    assert _norm(L, t, t, t, _t2(5, 64)) == -2
    assert _norm(L, t, t, t, t, gate=_t2(3, 64)) == -2
    assert _norm(L, None, _t2(1, 0), None, _t2(1, 0)) == -2
    big = _t2(1, 32769)
    assert _norm(L, big, big, big, big) == -2
    assert b"32768" in L.llk_last_error()
    for k in ("y_dtype", "residual_dtype", "out_dtype", "weight_dtype"):
        assert _norm(L, t, t, t, t, **{k: 1}) == -3, k
        assert _norm(L, t, t, t, t, **{k: 7}) == -3, k
    assert _norm(L, _t2(4, 64, one=2), t, t, t) == -4
    assert _norm(L, t, _t2(4, 64, stride=63), t, t) == -4
    assert _norm(L, t, t, t, _t2(4, 64, stride=0)) == -4      # only the gate may repeat a row
    assert _norm(L, t, t, t, _t2(4, 64, data=FAKE + 1)) == -4
    assert _norm(L, t, t, t, t, out_dtype=2, pre_weight=FAKE + 1) == -4
    assert _norm(L, _t2(4, 64, data=None), t, t, t) == -1
    e = _t2(0, 64, data=None)
    assert _norm(L, e, e, e, e) == 0                           # no rows: nothing to do


def _kv(T=3, H=2, D=128, s0=None, s1=None, data=FAKE, s2=1):
    from dslcompiler_amd._lib import Tensor3D
    return Tensor3D(data, T, H, D, H * D if s0 is None else s0, D if s1 is None else s1, s2)


def _cache(**kw):
    from dslcompiler_amd._lib import Kv4Cache
    d = dict(data=FAKE, pages=10, page_stride=2 * 4 * 17 * 128, heads=2, page_size=64, head_dim=128)
    d.update(kw)
    return Kv4Cache(**d)


def _batch(**kw):
    from dslcompiler_amd._lib import Kv4Batch
    d = dict(table=FAKE, table_stride=5, table_pages=5, lens=FAKE, starts=None, sequences=3,
             tokens=3, max_len=0)
    d.update(kw)
    return Kv4Batch(**d)


def _par(scale=0.1, window=0, sinks=0):
    from dslcompiler_amd._lib import AttentionParams
    return AttentionParams(scale, window, sinks)


def test_head_bytes(L):
    assert L.llk_kv4_head_bytes(16, 64) == 17 * 64
    assert L.llk_kv4_head_bytes(64, 128) == 4 * 17 * 128
    for page, dim in ((0, 64), (8, 64), (24, 64), (8192, 64), (-16, 64), (16, 96), (16, 0), (16, 32)):
        assert L.llk_kv4_head_bytes(page, dim) == 0, (page, dim)


BAD_CACHES = [(dict(data=None), -1), (dict(data=FAKE + 8), -4), (dict(page_stride=17), -4),
              (dict(page_stride=16), -4), (dict(page_size=48), -2), (dict(page_size=8), -2),
              (dict(head_dim=96), -2), (dict(pages=0), -2), (dict(heads=0), -2),
              (dict(heads=70000), -2), (dict(pages=1 << 31), -2)]
BAD_BATCHES = [(dict(lens=None), -1), (dict(table=None), -1), (dict(tokens=4), -2),
               (dict(tokens=-1), -2), (dict(sequences=-1), -2), (dict(table_pages=-1), -2),
               (dict(table_stride=-1), -4), (dict(tokens=1 << 31, starts=FAKE), -2)]
BAD_ROWS = [(dict(T=4), -2), (dict(H=3), -2), (dict(D=64), -2), (dict(data=None), -1),
            (dict(data=FAKE + 1), -4), (dict(s2=2), -4), (dict(s0=-5), -4)]
BAD_RESULTS = BAD_ROWS + [(dict(s0=128, s1=128), -4), (dict(s0=255), -4), (dict(s1=127), -4),
                          (dict(s0=128, s1=256), -4), (dict(s0=0), -4),
                          (dict(s0=1 << 62, s1=1 << 62), -4)]


def test_cache_refusals(L):
    from dslcompiler_amd._lib import AttentionPlan
    k, plan = _kv(), AttentionPlan()
    q = _kv(H=8)
    for bad, code in BAD_CACHES:
        c = _cache(**bad)
        assert L.llk_kv4_write(k, k, c, _batch(), None) == code, bad
        assert L.llk_kv4_read(c, _batch(), k, k, None) == code, bad
        assert L.llk_kv4_attention(q, c, _batch(), _par(), q, None) == code, bad
        assert L.llk_kv4_attention_describe(q, c, _batch(), _par(), plan) == code, bad
        assert L.llk_last_error()
    for bad, code in BAD_BATCHES:
        b = _batch(**bad)
        assert L.llk_kv4_write(k, k, _cache(), b, None) == code, bad
        assert L.llk_kv4_read(_cache(), b, k, k, None) == code, bad
        assert L.llk_kv4_attention(q, _cache(), b, _par(), q, None) == code, bad
    assert L.llk_kv4_write(k, k, None, _batch(), None) == -1
    assert L.llk_kv4_write(k, k, _cache(), None, None) == -1
    assert L.llk_kv4_write(None, k, _cache(), _batch(), None) == -1
    assert L.llk_kv4_read(_cache(), _batch(), k, None, None) == -1
    for bad, code in BAD_ROWS:
        assert L.llk_kv4_write(_kv(**bad), k, _cache(), _batch(), None) == code, bad
        assert L.llk_kv4_write(k, _kv(**bad), _cache(), _batch(), None) == code, bad
    for bad, code in BAD_RESULTS:
        assert L.llk_kv4_read(_cache(), _batch(), _kv(**bad), k, None) == code, bad
        assert L.llk_kv4_read(_cache(), _batch(), k, _kv(**bad), None) == code, bad


def test_attention_refusals(L):
    from dslcompiler_amd._lib import AttentionPlan
    q = _kv(H=8)

    def call(q_=q, par=None, out=None, **b):
        return L.llk_kv4_attention(q_, _cache(), _batch(**b), par or _par(), out or q, None)

    assert L.llk_kv4_attention(None, _cache(), _batch(), _par(), q, None) == -1
    assert L.llk_kv4_attention(q, _cache(), _batch(), None, q, None) == -1
    assert L.llk_kv4_attention(q, _cache(), _batch(), _par(), None, None) == -1
    assert L.llk_kv4_attention_describe(q, _cache(), _batch(), _par(), None) == -1
    assert call(_kv(H=7)) == -2 and b"multiple" in L.llk_last_error()
    assert call(_kv(H=0)) == -2
    assert call(_kv(H=2 * 4097)) == -2
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        assert call(par=_par(scale=bad)) == -1, bad
    assert call(par=_par(window=-1)) == -1
    assert call(par=_par(sinks=-1)) == -1
    assert call(max_len=-1) == -1
    for bad, code in BAD_ROWS:
        assert call(_kv(**{"H": 8, **bad})) == (code if "H" not in bad else -2), bad
    assert call(out=_kv(H=4)) == -2
    assert call(out=_kv(H=8, s0=0)) == -4
    # empty calls do nothing
    assert call(_kv(T=0, H=8), out=_kv(T=0, H=8), tokens=0, sequences=0) == 0
    plan = AttentionPlan()
    assert L.llk_kv4_attention_describe(_kv(T=0, H=8), _cache(), _batch(tokens=0, sequences=0),
                                        _par(), plan) == 0
    assert plan.workspace_bytes == 0 and plan.launches == 0


def test_attention_plans(L):
    """Workspace only where keys are split; a window bounds the splits; the hint
    at the longest length takes the place of the table's size."""
    from dslcompiler_amd._lib import AttentionPlan

    def plan(T, H, window=0, **b):
        p = AttentionPlan()
        assert L.llk_kv4_attention_describe(_kv(T=T, H=H), _cache(), _batch(**b),
                                            _par(window=window), p) == 0
        return p

    one = plan(1, 8, sequences=1, tokens=1, table_pages=2048, table_stride=2048)
    assert one.splits > 8 and one.launches == 2
    # 2 key heads, fp32 sums of 128 and two statistics for each row of each split
    assert one.workspace_bytes == 2 * one.splits * one.rows * 130 * 4
    short = plan(1, 8, sequences=1, tokens=1, table_pages=2048, table_stride=2048, max_len=100)
    assert short.splits == 1 and short.launches == 1 and short.workspace_bytes == 0
    window = plan(1, 8, window=256, sequences=1, tokens=1, table_pages=2048, table_stride=2048)
    assert window.splits <= 2
    many = plan(2048, 8, sequences=2048, tokens=2048, table_pages=64, table_stride=64)
    assert many.splits == 1


def test_python_refusals(llk):
    """The Python layer wants device tensors of the right type and shape."""
    import torch
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.zeros(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        llk.block_norm(x, x, w)
    with pytest.raises(ValueError, match="CUDA"):
        llk.kv4_write(x[None], x[None], x, x, x)
    with pytest.raises(ValueError, match="page_size"):
        llk.kv4_cache(4, 2, 48, 128, device="cpu")
    cache = llk.kv4_cache(4, 2, 64, 128, device="cpu")
    assert cache.shape == (4, 2, 4 * 17 * 128) and cache.dtype == torch.uint8


def test_sizes_beyond_one_launch(L):
    """A dimension of a launch takes fewer than 2^32 threads: 2^24 - 1 workgroups of
    256; what needs more is refused by its size, before any device work."""
    from dslcompiler_amd._lib import AttentionPlan
    plan, n = AttentionPlan(), 1 << 23

    def describe(sequences):
        return L.llk_kv4_attention_describe(_kv(T=sequences, H=8), _cache(),
                                            _batch(sequences=sequences, tokens=sequences), _par(),
                                            plan)

    assert describe(n - 1) == 0 and plan.workgroups == 2 * (n - 1)  # 2 key heads
    assert describe(n) == -2 and b"too many" in L.llk_last_error()
    q = _kv(T=n, H=8)
    assert L.llk_kv4_attention(q, _cache(), _batch(sequences=n, tokens=n), _par(), q, None) == -2
    most = ((1 << 24) - 1) * 16  # tokens written or read, 16 to a workgroup
    k = _kv(T=most + 1)
    b = _batch(sequences=1, tokens=most + 1, starts=FAKE)
    assert L.llk_kv4_write(k, k, _cache(), b, None) == -2
    assert L.llk_kv4_read(_cache(), b, k, k, None) == -2
    assert str(most).encode() in L.llk_last_error()
