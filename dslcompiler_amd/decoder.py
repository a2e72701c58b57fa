"""The operators around the MLP in a decoder block, on torch tensors.

- :func:`block_norm`: the norm after a block, its gate and residual scale, the
  residual sum and the norm before the next block, in one launch;
- :func:`kv4_cache`, :func:`kv4_write`, :func:`kv4_read`: a paged cache of keys
  and values in 4 bits, quantised as it is written;
- :func:`kv4_attention`: attention over that cache, for single tokens and for
  prompts, with a sliding window and first positions that stay visible;
- :func:`kv4_marks`, :func:`kv4_evict_plan`, :func:`kv4_evict`: the attention
  weight that each cached token got, and a cache bounded by it.

The cache is a uint8 tensor [pages, heads, bytes] (the layout is in
``include/llk/llk_abi.h``), which may be a slice of a larger pool.  A call's
sequences are int32 tensors on the device: ``table[s, i]`` names the page of
positions ``i * page_size`` on, ``lens[s]`` counts the positions with the new
tokens, and ``starts`` (sequences + 1 entries; None: one new token each) says
which rows of the call's tensors are a sequence's new tokens, its last
positions.  Nothing is read back to the host.
"""
from __future__ import annotations

from . import _lib
from ._lib import LLK_BF16, LLK_FP32, check, lib
from .ops import _check_operand, _check_scratch, _torch

_NO_GATE = _lib.Tensor2D(None, 0, 0, 0, 0)
_get_device = _raw_stream = None  # torch's current device and its stream's handle
_FLOATS = _BF16 = _INT32 = _UINT8 = _FP32 = None  # torch dtype -> llk_dtype (0 for the others)


def _begin() -> int:
    """The current device.  (A call of these operators is a few microseconds of
    GPU work in a decode step: the checks below take 0.2 us an operand.)"""
    global _get_device, _raw_stream, _FLOATS, _BF16, _INT32, _UINT8, _FP32
    if _get_device is None:
        torch = _torch()
        _FLOATS = {torch.bfloat16: LLK_BF16, torch.float32: LLK_FP32}
        _FP32 = {torch.float32: LLK_FP32}
        _BF16, _INT32, _UINT8 = {torch.bfloat16: LLK_BF16}, {torch.int32: 0}, {torch.uint8: 0}
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda d: int(torch.cuda.current_stream(d).cuda_stream))
        if not torch.cuda.is_available():
            return -2  # no operand is there
        torch.cuda.init()
        _get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    return _get_device()


def _kind(t, name: str, dev: int, kinds) -> int:
    """kinds' entry for the type of an operand on the current device."""
    kind = kinds.get(getattr(t, "dtype", None))
    if kind is None or t.get_device() != dev:
        _check_operand(t, name, kinds)  # says what is wrong
        raise ValueError(f"{name} is not on the current device")
    return kind


def _context(dev: int, stream, scratch=None) -> _lib.KernelContext:
    handle = _raw_stream(dev) if stream is None else int(stream.cuda_stream)
    if scratch is None:
        return _lib.KernelContext(None, 0, handle)
    _check_scratch(scratch)
    return _lib.KernelContext(scratch.data_ptr(), scratch.numel() * scratch.element_size(), handle)


def _result(like, dtype):
    """An uninitialised contiguous tensor of like's shape and device."""
    torch = _torch()
    if like.is_contiguous():
        return torch.empty_like(like, dtype=dtype)
    return torch.empty(like.shape, dtype=dtype, device=like.device)


def _rows(t, name: str) -> _lib.Tensor2D:
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D")
    return _lib.Tensor2D(t.data_ptr(), *t.shape, *t.stride())


def _weight(w, name: str, n: int):
    if w.dim() != 1 or w.shape[0] != n or (n > 1 and w.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous vector of {n} elements")
    return w.data_ptr()


def block_norm(y, residual, pre_weight, *, post_weight=None, gate=None, scale: float = 1.0,
               eps: float = 1e-6, weight_offset: float = 0.0, residual_out=None, out=None,
               out_dtype=None, stream=None):
    """(residual_out, out) of the step between two blocks of a decoder layer:

        u = y * rsqrt(mean(y^2) + eps) * (post_weight + weight_offset), or y
        residual_out = residual + scale * gate * u
        out = r * rsqrt(mean(r^2) + eps) * (pre_weight + weight_offset)

    with r the sum before its rounding to the residual's type.  y, residual and
    out are [M, N], bf16 or fp32 each; gate is [M, N] or [N], of y's type; the
    weights are [N], both bf16 or both fp32.  y None: the norm alone (r =
    residual, which is also returned unless residual_out is given).
    residual_out may be residual itself.  out_dtype defaults to bf16."""
    dev = _begin()
    rtype = _kind(residual, "residual", dev, _FLOATS)
    rd = _rows(residual, "residual")
    n = rd.dim1
    wtype = _kind(pre_weight, "pre_weight", dev, _FLOATS)
    post = None
    if post_weight is not None:
        if _kind(post_weight, "post_weight", dev, _FLOATS) != wtype:
            raise ValueError("post_weight and pre_weight have different types")
        post = _weight(post_weight, "post_weight", n)
    yd, ytype, gd, od = None, LLK_BF16, _NO_GATE, None
    if y is not None:
        ytype = _kind(y, "y", dev, _FLOATS)
        yd = _rows(y, "y")
    if gate is not None:
        if y is None or _kind(gate, "gate", dev, _FLOATS) != ytype:
            raise ValueError("gate must have y's type")
        if gate.dim() == 1:
            if gate.shape[0] > 1 and gate.stride(0) != 1:
                raise ValueError("gate must have unit stride")
            gd = _lib.Tensor2D(gate.data_ptr(), rd.dim0, gate.shape[0], 0, 1)
        else:
            gd = _rows(gate, "gate")
    if residual_out is not None:
        if _kind(residual_out, "residual_out", dev, _FLOATS) != rtype:
            raise ValueError("residual_out must have residual's type")
        od = _rows(residual_out, "residual_out")
    elif y is None:
        residual_out = residual
    else:
        residual_out = _result(residual, residual.dtype)
        od = _lib.Tensor2D(residual_out.data_ptr(), rd.dim0, n, n, 1)
    if out is None:
        out = _result(residual, out_dtype or _torch().bfloat16)
        nd = _lib.Tensor2D(out.data_ptr(), rd.dim0, n, n, 1)
    else:
        nd = _rows(out, "out")
    params = _lib.BlockNormParams(ytype, rtype, _kind(out, "out", dev, _FLOATS), wtype, post,
                                  _weight(pre_weight, "pre_weight", n), gd, scale, eps,
                                  weight_offset)
    check(lib().llk_block_norm(yd, rd, od, nd, params, _context(dev, stream)))
    return residual_out, out


def kv4_cache(pages: int, heads: int, page_size: int, head_dim: int, device="cuda"):
    """A zeroed cache: uint8 [pages, heads, page_size * head_dim * 17 / 16].
    page_size: a power of two from 16 to 4096; head_dim: 64, 128 or 256."""
    torch = _torch()
    n = lib().llk_kv4_head_bytes(page_size, head_dim)
    if n == 0:
        raise ValueError(f"no cache of page_size {page_size} and head_dim {head_dim}")
    return torch.zeros((pages, heads, n), dtype=torch.uint8, device=device)


def _cache(cache, head_dim: int, dev: int) -> _lib.Kv4Cache:
    _kind(cache, "cache", dev, _UINT8)
    if cache.dim() != 3:
        raise ValueError("cache must be [pages, heads, bytes]")
    pages, heads, n = cache.shape
    step, head, one = cache.stride()
    if (n > 1 and one != 1) or (heads > 1 and head != n):
        raise ValueError("the heads of a cache page must be contiguous")
    size, rest = divmod(n * 16, 17 * head_dim) if head_dim > 0 else (0, 1)
    if rest or n == 0:
        raise ValueError(f"{n} bytes to a head are no pages of head_dim {head_dim}")
    return _lib.Kv4Cache(cache.data_ptr(), pages, step, heads, size, head_dim)


def _batch(table, lens, starts, tokens: int, max_len, dev: int) -> _lib.Kv4Batch:
    _kind(table, "table", dev, _INT32)
    _kind(lens, "lens", dev, _INT32)
    if table.dim() != 2 or lens.dim() != 1:
        raise ValueError("table must be [sequences, pages] and lens [sequences]")
    n, pages = table.shape
    step, one = table.stride()
    if lens.shape[0] != n:
        raise ValueError(f"table has {n} sequences and lens {lens.shape[0]}")
    if (pages > 1 and one != 1) or (n > 1 and lens.stride(0) != 1):
        raise ValueError("table and lens must have unit inner stride")
    first = None
    if starts is not None:
        _kind(starts, "starts", dev, _INT32)
        if starts.dim() != 1 or starts.shape[0] != n + 1 or starts.stride(0) != 1:
            raise ValueError("starts must be a contiguous vector of sequences + 1 entries")
        first = starts.data_ptr()
    return _lib.Kv4Batch(table.data_ptr(), step, pages, lens.data_ptr(), first, n, tokens,
                         max_len or 0)


def _rows3(t, name: str, dev: int) -> _lib.Tensor3D:
    _kind(t, name, dev, _BF16)
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim]")
    return _lib.Tensor3D(t.data_ptr(), *t.shape, *t.stride())


def kv4_marks(pages: int, heads: int, page_size: int, device="cuda"):
    """(weights fp32, positions int32) of a cache's slots, zeroed [pages, heads,
    page_size]: the attention weight each slot's token got, and its position."""
    torch = _torch()
    shape = (pages, heads, page_size)
    return (torch.zeros(shape, dtype=torch.float32, device=device),
            torch.zeros(shape, dtype=torch.int32, device=device))


def _mark(t, name: str, shape, kinds, dev: int) -> tuple:
    """(address, page stride) of one of a cache's marks; shape: (pages, heads,
    page_size)."""
    _kind(t, name, dev, kinds)
    if t.shape != shape:
        raise ValueError(f"{name} must be [pages, heads, page_size] = {list(shape)}")
    step, head, one = t.stride()
    if (shape[2] > 1 and one != 1) or (shape[1] > 1 and head != shape[2]):
        raise ValueError(f"the heads of a page of {name} must be contiguous")
    return t.data_ptr(), step


def _marks(weights, positions, shape, dev: int) -> _lib.Kv4Marks:
    w, ws = (None, 0) if weights is None else _mark(weights, "weights", shape, _FP32, dev)
    p, ps = (None, 0) if positions is None else _mark(positions, "positions", shape, _INT32, dev)
    return _lib.Kv4Marks(w, p, ws, ps)


def kv4_write(k, v, cache, table, lens, *, starts=None, weights=None, positions=None, at=None,
              stream=None) -> None:
    """Quantises the new tokens' keys and values, bf16 [tokens, heads,
    head_dim], into the cache; tokens without a place in it are skipped.

    With marks (:func:`kv4_marks`), those of the slots that are written are set:
    `weights` to 0, `positions` to at[token], int32 (None: the slot's number)."""
    dev = _begin()
    kd = _rows3(k, "k", dev)
    cd, batch = _cache(cache, kd.dim2, dev), _batch(table, lens, starts, kd.dim0, None, dev)
    if weights is None and positions is None:
        if at is not None:
            raise ValueError("at without positions")
        check(lib().llk_kv4_write(kd, _rows3(v, "v", dev), cd, batch, _context(dev, stream)))
        return
    marks = _marks(weights, positions, (cd.pages, cd.heads, cd.page_size), dev)
    if at is not None:
        _kind(at, "at", dev, _INT32)
        if positions is None or at.dim() != 1 or at.shape[0] != kd.dim0 or (
                kd.dim0 > 1 and at.stride(0) != 1):
            raise ValueError("at must be a contiguous vector of the tokens' positions, for positions")
        at = at.data_ptr()
    check(lib().llk_kv4_write_marked(kd, _rows3(v, "v", dev), cd, batch, marks, at,
                                     _context(dev, stream)))


def kv4_read(cache, table, lens, *, head_dim: int, starts=None, tokens: int | None = None, k=None,
             v=None, stream=None):
    """(k, v) of the last starts[s + 1] - starts[s] positions of every
    sequence, bf16 [tokens, heads, head_dim]; with `starts`, `tokens` gives the
    number of rows (unless k or v is given)."""
    dev = _begin()
    cd = _cache(cache, head_dim, dev)
    if tokens is None:
        given = k if k is not None else v
        if given is not None:
            tokens = given.shape[0]
        elif starts is None:
            tokens = lens.shape[0]
        else:
            raise ValueError("kv4_read with starts needs `tokens`")
    batch = _batch(table, lens, starts, tokens, None, dev)
    if k is None:
        torch = _torch()
        k = cache.new_empty((tokens, cd.heads, head_dim), dtype=torch.bfloat16)
        if v is None:
            v = torch.empty_like(k)
    elif v is None:
        v = _result(k, k.dtype)
    check(lib().llk_kv4_read(cd, batch, _rows3(k, "k", dev), _rows3(v, "v", dev),
                             _context(dev, stream)))
    return k, v


def _attention(q, cache, table, lens, starts, scale, window, sinks, max_len, dev):
    qd = _rows3(q, "q", dev)
    if scale is None:
        scale = qd.dim2 ** -0.5
    return (qd, _cache(cache, qd.dim2, dev), _batch(table, lens, starts, qd.dim0, max_len, dev),
            _lib.AttentionParams(scale, window, sinks))


def kv4_attention(q, cache, table, lens, *, starts=None, scale: float | None = None,
                  window: int = 0, sinks: int = 0, max_len: int | None = None, out=None,
                  weights=None, decay: float = 1.0, stream=None, scratch=None):
    """softmax(scale q k^T) v of the new tokens' queries, bf16 [tokens, q_heads,
    head_dim], over the cached keys and values.

    q_heads is a multiple of the cache's heads; scale defaults to head_dim **
    -0.5.  The query at position p sees key j if j <= p and, with a window, j >
    p - window or j < sinks; one that sees none gives zeros.  Rows outside every
    sequence (padding of a captured step) are not written: what `out` held, or
    nothing defined.  max_len, if the caller knows it, is at least the longest
    of lens: the launch is planned by it (by the table's size otherwise), and
    any value gives right results.

    weights (of :func:`kv4_marks`): in every slot of a sequence with new tokens,
    decay times what was there (with 0 it is not read) plus the softmax weights
    that the new tokens' query heads gave it.  A page that is in the table twice
    (a prefix that two sequences share) gets sums without order.  out must not be
    q then."""
    dev = _begin()
    args = _attention(q, cache, table, lens, starts, scale, window, sinks, max_len, dev)
    if out is None:
        out = _result(q, q.dtype)
        qd = args[0]
        od = _lib.Tensor3D(out.data_ptr(), qd.dim0, qd.dim1, qd.dim2, qd.dim1 * qd.dim2, qd.dim2, 1)
    else:
        od = _rows3(out, "out", dev)
    if weights is None:
        check(lib().llk_kv4_attention(*args, od, _context(dev, stream, scratch)))
    else:
        c = args[1]
        marks = _marks(weights, None, (c.pages, c.heads, c.page_size), dev)
        check(lib().llk_kv4_attention_weigh(*args, marks, decay, od, _context(dev, stream, scratch)))
    return out


def kv4_evict_plan(weights, table, lens, keep: int, *, positions=None, recent: int = 0,
                   first: int = 0, max_len: int | None = None, lens_out=None, stream=None):
    """(new lens, source): which slots stay where a sequence has more than `keep`.

    Of each head's slots stay the `recent` newest positions and those below
    `first` (which need `positions`; recent + first <= keep), then those of the
    largest weights, ties to the lowest slot.  source int32 [sequences, heads,
    keep] names the slot each slot below keep takes its token from (itself, if it
    does not change): slots below keep that stay are not moved, the others take
    those from keep on that stay, both in order.  Nothing is moved, and lens stays
    as it is (lens_out must be other memory)."""
    dev = _begin()
    _kind(weights, "weights", dev, _FP32)
    if weights.dim() != 3:
        raise ValueError("weights must be [pages, heads, page_size]")
    pages, heads, size = shape = weights.shape
    marks = _marks(weights, positions, shape, dev)
    batch = _batch(table, lens, None, table.shape[0], max_len, dev)
    if lens_out is None:
        lens_out = lens.new_empty(lens.shape)
    else:
        _kind(lens_out, "lens_out", dev, _INT32)
        if lens_out.shape != lens.shape or (lens.shape[0] > 1 and lens_out.stride(0) != 1):
            raise ValueError("lens_out must be a contiguous vector like lens")
    # (a keep that the call refuses takes no memory)
    source = lens.new_empty((batch.sequences, heads, keep if 0 < keep <= 1 << 30 else 0))
    check(lib().llk_kv4_evict_plan(marks, pages, heads, size, batch,
                                   _lib.EvictParams(keep, recent, first), lens_out.data_ptr(),
                                   source.data_ptr(), _context(dev, stream)))
    return lens_out, source


def kv4_evict(cache, table, source, *, head_dim: int, weights=None, positions=None, lens=None,
              stream=None) -> None:
    """Moves the cache's tokens, and their marks if given, as `source` of
    :func:`kv4_evict_plan` says; lens, if given, is cut to source's `keep` in
    place.  The pages behind the new lengths are free.  A page that two sequences
    share would be changed for both: copy it before."""
    dev = _begin()
    cd = _cache(cache, head_dim, dev)
    marks = _marks(weights, positions, (cd.pages, cd.heads, cd.page_size), dev)
    _kind(table, "table", dev, _INT32)
    if table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError("table must be [sequences, pages] with unit inner stride")
    n, pages = table.shape
    _kind(source, "source", dev, _INT32)
    if source.dim() != 3 or source.shape[:2] != (n, cd.heads) or not source.is_contiguous():
        raise ValueError(f"source must be contiguous [{n}, {cd.heads}, keep]")
    if lens is not None:
        _kind(lens, "lens", dev, _INT32)
        if lens.dim() != 1 or lens.shape[0] != n or (n > 1 and lens.stride(0) != 1):
            raise ValueError("lens must be a contiguous vector of the sequences")
        lens = lens.data_ptr()
    batch = _lib.Kv4Batch(table.data_ptr(), table.stride(0), pages, None, None, n, n, 0)
    check(lib().llk_kv4_evict(cd, batch, source.data_ptr(), source.shape[2], marks, lens,
                              _context(dev, stream)))


def describe_kv4_attention(q, cache, table, lens, *, starts=None, scale: float | None = None,
                           window: int = 0, sinks: int = 0, max_len: int | None = None,
                           weigh: bool = False) -> dict:
    """The launch kv4_attention chooses for these arguments (weigh: with
    `weights`)."""
    p = _lib.AttentionPlan()
    describe = lib().llk_kv4_attention_weigh_describe if weigh else lib().llk_kv4_attention_describe
    check(describe(*_attention(q, cache, table, lens, starts, scale, window, sinks, max_len, _begin()),
                   p))
    return {"rows": p.rows, "splits": p.splits, "workgroups": p.workgroups,
            "launches": p.launches, "workspace_bytes": p.workspace_bytes}
