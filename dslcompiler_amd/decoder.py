"""The operators around the MLP in a decoder block, on torch tensors.

- :func:`block_norm`: the norm after a block, its gate and residual scale, the
  residual sum and the norm before the next block, in one launch;
- :func:`kv4_cache`, :func:`kv4_write`, :func:`kv4_read`: a paged cache of keys
  and values in 4 bits, quantised as it is written;
- :func:`kv4_attention`: attention over that cache, for single tokens and for
  prompts, with a sliding window and first positions that stay visible.

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
from .ops import _check_operand, _ctx, _torch

_NO_GATE = _lib.Tensor2D(None, 0, 0, 0, 0)
_TYPES = None  # torch dtype -> llk_dtype


def _type(t, name: str) -> int:
    """The element type of a bf16 or fp32 operand on the current device."""
    global _TYPES
    if _TYPES is None:
        torch = _torch()
        _TYPES = {torch.bfloat16: LLK_BF16, torch.float32: LLK_FP32}
    _check_operand(t, name, _TYPES)
    return _TYPES[t.dtype]


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
    torch = _torch()
    rtype = _type(residual, "residual")
    rd = _rows(residual, "residual")
    n = rd.dim1
    wtype = _type(pre_weight, "pre_weight")
    post = None
    if post_weight is not None:
        if _type(post_weight, "post_weight") != wtype:
            raise ValueError("post_weight and pre_weight have different types")
        post = _weight(post_weight, "post_weight", n)
    yd, ytype, gd = None, LLK_BF16, _NO_GATE
    if y is not None:
        ytype = _type(y, "y")
        yd = _rows(y, "y")
    if gate is not None:
        if _type(gate, "gate") != ytype or y is None:
            raise ValueError("gate must have y's type")
        if gate.dim() == 1:
            if gate.shape[0] > 1 and gate.stride(0) != 1:
                raise ValueError("gate must have unit stride")
            gd = _lib.Tensor2D(gate.data_ptr(), rd.dim0, gate.shape[0], 0, 1)
        else:
            gd = _rows(gate, "gate")
    if residual_out is None:
        if y is not None:
            residual_out = torch.empty(residual.shape, dtype=residual.dtype, device=residual.device)
        od = None if y is None else _lib.Tensor2D(residual_out.data_ptr(), rd.dim0, n, n, 1)
    else:
        if _type(residual_out, "residual_out") != rtype:
            raise ValueError("residual_out must have residual's type")
        od = _rows(residual_out, "residual_out")
    if out is None:
        out = torch.empty(residual.shape, dtype=out_dtype or torch.bfloat16, device=residual.device)
    params = _lib.BlockNormParams(ytype, rtype, _type(out, "out"), wtype, post,
                                  _weight(pre_weight, "pre_weight", n), gd, scale, eps,
                                  weight_offset)
    check(lib().llk_block_norm(yd, rd, od, _rows(out, "out"), params, _ctx(stream)))
    return (residual if residual_out is None else residual_out), out


def kv4_cache(pages: int, heads: int, page_size: int, head_dim: int, device="cuda"):
    """A zeroed cache: uint8 [pages, heads, page_size * head_dim * 17 / 16].
    page_size: a power of two from 16 to 4096; head_dim: 64, 128 or 256."""
    torch = _torch()
    n = lib().llk_kv4_head_bytes(page_size, head_dim)
    if n == 0:
        raise ValueError(f"no cache of page_size {page_size} and head_dim {head_dim}")
    return torch.zeros((pages, heads, n), dtype=torch.uint8, device=device)


def _cache(cache, head_dim: int) -> _lib.Kv4Cache:
    _check_operand(cache, "cache", (_torch().uint8,))
    if cache.dim() != 3:
        raise ValueError("cache must be [pages, heads, bytes]")
    pages, heads, n = cache.shape
    step, head, one = cache.stride()
    if (n > 1 and one != 1) or (heads > 1 and head != n):
        raise ValueError("the heads of a cache page must be contiguous")
    size, rest = divmod(n * 16, 17 * head_dim)
    if rest or n == 0:
        raise ValueError(f"{n} bytes to a head are no pages of head_dim {head_dim}")
    return _lib.Kv4Cache(cache.data_ptr(), pages, step, heads, size, head_dim)


def _batch(table, lens, starts, tokens: int, max_len) -> _lib.Kv4Batch:
    i32 = (_torch().int32,)
    _check_operand(table, "table", i32)
    _check_operand(lens, "lens", i32)
    n = lens.shape[0]
    if table.dim() != 2 or lens.dim() != 1 or table.shape[0] != n:
        raise ValueError("table must be [sequences, pages] and lens [sequences]")
    step, one = table.stride()
    if (table.shape[1] > 1 and one != 1) or (n > 1 and lens.stride(0) != 1):
        raise ValueError("table and lens must have unit inner stride")
    first = None
    if starts is not None:
        _check_operand(starts, "starts", i32)
        if starts.dim() != 1 or starts.shape[0] != n + 1 or starts.stride(0) != 1:
            raise ValueError("starts must be a contiguous vector of sequences + 1 entries")
        first = starts.data_ptr()
    return _lib.Kv4Batch(table.data_ptr(), step, table.shape[1], lens.data_ptr(), first, n, tokens,
                         max_len or 0)


def _rows3(t, name: str) -> _lib.Tensor3D:
    _check_operand(t, name, (_torch().bfloat16,))
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim]")
    return _lib.Tensor3D(t.data_ptr(), *t.shape, *t.stride())


def kv4_write(k, v, cache, table, lens, *, starts=None, stream=None) -> None:
    """Quantises the new tokens' keys and values, bf16 [tokens, heads,
    head_dim], into the cache; tokens without a place in it are skipped."""
    kd = _rows3(k, "k")
    check(lib().llk_kv4_write(kd, _rows3(v, "v"), _cache(cache, kd.dim2),
                              _batch(table, lens, starts, kd.dim0, None), _ctx(stream)))


def kv4_read(cache, table, lens, *, head_dim: int, starts=None, tokens: int | None = None, k=None,
             v=None, stream=None):
    """(k, v) of the last starts[s + 1] - starts[s] positions of every
    sequence, bf16 [tokens, heads, head_dim]; with `starts`, `tokens` gives the
    number of rows (unless k or v is given)."""
    torch = _torch()
    cd = _cache(cache, head_dim)
    if tokens is None:
        given = k if k is not None else v
        if given is not None:
            tokens = given.shape[0]
        elif starts is None:
            tokens = lens.shape[0]
        else:
            raise ValueError("kv4_read with starts needs `tokens`")
    shape = (tokens, cd.heads, head_dim)
    if k is None:
        k = torch.empty(shape, dtype=torch.bfloat16, device=cache.device)
    if v is None:
        v = torch.empty(shape, dtype=torch.bfloat16, device=cache.device)
    check(lib().llk_kv4_read(cd, _batch(table, lens, starts, tokens, None), _rows3(k, "k"),
                             _rows3(v, "v"), _ctx(stream)))
    return k, v


def _attention(q, cache, table, lens, starts, scale, window, sinks, max_len):
    qd = _rows3(q, "q")
    if scale is None:
        scale = qd.dim2 ** -0.5
    return (qd, _cache(cache, qd.dim2), _batch(table, lens, starts, qd.dim0, max_len),
            _lib.AttentionParams(scale, window, sinks))


def kv4_attention(q, cache, table, lens, *, starts=None, scale: float | None = None,
                  window: int = 0, sinks: int = 0, max_len: int | None = None, out=None,
                  stream=None, scratch=None):
    """softmax(scale q k^T) v of the new tokens' queries, bf16 [tokens, q_heads,
    head_dim], over the cached keys and values.

    q_heads is a multiple of the cache's heads; scale defaults to head_dim **
    -0.5.  The query at position p sees key j if j <= p and, with a window, j >
    p - window or j < sinks; one that sees none gives zeros.  max_len, if the
    caller knows it, is at least the longest of lens: the launch is planned by
    it (by the table's size otherwise), and any value gives right results."""
    args = _attention(q, cache, table, lens, starts, scale, window, sinks, max_len)
    if out is None:
        out = _torch().empty(q.shape, dtype=q.dtype, device=q.device)
    check(lib().llk_kv4_attention(*args, _rows3(out, "out"), _ctx(stream, scratch)))
    return out


def describe_kv4_attention(q, cache, table, lens, *, starts=None, scale: float | None = None,
                           window: int = 0, sinks: int = 0, max_len: int | None = None) -> dict:
    """The launch kv4_attention chooses for these arguments."""
    p = _lib.AttentionPlan()
    check(lib().llk_kv4_attention_describe(
        *_attention(q, cache, table, lens, starts, scale, window, sinks, max_len), p))
    return {"rows": p.rows, "splits": p.splits, "workgroups": p.workgroups,
            "launches": p.launches, "workspace_bytes": p.workspace_bytes}
