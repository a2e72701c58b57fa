"""The 4-bit cache and attention over it from their definitions, in 64 bits
(numpy; nothing of the library).  Pools are uint8 [pages, heads, bytes] as
include/llk/llk_abi.h lays them out."""
from __future__ import annotations

import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def bf16_round(x: np.ndarray) -> np.ndarray:
    """float32 values rounded to bf16 (nearest even), as float32."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32)
    return np.where(np.isnan(x), np.float32(np.nan), r.view(np.float32))


def quantise(x: np.ndarray):
    """(codes [..., D / 32, 32] 0..15, scale bytes [..., D / 32]) of x [..., D]."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(b).max(-1)
    ok = np.isfinite(top)
    e = np.full(top.shape, -126.0)
    some = ok & (top > 0)
    # smallest e with top <= 7 * 2^e
    e[some] = np.ceil(np.log2(top[some] / 7))
    for _ in range(2):  # log2's rounding
        e = np.where(some & (top > 7 * np.exp2(e)), e + 1, e)
        e = np.where(some & (top <= 7 * np.exp2(e - 1)), e - 1, e)
    e = np.clip(e, -126, 125)
    with np.errstate(invalid="ignore"):
        a = np.abs(b) / np.exp2(e)[..., None]
        d = np.abs(np.where(ok[..., None], a, 0)[..., None] - LEVELS)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = code + 8 * np.signbit(b)
    return (np.where(ok[..., None], code, 0).astype(np.uint8),
            np.where(ok, e + 127, 255).astype(np.uint8))


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """What codes and scales of quantise() stand for: [..., D]."""
    v = LEVELS[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    v = v * s[..., None]
    return v.reshape(*v.shape[:-2], -1)


def _views(pool: np.ndarray, D: int):
    """Code bytes [pages, heads, tiles, 2, D / 32, 16, 16] and scales [..., 16]."""
    t = pool.reshape(*pool.shape[:2], -1, 17 * D)
    return (t[..., :16 * D].reshape(*t.shape[:3], 2, D // 32, 16, 16),
            t[..., 16 * D:].reshape(*t.shape[:3], 2, D // 32, 16))


def page_size(pool, D: int) -> int:
    return pool.shape[2] * 16 // (17 * D)


def put(pool, page: int, off: int, k: np.ndarray, v: np.ndarray) -> None:
    """Writes one token's k and v [heads, D] at a place, in the pool itself."""
    D = k.shape[-1]
    codes, scales = _views(pool, D)
    for part, x in enumerate((k, v)):
        c, s = quantise(x)
        codes[page, :, off // 16, part, :, off % 16] = c[..., 0::2] | (c[..., 1::2] << 4)
        scales[page, :, off // 16, part, :, off % 16] = s


def get(pool, page: int, off: int, D: int):
    """(k, v) [heads, D] of a place."""
    codes, scales = _views(pool, D)
    out = []
    for part in (0, 1):
        b = codes[page, :, off // 16, part, :, off % 16]
        c = np.stack((b & 15, b >> 4), -1).reshape(*b.shape[:-1], 32)
        out.append(values(c, scales[page, :, off // 16, part, :, off % 16]))
    return out


def places(pool_pages: int, size: int, table, lens, starts, s: int):
    """(position, page or -1) of every new token of sequence s."""
    new = 1 if starts is None else int(starts[s + 1] - starts[s])
    for i in range(new):
        p = int(lens[s]) - new + i
        ok = 0 <= p < table.shape[1] * size
        page = int(table[s, p // size]) if ok else -1
        yield p, page if 0 <= page < pool_pages else -1


def attention(q, pool, table, lens, starts, scale, window=0, sinks=0):
    """(out, magnitude) [tokens, heads, D]: the result, and sum of weight * |v|,
    which rounding errors of the weights scale with."""
    T, H, D = q.shape
    pages, heads = pool.shape[:2]
    size, group = page_size(pool, D), H // heads
    out, mag = np.zeros((T, H, D)), np.zeros((T, H, D))
    for s in range(len(lens)):
        first = s if starts is None else int(starts[s])
        new = 1 if starts is None else int(starts[s + 1]) - first
        n = min(max(int(lens[s]), 0), table.shape[1] * size)
        kv = np.zeros((2, n, heads, D))
        here = np.zeros(n, bool)
        for j in range(n):
            page = int(table[s, j // size])
            if 0 <= page < pages:
                here[j] = True
                kv[0, j], kv[1, j] = get(pool, page, j % size, D)
        j = np.arange(n)
        for i in range(new):
            p = int(lens[s]) - new + i
            seen = here & (j <= p)
            if window:
                seen &= (j > p - window) | (j < sinks)
            if not seen.any():
                continue
            for h in range(H):
                with np.errstate(invalid="ignore", over="ignore"):
                    w = kv[0, seen, h // group] @ q[first + i, h].astype(np.float64) * scale
                    if (w == -np.inf).all():
                        continue
                    w = np.exp(w - w.max())
                    w /= w.sum()
                    out[first + i, h] = w @ kv[1, seen, h // group]
                    mag[first + i, h] = w @ np.abs(kv[1, seen, h // group])
    return out, mag
