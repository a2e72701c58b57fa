"""The operators around the MLP in a decoder block, as measurable cases.

  norm    block_norm: the norm after a block, its gate and residual scale, the
          residual sum and the norm before the next block
  append  kv4_write, then kv4_read: keys and values quantised to 4 bits as they
          are written to a paged cache, and the same tokens read back
  read    kv4_read: the cached keys and values of whole sequences
  attend  kv4_attention: attention over the 4-bit paged cache, for single
          tokens and for prompts, with a sliding window and visible first tokens

The cache.  A token's key (value) of one head is cut into blocks of 32 values.
A block is stored as one scale byte E, standing for 2^(E - 127), and 32 codes of
4 bits: a sign bit over an index into 0, 0.5, 1, 1.5, 2, 3, 4, 6; E = 255 stands
for a block of NaN.  For a block's largest magnitude a, 2^(E - 127) is the
smallest power of two with a <= 7 * 2^(E - 127), held to 1 <= E <= 252, and a
value's code is the nearest one (ties to the even index, beyond 6 to 6).  16
consecutive tokens of a page and head lie together: key codes [block][token][16
bytes], value codes, key scales [block][token], value scales.  The pool is
[pages, heads, page_size / 16 such tiles], and table[s, i] names the page that
holds positions i * page_size on of sequence s.

A sequence s holds lens[s] positions, of which the last starts[s + 1] -
starts[s] (one, where there are no starts) are the call's new tokens; query i of
them sees key j if j <= its position p and (j > p - window or j < sinks).
"""
import math

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # One decoded token between the attention block and the MLP of an
        # 8B-class layer: residual sum and the next norm only.
        dict(name="norm m1", op="norm", M=1, N=4096, post=False, gate="none", y="f32",
             res="bf16", out="bf16"),
        # A ragged decode or prompt chunk through a 13B-class layer with a norm
        # after the block, a learned gate per channel and an fp32 residual.
        dict(name="norm m255 post", op="norm", M=255, N=5120, post=True, gate="channel",
             y="f32", res="f32", out="bf16"),
        # The largest prompt: a norm after the block and a gate for each value.
        dict(name="norm m4097 gated", op="norm", M=4097, N=5120, post=True, gate="token",
             y="bf16", res="bf16", out="bf16"),
        # A decode step of 64 sequences: one token each into 8 heads.
        dict(name="append decode s64", op="append", seqs=64, new=1, ctx=4097, kv_heads=8, dim=128,
             page=64),
        # A prompt of 2048 tokens into 32 heads.
        dict(name="append prompt 2048", op="append", seqs=1, new=2048, ctx=2048, kv_heads=32,
             dim=128, page=64),
        # A short sequence read back whole, odd length, narrow heads.
        dict(name="read ctx17 d64", op="read", seqs=1, new=17, ctx=17, kv_heads=8, dim=64,
             page=16),
        # 16 ragged sequences read back whole, as for moving them elsewhere.
        dict(name="read s16 ctx4097", op="read", seqs=16, new=4097, ctx=4097, kv_heads=8,
             dim=128, page=64),
        # One decoded token of one short sequence: the latency of a step.
        dict(name="attend decode s1", op="attend", seqs=1, new=1, ctx=1000, heads=32, kv_heads=8,
             dim=128, page=64, window=0, sinks=0),
        # A decode step of 64 ragged sequences, four query heads to a key head.
        dict(name="attend decode s64", op="attend", seqs=64, new=1, ctx=8192, heads=32,
             kv_heads=8, dim=128, page=64, window=0, sinks=0),
        # One token over one long sequence.
        dict(name="attend decode long", op="attend", seqs=1, new=1, ctx=131072, heads=32,
             kv_heads=8, dim=128, page=64, window=0, sinks=0),
        # A prompt of 2048 tokens, a key head to each query head.
        dict(name="attend prompt 2048", op="attend", seqs=1, new=2048, ctx=2048, heads=32,
             kv_heads=32, dim=128, page=64, window=0, sinks=0),
        # Ragged prompt chunks on top of ragged contexts, a window of 1024 and
        # the first 4 tokens, pages of 16 tokens.
        dict(name="attend chunks window", op="attend", seqs=4, new=1000, ctx=4097, heads=40,
             kv_heads=8, dim=128, page=16, window=1024, sinks=4),
    ]


def _log_int(rng, lo, hi):
    """A number from lo to hi, even over their logarithm: above 64 an odd one or a
    multiple of 40."""
    n = min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    if n > 64:
        n = n // 40 * 40 if rng.random() < 0.5 else (n - 1) | 1
    return max(lo, n)


def draw(rng):
    op = rng.choices(["norm", "append", "read", "attend"], [25, 15, 10, 50])[0]
    if op == "norm":
        return dict(op=op, M=_log_int(rng, 1, 4097),
                    N=rng.choice([512, 1376, 2048, 4096, 5120, _log_int(rng, 512, 5120)]),
                    post=rng.random() < 0.6, gate=rng.choice(["none", "channel", "token"]),
                    y=rng.choice(["bf16", "f32"]), res=rng.choice(["bf16", "f32"]),
                    out=rng.choice(["bf16", "bf16", "f32"]))
    # key heads and width; query heads to a key head
    kv_heads, dim = rng.choice([(8, 128), (32, 128), (40, 128), (8, 64), (4, 64), (2, 256), (1, 128)])
    c = dict(op=op, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128, 256]))
    if op != "attend":
        new = 1 if op == "append" and rng.random() < 0.4 else _log_int(rng, 2, 4097)
        seqs = _log_int(rng, 1, max(1, min(64, 40960 * 8 * 128 // (new * kv_heads * dim))))
        return dict(c, seqs=seqs, new=new, ctx=new if op == "read" else _log_int(rng, new, 8192))
    c.update(heads=kv_heads * rng.choice([1, 4, 5, 8] if kv_heads <= 8 else [1]))
    if rng.random() < 0.5:  # single tokens
        seqs = _log_int(rng, 1, 64)
        new, most = 1, min(131072, 32 * 8192 * 8 * 128 // (seqs * kv_heads * dim))
    else:  # prompts, and chunks of them
        new = _log_int(rng, 2, 2048)
        seqs = _log_int(rng, 1, max(1, min(8, 4096 // new)))
        most = max(new, min(32768, 2048 * 2048 * 32 // (seqs * new * c["heads"]),
                            32 * 8192 * 8 * 128 // (seqs * kv_heads * dim)))
    ctx = _log_int(rng, new, most)
    window = _log_int(rng, 1, 4096) if rng.random() < 0.4 else 0
    return dict(c, seqs=seqs, new=new, ctx=ctx, window=window,
                sinks=rng.choice([0, 1, 4, 64]) if window else 0)


def _lengths(case):
    """The sequences' lengths and numbers of new tokens: the longest first, the
    others spread below it; they go by the case alone."""
    lens, news = [], []
    for s in range(case["seqs"]):
        part = 1.0 - 0.75 * ((s * 0.6180339887) % 1.0)
        lens.append(max(1, int(case["ctx"] * part)))
        news.append(lens[-1] if case["op"] == "read" else
                    min(lens[-1], max(1, int(case["new"] * part))))
    return lens, news


def _quantise(x):
    """The codes, two to a byte, and scale bytes of x in blocks of 32."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    scale = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 2).clamp(1, 252)
    a = b.abs() * ((254 - scale) << 23).view(torch.float32).unsqueeze(-1)
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) +
            (a >= 3.5) + (a > 5.0) + 8 * torch.signbit(b).to(torch.uint8))
    scale = torch.where(torch.isfinite(top), scale, 255)
    return code[..., 0::2] + 16 * code[..., 1::2], scale.to(torch.uint8)


def _values(codes, scale):
    """What codes [..., 16 bytes] and scales [...] stand for, in 32 bits."""
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    s = (scale.to(torch.int32) << 23).view(torch.float32)
    return levels[both] * torch.where(scale == 255, torch.nan, s).unsqueeze(-1)


def _parts(pool, dim):
    """The codes [pages, heads, tiles, 2, blocks, 16 tokens, 16 bytes] and scales
    [pages, heads, tiles, 2, blocks, 16 tokens] of a pool."""
    blocks = dim // 32
    tiles = pool.unflatten(-1, (-1, 17 * dim))
    return (tiles[..., :16 * dim].unflatten(-1, (2, blocks, 16, 16)),
            tiles[..., 16 * dim:].unflatten(-1, (2, blocks, 16)))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    if case["op"] == "norm":
        M, N = case["M"], case["N"]
        branch = DTYPES[case["y"]]
        return dict(
            op="norm", y=normal(M, N, dtype=branch) * 0.5,
            residual=(normal(M, N) * 2.0).to(DTYPES[case["res"]]),
            post=(1 + 0.1 * normal(N)).bfloat16() if case["post"] else None,
            gate=None if case["gate"] == "none" else
            torch.sigmoid(normal(*((M, N) if case["gate"] == "token" else (N,)))).to(branch),
            pre=(1 + 0.1 * normal(N)).bfloat16(), out=DTYPES[case["out"]], scale=0.75, eps=1e-6)
    lens, news = _lengths(case)
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    # whole pages of every sequence, in any order in the pool
    used = torch.tensor([-(-n // page) for n in lens], device="cuda")
    pages = int(used.sum())
    at = torch.arange(int(used.max()), device="cuda").expand(len(lens), -1)
    held = at < used[:, None]
    table = torch.zeros(at.shape, dtype=torch.int32, device="cuda")
    table[held] = torch.randperm(pages, generator=gen, device="cuda").int()
    # keys have channels that are larger than the others, values have not
    wide = 1 + 3 * (torch.rand(heads, 1, dim, generator=gen, device="cuda") < 0.05)
    pool = torch.empty(pages, heads, page // 16 * 17 * dim, dtype=torch.uint8, device="cuda")
    codes, scales = _parts(pool, dim)
    for first in range(0, pages, 4096 * 8 * 64 // (heads * page) + 1):
        some = slice(first, first + 4096 * 8 * 64 // (heads * page) + 1)
        for part, big in ((0, wide), (1, 1.0)):
            shape = (*codes[some].shape[:2], page, dim)
            c, s = _quantise((normal(*shape) * big).bfloat16())  # [page, head, token, block, 16]
            codes[some, :, :, part] = c.unflatten(2, (-1, 16)).transpose(3, 4)
            scales[some, :, :, part] = s.unflatten(2, (-1, 16)).transpose(3, 4)
    tokens = sum(news)
    state = dict(
        op=case["op"], pool=pool, table=table, tokens=tokens, dim=dim, page=page,
        lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
        starts=None if max(news) == 1 else torch.tensor(
            [sum(news[:s]) for s in range(len(news) + 1)], dtype=torch.int32, device="cuda"),
        max_len=max(lens), max_new=max(news))
    if case["op"] == "append":
        # keys and values as slices of one product's result, as a layer has them
        kv = normal(tokens, 2 * heads, dim, dtype=torch.bfloat16)
        state.update(k=kv[:, :heads], v=kv[:, heads:])
    elif case["op"] == "attend":
        state.update(q=normal(tokens, case["heads"], dim, dtype=torch.bfloat16),
                     window=case["window"], sinks=case["sinks"], scale=dim ** -0.5)
    return state


def _places(s):
    """The new tokens' sequence, number in it and position; then their page,
    tile and token in the tile."""
    t = torch.arange(s["tokens"], device="cuda")
    starts = torch.arange(s["tokens"] + 1, device="cuda") if s["starts"] is None else s["starts"]
    seq = torch.searchsorted(starts, t.to(starts.dtype), right=True) - 1
    i = t - starts[seq]
    pos = s["lens"][seq] - (starts[seq + 1] - starts[seq]) + i
    page, off = s["table"][seq, (pos // s["page"]).long()].long(), (pos % s["page"]).long()
    return seq, i.long(), pos, (page, off // 16, off % 16)


def _plain_norm(s):
    y = s["y"].float()
    if s["post"] is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + s["eps"]) * s["post"].float()
    if s["gate"] is not None:
        y = y * s["gate"].float()
    h = s["residual"].float() + s["scale"] * y
    n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"]) * s["pre"].float()
    return h.to(s["residual"].dtype), n.to(s["out"])


def _plain_read(s):
    codes, scales = _parts(s["pool"], s["dim"])
    page, tile, tok = _places(s)[3]
    got = _values(codes[page, :, tile, :, :, tok], scales[page, :, tile, :, :, tok])
    k, v = got.flatten(-2).bfloat16().unbind(2)  # [tokens, heads, 2, dim]
    return k, v


def _plain_append(s):
    codes, scales = _parts(s["pool"], s["dim"])
    page, tile, tok = _places(s)[3]
    c, e = _quantise(torch.stack((s["k"], s["v"]), 2))  # [tokens, heads, 2, blocks(, 16)]
    codes[page, :, tile, :, :, tok] = c
    scales[page, :, tile, :, :, tok] = e
    return _plain_read(s)


def _plain_attend(s):
    q, longest, most = s["q"], s["max_len"], s["max_new"]
    codes, scales = _parts(s["pool"], s["dim"])
    seqs, pages = s["table"].shape
    table = s["table"].long()
    # [sequence, page, head, tile, 2, block, token, 32] -> [2, sequence, head, position, dim]
    kv = _values(codes[table], scales[table]).permute(4, 0, 2, 1, 3, 6, 5, 7)
    kv = kv.reshape(2, seqs, kv.shape[2], pages * s["page"], s["dim"])[:, :, :, :longest]
    j = torch.arange(longest, device="cuda")
    inside = (j < s["lens"][:, None])[:, None, :, None]
    k, v = torch.where(inside, kv, 0.0).unbind(0)
    # queries [sequence, key head, new token x its query heads, dim]
    seq, i, pos, _ = _places(s)
    heads = k.shape[1]
    group = q.shape[1] // heads
    wide = torch.zeros(seqs, most, *q.shape[1:], device="cuda")
    wide[seq, i] = q.float()
    wide = wide.unflatten(2, (heads, group)).transpose(1, 2).flatten(2, 3)
    at = torch.full((seqs, most), -1, dtype=torch.int32, device="cuda")
    at[seq, i] = pos.int()
    p = at[:, :, None]
    seen = (j <= p) & ((j > p - s["window"]) | (j < s["sinks"])) if s["window"] else j <= p
    seen = seen.repeat_interleave(group, 1)[:, None]
    score = torch.where(seen, (wide @ k.transpose(2, 3)) * s["scale"], -torch.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = (weight @ v) / torch.where(total == 0, 1.0, total)
    out = out.unflatten(2, (most, group)).transpose(1, 2).flatten(2, 3)
    return out[seq, i].to(q.dtype)


def run(state):
    s = state
    if not own:
        return {"norm": _plain_norm, "append": _plain_append, "read": _plain_read,
                "attend": _plain_attend}[s["op"]](s)
    import dslcompiler_amd as llk
    if s["op"] == "norm":
        return llk.block_norm(s["y"], s["residual"], s["pre"], post_weight=s["post"],
                              gate=s["gate"], scale=s["scale"], eps=s["eps"], out_dtype=s["out"])
    if s["op"] == "append":
        llk.kv4_write(s["k"], s["v"], s["pool"], s["table"], s["lens"], starts=s["starts"])
    if s["op"] in ("append", "read"):
        return llk.kv4_read(s["pool"], s["table"], s["lens"], head_dim=s["dim"],
                            starts=s["starts"], tokens=s["tokens"])
    return llk.kv4_attention(s["q"], s["pool"], s["table"], s["lens"], starts=s["starts"],
                             scale=s["scale"], window=s["window"], sinks=s["sinks"],
                             max_len=s["max_len"])


def _visible(case):
    """For each sequence the cached positions that its new tokens see, and the
    pairs of a new token and a position that it sees."""
    for n, new in zip(*_lengths(case)):
        w, sinks = case["window"], case["sinks"]
        first = n - new  # position of the first new token
        low = max(0, first - w + 1) if w else 0
        pairs = 0
        for p in range(first, n):
            low_p = max(0, p - w + 1) if w else 0
            pairs += p + 1 - low_p + min(sinks, low_p)
        yield n - low + min(sinks, low), pairs


def work(case):
    if case["op"] == "norm":
        M, N = case["M"], case["N"]
        size = {"bf16": 2, "f32": 4}
        y, res, out = (size[case[k]] for k in ("y", "res", "out"))
        gate = {"none": 0, "channel": N, "token": M * N}[case["gate"]]
        return {"bytes": M * N * (y + 2 * res + out) + gate * y + 2 * N * (2 if case["post"] else 1),
                "flops": M * N * (6 + 4 * case["post"])}
    lens, news = _lengths(case)
    T, D, H = sum(news), case["dim"], case["kv_heads"]
    packed = T * H * 2 * (D // 2 + D // 32)
    whole = T * H * 2 * D * 2
    if case["op"] == "append":  # read, pack, read the packed, write
        return {"bytes": 2 * whole + 2 * packed, "flops": 4 * T * H * 2 * D}
    if case["op"] == "read":
        return {"bytes": whole + packed, "flops": T * H * 2 * D}
    keys, pairs = (sum(x) for x in zip(*_visible(case)))
    return {"bytes": 2 * T * case["heads"] * D * 2 + keys * H * 2 * (D // 2 + D // 32),
            "flops": 4 * pairs * case["heads"] * D}


# ---- the definition, in 64 bits -------------------------------------------


def _exact_blocks(x):
    """What each block of 32 of x stands for once quantised."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    a = b.abs().max(-1, keepdim=True).values
    mant, exp = torch.frexp(a)  # a = mant * 2^exp, mant in [0.5, 1)
    e = (exp - torch.where(mant <= 0.875, 3, 2)).clamp(-126, 125)
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), e)
    level = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    # nearest level; of two as near, the one of even index: even ones are asked first
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device=x.device)
    best, dist = torch.zeros_like(b), torch.full_like(b, torch.inf)
    for k in order.tolist():
        d = (b.abs() / unit - level[k]).abs()
        best = torch.where(d < dist, level[k], best)
        dist = torch.minimum(d, dist)
    return (torch.copysign(best, b) * unit).reshape(x.shape)


def _exact_cached(s, q, part):
    """Keys (part 0) or values (1) of sequence q's positions: [positions, heads, dim]."""
    n, page, blocks, D = int(s["lens"][q]), s["page"], s["dim"] // 32, s["dim"]
    ids = s["table"][q, :-(-n // page)].long()
    raw = s["pool"][ids].reshape(len(ids), s["pool"].shape[1], page // 16, 17 * D)
    half = 8 * D
    byte = raw[..., part * half:(part + 1) * half].reshape(*raw.shape[:3], blocks, 16, 16)
    exp = raw[..., 2 * half + part * D // 2:2 * half + (part + 1) * D // 2]
    exp = exp.reshape(*raw.shape[:3], blocks, 16).double() - 127.0
    level = torch.tensor(LEVELS, dtype=torch.float64, device=raw.device)
    out = torch.empty(*byte.shape[:-1], 32, dtype=torch.float64, device=raw.device)
    for shift in (0, 4):
        nib = (byte >> shift) & 15
        out[..., shift // 4::2] = level[(nib & 7).long()] * torch.where(nib > 7, -1.0, 1.0)
    out = out * torch.exp2(exp)[..., None]
    return out.permute(0, 2, 4, 1, 3, 5).reshape(-1, raw.shape[1], D)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "norm":
        y, h = s["y"].double(), s["residual"].double()
        if s["post"] is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + s["eps"]).sqrt() * s["post"].double()
        h = h + s["scale"] * (y if s["gate"] is None else y * s["gate"].double())
        return h, h / (h.pow(2).sum(-1, keepdim=True) / h.shape[-1] + s["eps"]).sqrt() * s["pre"].double()
    lens, news = _lengths(case)
    if s["op"] == "append":
        return _exact_blocks(s["k"]), _exact_blocks(s["v"])
    if s["op"] == "read":
        return tuple(torch.cat([_exact_cached(s, q, part) for q in range(len(lens))])
                     for part in (0, 1))
    outs, first = [], 0
    for q, (n, new) in enumerate(zip(lens, news)):
        k, v = _exact_cached(s, q, 0), _exact_cached(s, q, 1)
        asked = s["q"][first:first + new].double()
        first += new
        p = torch.arange(n - new, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None]
        hidden = j > p
        if s["window"]:
            hidden |= (j <= p - s["window"]) & (j >= s["sinks"])
        group = asked.shape[1] // k.shape[1]
        heads = []
        for h in range(asked.shape[1]):
            w = (asked[:, h] @ k[:, h // group].T.contiguous() * s["scale"]).masked_fill(hidden, -torch.inf)
            heads.append(torch.softmax(w, -1) @ v[:, h // group].contiguous())
        outs.append(torch.stack(heads, 1))
    return torch.cat(outs)
