"""Operators of a decode step with 4-bit weights and a bounded cache, as
measurable cases.

  matmul  q4_matmul: products with 4-bit weights and group scales
  swiglu  q4_swiglu: SiLU(X Wg) * (X Wu) on such weights
  rotary  rotary: rotary positions of q and k
  weigh   kv4_attention with marks: attention over the 4-bit paged cache that
          also adds up what weight each cached key gets
  evict   kv4_evict_plan, then kv4_evict: which slots of the cache stay, by that
          weight, and the cache moved together

4-bit weights.  W[k, n] = scale[k // group, n] * (code[k, n] - zero[k // group,
n]), codes and zeros 0..15 (zero 8 where there are none), the last group as long
as K leaves it.

Rotary positions.  Pair i of the first `rot` values of a head, at position p, is
turned by the angle p * f[i] and multiplied by a factor.  f[i] = base ** (-2 i /
rot), or scaled for long contexts:
  linear  f / s
  base    of the base base * s ** (rot / (rot - 2))
  yarn    r f / s + (1 - r) f, r rising from 0 to 1 between the pairs that turn
          32 times and once over the trained length; factor 0.1 ln s + 1
  bands   f / s for wavelengths above the trained length, f for those below a
          quarter of it, and in between by the wavelength
A pair is (i, i + rot / 2), or (2 i, 2 i + 1) where "interleaved".

The cache.  A block of 32 values of a token's key (value) is a scale byte E,
2^(E - 127), and 32 codes of 4 bits: a sign over an index into 0, 0.5, 1, 1.5,
2, 3, 4, 6.  16 consecutive tokens of a page and head lie together: key codes
[block][token][16 bytes], value codes, key scales [block][token], value scales.
The pool is [pages, heads, page / 16 such tiles]; table[s, i] names the page of
slots i * page on of sequence s, which holds lens[s] slots.  The last new[s] are
the call's tokens; the one in slot p sees slots 0 to p.

Marks.  weights[page, head, slot] is decay times what it was, plus the weights
that the call's tokens' query heads give to the slot; positions[page, head,
slot] the position its token came from.  Of a head's first lens[s] slots `keep`
stay: those among the last `recent` positions and the first `first`, then those
of the largest weights (ties to the lowest slot).  Slots below `keep` that stay
are not moved; the others below `keep`, in order, take those from `keep` on that
stay, in order.
"""
import math

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TRAINED = 8192  # positions a model was trained on, where its frequencies are scaled


def listed():
    return [
        # One decoded token through the output projection of an 8B-class layer.
        dict(name="matmul m1 4096", op="matmul", M=1, K=4096, N=4096, group=128, zeros=False,
             scales="bf16", out="bf16", add=False),
        # Five sequences' tokens through a 13B-class down projection, added to an
        # fp32 residual stream; asymmetric groups of 64.
        dict(name="matmul += m5 13824", op="matmul", M=5, K=13824, N=5120, group=64, zeros=True,
             scales="f16", out="f32", add=True),
        # A chunk of a prompt through the same projection, ragged.
        dict(name="matmul m255 13824", op="matmul", M=255, K=13824, N=5120, group=128, zeros=True,
             scales="f16", out="bf16", add=False),
        # One decoded token through an 8B-class MLP's gate and up projections.
        dict(name="swiglu m1 14336", op="swiglu", M=1, K=4096, N=14336, group=128, zeros=True,
             scales="bf16", out="bf16", add=False),
        # A decode batch of 17 through a 13B-class one, groups of 32.
        dict(name="swiglu m17 13824", op="swiglu", M=17, K=5120, N=13824, group=32, zeros=False,
             scales="bf16", out="bf16", add=False),
        # A decode step of 64 sequences at positions to 32768, scaled by bands.
        dict(name="rotary t64", op="rotary", T=64, heads=32, kv_heads=8, dim=128, rot=128,
             interleaved=False, scaling="bands", stretch=4.0, far=32768, type="bf16"),
        # A long prompt's chunk far into a context of a million, half of each
        # head, interleaved pairs.
        dict(name="rotary t4097 far", op="rotary", T=4097, heads=40, kv_heads=40, dim=128, rot=64,
             interleaved=True, scaling="yarn", stretch=128.0, far=1048576, type="bf16"),
        # One decoded token of one short sequence: the latency of a step.
        dict(name="weigh decode s1", op="weigh", seqs=1, new=1, ctx=1000, heads=32, kv_heads=8,
             dim=128, page=64, decay=0.0),
        # A decode step of 64 ragged sequences, sums kept from step to step (the
        # pass begins with a copy of them, so that each begins from the same).
        dict(name="weigh decode s64", op="weigh", seqs=64, new=1, ctx=8192, heads=32, kv_heads=8,
             dim=128, page=64, decay=1.0),
        # A prompt of 2048 tokens, a key head to each query head.
        dict(name="weigh prompt 2048", op="weigh", seqs=1, new=2048, ctx=2048, heads=32,
             kv_heads=32, dim=128, page=64, decay=0.0),
        # One sequence a little beyond its bound, as after a few decoded tokens;
        # the marks move with the cache (they are copied first, as above).
        dict(name="evict s1", op="evict", seqs=1, ctx=1055, kv_heads=8, dim=128, page=64, keep=1024,
             recent=128, first=4, marks=True),
        # 64 ragged sequences cut to a quarter of the longest, once and for all:
        # the marks are not needed any more.
        dict(name="evict s64", op="evict", seqs=64, ctx=8192, kv_heads=8, dim=128, page=64,
             keep=2048, recent=256, first=4, marks=False),
    ]


def _log_int(rng, lo, hi):
    """A number from lo to hi, even over their logarithm: above 64 an odd one or a
    multiple of 40."""
    n = min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    if n > 64:
        n = n // 40 * 40 if rng.random() < 0.5 else (n - 1) | 1
    return max(lo, n)


def draw(rng):
    op = rng.choices(["matmul", "swiglu", "rotary", "weigh", "evict"], [30, 15, 15, 25, 15])[0]
    if op in ("matmul", "swiglu"):
        M = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 2, 255)])
        K = rng.choice([2048, 4096, 5120, 13824, _log_int(rng, 512, 13824)])
        most = 13824 * 5120 * 255 // (K * max(M, 32)) // (2 if op == "swiglu" else 1)
        N = min(rng.choice([1376, 4096, 5120, 11008, 14336, _log_int(rng, 512, 14336)]), most)
        out = rng.choice(["bf16", "bf16", "f32"] if op == "swiglu" else ["bf16", "f16", "f32"])
        return dict(op=op, M=M, K=K, N=N, group=rng.choice([32, 64, 128, 128]),
                    zeros=rng.random() < 0.5, scales=rng.choice(["bf16", "f16"]), out=out,
                    add=op == "matmul" and rng.random() < 0.3)
    if op == "rotary":
        dim = rng.choice([64, 80, 128, 128, 256])
        heads, kv = rng.choice([(32, 8), (32, 32), (40, 40), (16, 1), (7, 7)])
        return dict(op=op, T=min(_log_int(rng, 1, 8192), 4097 * 80 * 128 // ((heads + kv) * dim)),
                    heads=heads, kv_heads=kv, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, dim // 4 + 2]),
                    interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "base", "yarn", "bands"]),
                    stretch=rng.choice([2.0, 4.0, 32.0]), far=_log_int(rng, 2048, 1048576),
                    type=rng.choice(["bf16", "bf16", "f32"]))
    kv_heads, dim = rng.choice([(8, 128), (32, 128), (8, 64), (4, 64), (2, 256), (1, 128)])
    c = dict(op=op, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 256]))
    if op == "evict":
        ctx = _log_int(rng, 40, 16384)
        most = 64 * 8192 * 8 * 128 // (ctx * kv_heads * dim)
        keep = max(8, int(ctx * rng.choice([0.25, 0.5, 0.9, 0.99])))
        return dict(c, seqs=_log_int(rng, 1, max(1, min(64, most))), ctx=ctx, keep=keep,
                    recent=rng.choice([0, 1, keep // 8, keep // 2]), first=rng.choice([0, 1, 4]),
                    marks=rng.random() < 0.5)
    c.update(heads=kv_heads * rng.choice([1, 4, 5, 8] if kv_heads <= 8 else [1]),
             decay=rng.choice([0.0, 0.0, 0.75, 1.0]))
    if rng.random() < 0.6:  # single tokens
        seqs = _log_int(rng, 1, 64)
        new, most = 1, min(65536, 64 * 8192 * 8 * 128 // (seqs * kv_heads * dim))
    else:  # prompts, and chunks of them
        new = _log_int(rng, 2, 2048)
        seqs = _log_int(rng, 1, max(1, min(8, 4096 // new)))
        most = max(new, min(16384, 2048 * 2048 * 32 // (seqs * new * c["heads"]),
                            64 * 8192 * 8 * 128 // (seqs * kv_heads * dim)))
    return dict(c, seqs=seqs, new=new, ctx=_log_int(rng, new, most))


def _lengths(case):
    """The sequences' slots and new tokens: the longest first, the others spread
    below it; they go by the case alone."""
    lens, news = [], []
    for s in range(case["seqs"]):
        part = 1.0 - 0.75 * ((s * 0.6180339887) % 1.0)
        lens.append(max(1, int(case["ctx"] * part)))
        news.append(min(lens[-1], max(1, int(case.get("new", 1) * part))))
    return lens, news


def _frequencies(case):
    """(f, factor) of a rotary case, in 64 bits."""
    rot, s, base = case["rot"], case["stretch"], 500000.0
    i = torch.arange(rot // 2, dtype=torch.float64)
    if case["scaling"] == "base":
        base *= s ** (rot / (rot - 2))
    f = base ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        f = f / s
    if case["scaling"] == "yarn":
        def pair(turns):  # that turns so often over the trained length
            return rot * math.log(TRAINED / (2 * math.pi * turns)) / (2 * math.log(base))

        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        r = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return r * f / s + (1 - r) * f, 0.1 * math.log(s) + 1
    if case["scaling"] == "bands":
        part = ((TRAINED * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = (1 - part) * f / s + part * f
    return f, 1.0


def _quantise(x):
    """The codes, two to a byte, and scale bytes of x in blocks of 32."""
    b = x.float().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    scale = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 2).clamp(1, 252)
    a = b.abs() * ((254 - scale) << 23).view(torch.float32).unsqueeze(-1)
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) +
            (a >= 3.5) + (a > 5.0) + 8 * torch.signbit(b).to(torch.uint8))
    return code[..., 0::2] + 16 * code[..., 1::2], scale.to(torch.uint8)


def _parts(pool, dim):
    """The codes [pages, heads, tiles, 2, blocks, 16 tokens, 16 bytes] and scales
    [pages, heads, tiles, 2, blocks, 16 tokens] of a pool."""
    blocks = dim // 32
    tiles = pool.unflatten(-1, (-1, 17 * dim))
    return (tiles[..., :16 * dim].unflatten(-1, (2, blocks, 16, 16)),
            tiles[..., 16 * dim:].unflatten(-1, (2, blocks, 16)))


def _prepare_weights(case, gen):
    K, N, group = case["K"], case["N"], case["group"]
    groups = -(-K // group)
    sides = []
    for _ in range(2 if case["op"] == "swiglu" else 1):
        codes = torch.empty(K, N, dtype=torch.uint8, device="cuda")
        # codes of normally distributed weights, whose largest of a group is 15 or 0
        for k in range(0, K, 1024):
            n = torch.randn(min(1024, K - k), N, generator=gen, device="cuda")
            codes[k:k + 1024] = (8 + n * 2.8).round().clamp(0, 15).to(torch.uint8)
        scales = torch.rand(groups, N, generator=gen, device="cuda") * 0.5 + 0.75
        scales = (scales * K ** -0.5 / 2.8).to(DTYPES[case["scales"]])
        zeros = None
        if case["zeros"]:
            zeros = torch.randint(5, 12, (groups, N), generator=gen, device="cuda").to(torch.uint8)
        sides.append([codes, scales, zeros])
    x = torch.randn(case["M"], K, generator=gen, device="cuda").bfloat16()
    state = dict(op=case["op"], x=x, group=group, out=DTYPES[case["out"]], sides=sides, add=None)
    if case["add"]:
        state["add"] = torch.randn(case["M"], N, generator=gen, device="cuda").to(state["out"])
    if own:
        import dslcompiler_amd as llk
        state["packed"] = [llk.Q4Weights.from_codes(c, s, z, group=group) for c, s, z in sides]
    return state


def _prepare_rotary(case, gen):
    T, heads, kv = case["T"], case["heads"], case["kv_heads"]
    # q and k as slices of one product's result, as a layer has them
    qkv = torch.randn(T, heads + 2 * kv, case["dim"], generator=gen, device="cuda")
    qkv = qkv.to(DTYPES[case["type"]])
    if T <= 64:  # one token each of as many sequences
        pos = torch.randint(0, case["far"], (T,), generator=gen, device="cuda")
    else:  # a chunk that ends far out
        pos = torch.arange(T, device="cuda") + max(0, case["far"] - T)
    f, factor = _frequencies(case)
    state = dict(op="rotary", q=qkv[:, :heads], k=qkv[:, heads:heads + kv], pos=pos.int(),
                 f=f.cuda(), factor=factor, rot=case["rot"], interleaved=case["interleaved"])
    if own:
        import dslcompiler_amd as llk
        scaling = None if case["scaling"] == "none" else case["scaling"]
        state["table"] = llk.RotaryTable(case["rot"], base=500000.0, scaling=scaling,
                                         factor=case["stretch"], trained=TRAINED)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] in ("matmul", "swiglu"):
        return _prepare_weights(case, gen)
    if case["op"] == "rotary":
        return _prepare_rotary(case, gen)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

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
    step = 4096 * 8 * 64 // (heads * page) + 1
    for first in range(0, pages, step):
        some = slice(first, first + step)
        for part, big in ((0, wide), (1, 1.0)):
            shape = (*codes[some].shape[:2], page, dim)
            c, s = _quantise((normal(*shape) * big).bfloat16())  # [page, head, token, block, 16]
            codes[some, :, :, part] = c.unflatten(2, (-1, 16)).transpose(3, 4)
            scales[some, :, :, part] = s.unflatten(2, (-1, 16)).transpose(3, 4)
    tokens = sum(news)
    # attention weights are spread over orders of magnitude; few of them are equal
    weights = torch.exp(1.5 * normal(pages, heads, page)).bfloat16().float()
    state = dict(op=case["op"], pool=pool, table=table, dim=dim, page=page, weights=weights,
                 lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if case["op"] == "weigh":
        state.update(
            q=normal(tokens, case["heads"], dim, dtype=torch.bfloat16), tokens=tokens,
            max_len=max(lens), max_new=max(news), scale=dim ** -0.5, decay=case["decay"],
            starts=None if max(news) == 1 else torch.tensor(
                [sum(news[:s]) for s in range(len(news) + 1)], dtype=torch.int32, device="cuda"))
        return state
    # positions of a cache that lost tokens before: slots from half of `keep` on
    # in order, those below it in any order, and gaps
    keep = case["keep"]
    positions = torch.zeros(pages, heads, page, dtype=torch.int32, device="cuda")
    for s, n in enumerate(lens):
        gaps = torch.randint(1, 4, (heads, n), generator=gen, device="cuda")
        pos = gaps.cumsum(1) - gaps[:, :1]
        mixed = min(keep // 2, n)
        order = torch.rand(heads, mixed, generator=gen, device="cuda").argsort(1)
        pos[:, :mixed] = pos[:, :mixed].gather(1, order)
        j = torch.arange(n, device="cuda")
        positions[table[s, j // page].long(), :, j % page] = pos.T.int()
    state.update(positions=positions, keep=keep, recent=case["recent"], first=case["first"],
                 max_len=max(lens), marks=case["marks"])
    return state


def _dense(side, group, K):
    codes, scales, zeros = side
    c = codes.float()
    z = 8.0 if zeros is None else zeros.float().repeat_interleave(group, 0)[:K]
    return (c - z) * scales.float().repeat_interleave(group, 0)[:K]


def _plain_product(s):
    x = s["x"].float()
    y = x @ _dense(s["sides"][0], s["group"], x.shape[1])
    if s["op"] == "swiglu":
        y = y / (1 + torch.exp(-y)) * (x @ _dense(s["sides"][1], s["group"], x.shape[1]))
    if s["add"] is not None:
        y = y + s["add"].float()
    return y.to(s["out"])


def _plain_rotary(s):
    angle = s["pos"].double()[:, None] * s["f"]  # far positions need 64 bits
    cos = (torch.cos(angle) * s["factor"]).float()[:, None]
    sin = (torch.sin(angle) * s["factor"]).float()[:, None]
    rot, out = s["rot"], []
    for x in (s["q"], s["k"]):
        y = x.clone()
        if s["interleaved"]:
            a, b = x[..., 0:rot:2].float(), x[..., 1:rot:2].float()
            y[..., 0:rot:2] = (a * cos - b * sin).to(y.dtype)
            y[..., 1:rot:2] = (b * cos + a * sin).to(y.dtype)
        else:
            a, b = x[..., :rot // 2].float(), x[..., rot // 2:rot].float()
            y[..., :rot // 2] = (a * cos - b * sin).to(y.dtype)
            y[..., rot // 2:rot] = (b * cos + a * sin).to(y.dtype)
        out.append(y)
    return tuple(out)


def _plain_weigh(s):
    longest, most, page = s["max_len"], s["max_new"], s["page"]
    codes, scales = _parts(s["pool"], s["dim"])
    seqs, pages = s["table"].shape
    table = s["table"].long()
    levels = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device="cuda")
    c = codes[table]
    both = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    kv = levels[both.int()] * (scales[table].to(torch.int32) << 23).view(torch.float32)[..., None]
    # [sequence, page, head, tile, 2, block, token, 32] -> [2, sequence, head, slot, dim]
    kv = kv.permute(4, 0, 2, 1, 3, 6, 5, 7)
    kv = kv.reshape(2, seqs, kv.shape[2], pages * page, s["dim"])[:, :, :, :longest]
    j = torch.arange(longest, device="cuda")
    inside = j < s["lens"][:, None]
    k, v = torch.where(inside[:, None, :, None], kv, 0.0).unbind(0)
    # the call's tokens: sequence, number in it, slot
    t = torch.arange(s["tokens"], device="cuda")
    starts = torch.arange(seqs + 1, device="cuda") if s["starts"] is None else s["starts"]
    seq = torch.searchsorted(starts, t.to(starts.dtype), right=True) - 1
    i = (t - starts[seq]).long()
    slot = s["lens"][seq] - (starts[seq + 1] - starts[seq]) + i
    heads = k.shape[1]
    group = s["q"].shape[1] // heads
    wide = torch.zeros(seqs, most, *s["q"].shape[1:], device="cuda")
    wide[seq, i] = s["q"].float()
    wide = wide.unflatten(2, (heads, group)).transpose(1, 2).flatten(2, 3)
    at = torch.full((seqs, most), -1, dtype=torch.int32, device="cuda")
    at[seq, i] = slot.int()
    seen = (j <= at[:, :, None]).repeat_interleave(group, 1)[:, None]
    score = torch.where(seen, (wide @ k.transpose(2, 3)) * s["scale"], -torch.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = e.sum(-1, keepdim=True)
    e = e / torch.where(total == 0, 1.0, total)
    out = (e @ v).unflatten(2, (most, group)).transpose(1, 2).flatten(2, 3)
    # what each slot gets, to its place in the pool
    sums = s["weights"].clone() if s["decay"] else s["weights"]
    q, n = inside.nonzero(as_tuple=True)
    place = (table[q, n // page], slice(None), n % page)
    got = e.sum(2)[q, :, n]
    sums[place] = s["decay"] * sums[place] + got if s["decay"] else got
    return out[seq, i].to(s["q"].dtype), sums


def _plain_evict(s):
    keep, page, heads = s["keep"], s["page"], s["weights"].shape[1]
    seqs = len(s["lens"])
    longest = max(s["max_len"], keep)
    j = torch.arange(longest, device="cuda")
    where = s["table"].long()[:, (j // page).clamp(max=s["table"].shape[1] - 1)]  # [sequence, slot]
    inside = (j < s["lens"][:, None])[:, None]
    w = s["weights"][where, :, j % page].transpose(1, 2)  # [sequence, head, slot]
    pos = s["positions"][where, :, j % page].transpose(1, 2)
    last = torch.where(inside, pos, -1).amax(-1, keepdim=True)
    safe = (pos > last - s["recent"]) | (pos < s["first"])
    w = torch.where(safe, torch.inf, w)
    order = torch.where(inside, w, -torch.inf).sort(dim=-1, descending=True, stable=True).indices
    stays = torch.zeros(seqs, heads, longest, dtype=torch.bool, device="cuda")
    stays.scatter_(2, order[..., :keep], True)
    stays &= inside
    # n-th hole below keep <- n-th kept slot from keep on
    source = torch.arange(keep, device="cuda").expand(seqs, heads, -1).clone()
    hole = ~stays[..., :keep] & inside[..., :keep]
    a, b, dst = hole.nonzero(as_tuple=True)
    src = stays[..., keep:].nonzero(as_tuple=True)[2] + keep
    source[a, b, dst] = src
    weights, positions = s["weights"], s["positions"]
    if s["marks"]:
        weights, positions = weights.clone(), positions.clone()
    pd, ps = where[a, dst], where[a, src]
    codes, scales = _parts(s["pool"], s["dim"])
    to, of = dst % page, src % page
    codes[pd, b, to // 16, :, :, to % 16] = codes[ps, b, of // 16, :, :, of % 16]
    scales[pd, b, to // 16, :, :, to % 16] = scales[ps, b, of // 16, :, :, of % 16]
    if s["marks"]:
        weights[pd, b, to], positions[pd, b, to] = weights[ps, b, of], positions[ps, b, of]
    return s["lens"].clamp(max=keep), source.int(), s["pool"], weights, positions


def run(state):
    s = state
    if not own:
        return {"matmul": _plain_product, "swiglu": _plain_product, "rotary": _plain_rotary,
                "weigh": _plain_weigh, "evict": _plain_evict}[s["op"]](s)
    import dslcompiler_amd as llk
    if s["op"] == "swiglu":
        return llk.q4_swiglu(s["x"], *s["packed"], out_dtype=s["out"])
    if s["op"] == "matmul":
        if s["add"] is None:
            return llk.q4_matmul(s["x"], *s["packed"], out_dtype=s["out"])
        return llk.q4_matmul(s["x"], *s["packed"], out=s["add"].clone(), accumulate=True)
    if s["op"] == "rotary":
        return llk.rotary(s["q"], s["k"], s["pos"], s["table"], interleaved=s["interleaved"])
    weights = s["weights"]
    if s["op"] == "weigh":
        weights = weights.clone() if s["decay"] else weights
        out = llk.kv4_attention(s["q"], s["pool"], s["table"], s["lens"], starts=s["starts"],
                                scale=s["scale"], max_len=s["max_len"], weights=weights,
                                decay=s["decay"])
        return out, weights
    lens, source = llk.kv4_evict_plan(weights, s["table"], s["lens"], s["keep"],
                                      positions=s["positions"], recent=s["recent"],
                                      first=s["first"], max_len=s["max_len"])
    positions = s["positions"]
    if s["marks"]:
        weights, positions = weights.clone(), positions.clone()
        llk.kv4_evict(s["pool"], s["table"], source, head_dim=s["dim"], weights=weights,
                      positions=positions)
    else:
        llk.kv4_evict(s["pool"], s["table"], source, head_dim=s["dim"])
    return lens, source, s["pool"], weights, positions


def _moved(case):
    """Slots that move, of every head, if those that stay lie evenly over all but
    the protected ones: a number that goes by the case alone."""
    total = 0
    for n in _lengths(case)[0]:
        keep = case["keep"]
        if n > keep:
            safe = min(case["recent"], n - keep)  # newest, all beyond keep
            total += int(safe + max(0, n - keep - safe) * (keep - safe) / max(1, n - safe))
    return total


def work(case):
    if case["op"] in ("matmul", "swiglu"):
        M, K, N = case["M"], case["K"], case["N"]
        sides = 2 if case["op"] == "swiglu" else 1
        groups = -(-K // case["group"])
        out = 2 * M * N * DTYPES[case["out"]].itemsize if case["add"] else \
            M * N * DTYPES[case["out"]].itemsize
        weights = K * N / 2 + groups * N * (2.5 if case["zeros"] else 2)
        return {"bytes": int(sides * weights + 2 * M * K + out), "flops": 2 * sides * M * K * N}
    if case["op"] == "rotary":
        values = case["T"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * values * DTYPES[case["type"]].itemsize + 4 * case["T"],
                "flops": 3 * values}
    lens, news = _lengths(case)
    D, H = case["dim"], case["kv_heads"]
    if case["op"] == "evict":
        held = sum(min(n, case["keep"]) for n in lens) * H
        moved = _moved(case) * H
        return {"bytes": 8 * sum(lens) * H + 4 * held +
                2 * moved * (17 * D // 16 + (8 if case["marks"] else 0)),
                "flops": 2 * sum(lens) * H}
    pairs = sum(new * (n - new) + new * (new + 1) // 2 for n, new in zip(lens, news))
    return {"bytes": 4 * sum(news) * case["heads"] * D + sum(lens) * H * (17 * D // 16) +
            sum(lens) * H * (8 if case["decay"] else 4),
            "flops": 4 * pairs * case["heads"] * D}


# ---- the definition, in 64 bits -------------------------------------------


def _exact_product(s):
    x, outs = s["x"].double(), []
    for codes, scales, zeros in s["sides"]:
        y = torch.zeros(x.shape[0], codes.shape[1], dtype=torch.float64, device="cuda")
        for g in range(scales.shape[0]):
            rows = slice(g * s["group"], (g + 1) * s["group"])
            w = codes[rows].double() - (8 if zeros is None else zeros[g].double())
            y += x[:, rows] @ w * scales[g].double()
        outs.append(y)
    y = outs[0]
    if s["op"] == "swiglu":
        y = torch.sigmoid(y) * y * outs[1]
    return y if s["add"] is None else y + s["add"].double()


def _exact_rotary(s, case):
    f, factor = _frequencies(case)
    f, rot = f.cuda(), case["rot"]
    turn = torch.polar(torch.full_like(f, factor).expand(case["T"], -1),
                       s["pos"].double()[:, None] * f)[:, None]
    out = []
    for x in (s["q"].double(), s["k"].double()):
        head, rest = x[..., :rot], x[..., rot:]
        pairs = head.unflatten(-1, (-1, 2)) if case["interleaved"] else \
            head.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        out.append(torch.cat((z.flatten(-2), rest), -1))
    return tuple(out)


def _exact_cached(s, q, part):
    """Keys (part 0) or values (1) of sequence q's slots: [slots, heads, dim]."""
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


def _exact_weigh(s, case):
    outs, first, sums = [], 0, s["weights"].double()
    for q, (n, new) in enumerate(zip(*_lengths(case))):
        k, v = _exact_cached(s, q, 0), _exact_cached(s, q, 1)
        asked = s["q"][first:first + new].double()
        first += new
        hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - new, n, device="cuda")[:, None]
        group = asked.shape[1] // k.shape[1]
        heads, got = [], torch.zeros(n, k.shape[1], dtype=torch.float64, device="cuda")
        for h in range(asked.shape[1]):
            w = (asked[:, h] @ k[:, h // group].T.contiguous() * s["scale"]).masked_fill(hidden, -torch.inf)
            w = torch.softmax(w, -1)
            got[:, h // group] += w.sum(0)
            heads.append(w @ v[:, h // group].contiguous())
        outs.append(torch.stack(heads, 1))
        for i in range(-(-n // s["page"])):
            some = got[i * s["page"]:(i + 1) * s["page"]].T
            at = sums[int(s["table"][q, i]), :, :some.shape[1]]
            at.copy_(some + case["decay"] * at)
    return torch.cat(outs), sums


def _exact_evict(s, case):
    import numpy as np
    table, page = s["table"].cpu().numpy(), s["page"]
    w, pos = s["weights"].cpu().numpy().copy(), s["positions"].cpu().numpy().copy()
    pool, keep, D = s["pool"].cpu().numpy().copy(), case["keep"], s["dim"]
    lens, heads = _lengths(case)[0], w.shape[1]
    source = np.tile(np.arange(keep, dtype=np.int32), (len(lens), heads, 1))
    tiles = pool.reshape(*pool.shape[:2], -1, 17 * D)
    for q, n in enumerate(lens):
        if n <= keep:
            continue
        j = np.arange(n)
        pages = table[q, j // page]
        for h in range(heads):
            ww, pp = w[pages, h, j % page], pos[pages, h, j % page]
            safe = (pp > pp.max() - case["recent"]) | (pp < case["first"])
            rank = np.lexsort((j, -ww.astype(np.float64), ~safe))  # safe first, large first
            stay = np.sort(rank[:keep])
            to = np.setdiff1d(np.arange(keep), stay)
            of = stay[stay >= keep]
            source[q, h, to] = of
            a, b, to, of = pages[to], pages[of], to % page, of % page
            if case["marks"]:
                w[a, h, to], pos[a, h, to] = w[b, h, of], pos[b, h, of]
            for first, width, count in ((0, 16, D // 16), (16 * D, 1, D // 16)):
                for c in range(count):
                    for x in range(width):
                        base = first + c * 16 * width + x
                        tiles[a, h, to // 16, base + to % 16 * width] = \
                            tiles[b, h, of // 16, base + of % 16 * width]
    return (torch.tensor(lens, dtype=torch.int32).clamp(max=keep).cuda(),
            *(torch.from_numpy(a).cuda() for a in (source, pool, w, pos)))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("matmul", "swiglu"):
        return _exact_product(s)
    if case["op"] == "rotary":
        return _exact_rotary(s, case)
    return _exact_weigh(s, case) if case["op"] == "weigh" else _exact_evict(s, case)
