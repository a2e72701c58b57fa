"""The fused residual norm against its formula in 64 bits: every combination of
types, with and without the norm after the block, the gate and y; odd sizes,
row strides and alignments; in place; on another stream and in a graph.

Bounds.  fp32: sums of N squares in fp32 (at most 32 terms in a chain, then a
tree) and a handful of roundings are within 2^-18 of the magnitudes that are
added; bf16 results are rounded once more, by at most 2^-8 of the value."""
from __future__ import annotations

import itertools

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _f64(t):
    return None if t is None else t.double().cpu().numpy()


def reference(y, h, pre, post=None, gate=None, scale=1.0, eps=EPS, offset=0.0):
    """(r, out, size of r's terms, size of out's error scale)."""
    y, h, pre, post, gate = map(_f64, (y, h, pre, post, gate))
    r, mag = h, np.abs(h)
    if y is not None:
        u = y
        if post is not None:
            u = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * (post + offset)
        if gate is not None:
            u = u * gate
        r, mag = h + scale * u, mag + np.abs(scale * u)
    f = 1 / np.sqrt((r * r).mean(-1, keepdims=True) + eps)
    return r, r * f * (pre + offset), mag, mag * f * np.abs(pre + offset)


def close(got, want, mag, what):
    bf16 = str(got.dtype) == "torch.bfloat16"
    got = _f64(got)
    bound = 2.0 ** -18 * mag + (2.0 ** -8 * np.abs(want) if bf16 else 0) + 1e-30
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], want[bad][:3])


def make(torch, M, N, y, h, w, post, gate, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, generator=g, device="cuda")

    return dict(y=(0.5 * rnd(M, N)).to(y), h=(2 * rnd(M, N)).to(h), pre=(1 + 0.1 * rnd(N)).to(w),
                post=(1 + 0.1 * rnd(N)).to(w) if post else None,
                gate={"none": None, "row": torch.sigmoid(rnd(N)).to(y),
                      "all": torch.sigmoid(rnd(M, N)).to(y)}[gate])


@pytest.mark.parametrize("yt,ht,ot,wt", list(itertools.product(("bf16", "f32"), repeat=4)))
def test_types(llk, gpu, yt, ht, ot, wt):
    T = {"bf16": gpu.bfloat16, "f32": gpu.float32}
    for post, gate in itertools.product((False, True), ("none", "row", "all")):
        x = make(gpu, 5, 1000, T[yt], T[ht], T[wt], post, gate)
        r, n = llk.block_norm(x["y"], x["h"], x["pre"], post_weight=x["post"], gate=x["gate"],
                              scale=0.75, weight_offset=0.5, out_dtype=T[ot])
        want_r, want_n, mr, mn = reference(x["y"], x["h"], x["pre"], x["post"], x["gate"], 0.75,
                                           offset=0.5)
        assert r.dtype == T[ht] and n.dtype == T[ot]
        close(r, want_r, mr, ("residual", post, gate))
        close(n, want_n, mn, ("out", post, gate))


@pytest.mark.parametrize("N", [1, 2, 7, 8, 9, 63, 64, 65, 511, 512, 513, 2047, 2049, 4096, 5120,
                               8191, 8193, 16385, 32767, 32768])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_sizes(llk, gpu, N, kind):
    t = {"bf16": gpu.bfloat16, "f32": gpu.float32}[kind]
    for M in (1, 3):
        x = make(gpu, M, N, t, t, gpu.bfloat16, True, "all", seed=N + M)
        r, n = llk.block_norm(x["y"], x["h"], x["pre"], post_weight=x["post"], gate=x["gate"],
                              out_dtype=t)
        want_r, want_n, mr, mn = reference(x["y"], x["h"], x["pre"], x["post"], x["gate"])
        close(r, want_r, mr, N)
        close(n, want_n, mn, N)


@pytest.mark.parametrize("N,pad,skip", [(1000, 3, 1), (777, 0, 5), (4096, 40, 8)])
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_strides_and_alignment(llk, gpu, N, pad, skip, kind):
    """Rows of a wider buffer that begin at any element; what lies beside them
    keeps its values."""
    t = {"bf16": gpu.bfloat16, "f32": gpu.float32}[kind]
    M = 7
    x = make(gpu, M, N, t, t, t, True, "all")

    def inside(v, fill):
        buf = gpu.full((M, N + pad + skip), fill, dtype=t, device="cuda")
        buf[:, skip:skip + N] = v
        return buf, buf[:, skip:skip + N]

    _, y = inside(x["y"], float("nan"))
    _, h = inside(x["h"], float("nan"))
    _, gate = inside(x["gate"], float("nan"))
    rbuf, r = inside(gpu.zeros_like(x["h"]), 5.0)
    obuf, o = inside(gpu.zeros_like(x["h"]), 6.0)
    wide = gpu.full((N + 3,), float("nan"), dtype=t, device="cuda")
    wide[1:N + 1] = x["pre"]
    got_r, got_n = llk.block_norm(y, h, wide[1:N + 1], post_weight=x["post"], gate=gate,
                                  residual_out=r, out=o)
    assert got_r is r and got_n is o
    want_r, want_n, mr, mn = reference(x["y"], x["h"], x["pre"], x["post"], x["gate"])
    close(r, want_r, mr, "residual")
    close(o, want_n, mn, "out")
    for buf, fill in ((rbuf, 5.0), (obuf, 6.0)):
        beside = gpu.cat((buf[:, :skip], buf[:, skip + N:]), 1)
        assert bool((beside == fill).all())


def test_in_place_and_without_y(llk, gpu):
    x = make(gpu, 9, 1376, gpu.bfloat16, gpu.float32, gpu.bfloat16, False, "none")
    want_r, want_n, mr, mn = reference(x["y"], x["h"], x["pre"])
    h, y = x["h"].clone(), x["y"].clone()
    r, n = llk.block_norm(y, h, x["pre"], residual_out=h, out=y)
    assert r is h and n is y
    close(h, want_r, mr, "residual in place")
    close(y, want_n, mn, "out over y")
    r, n = llk.block_norm(None, x["h"], x["pre"])
    assert r is x["h"]
    _, want_n, _, mn = reference(None, x["h"], x["pre"])
    close(n, want_n, mn, "norm alone")
    copy = gpu.empty_like(x["h"])
    llk.block_norm(None, x["h"], x["pre"], residual_out=copy)
    assert bool((copy == x["h"]).all())


def test_zero_rows_and_zero_values(llk, gpu):
    w = gpu.ones(64, device="cuda", dtype=gpu.bfloat16)
    e = gpu.empty((0, 64), device="cuda", dtype=gpu.bfloat16)
    r, n = llk.block_norm(e, e, w)
    assert r.shape == n.shape == (0, 64)
    z = gpu.zeros((2, 64), device="cuda", dtype=gpu.bfloat16)
    r, n = llk.block_norm(z, z, w, post_weight=w)
    assert bool((r == 0).all()) and bool((n == 0).all())  # rsqrt(eps) * 0


def test_non_finite_rows_stay_their_own(llk, gpu):
    x = make(gpu, 4, 300, gpu.bfloat16, gpu.bfloat16, gpu.bfloat16, True, "none")
    x["y"][1, 17] = float("nan")
    x["h"][2, 299] = float("inf")
    r, n = llk.block_norm(x["y"], x["h"], x["pre"], post_weight=x["post"])
    assert bool(gpu.isnan(r[1]).all()) and bool(gpu.isnan(n[1]).all())
    assert bool(gpu.isinf(r[2, 299])) and bool(gpu.isnan(n[2, 299]))
    keep = [0, 3]
    want_r, want_n, mr, mn = reference(x["y"][keep], x["h"][keep], x["pre"], x["post"])
    close(r[keep], want_r, mr, "residual")
    close(n[keep], want_n, mn, "out")


def test_stream_and_graph(llk, gpu):
    x = make(gpu, 33, 5120, gpu.bfloat16, gpu.float32, gpu.bfloat16, True, "row")

    def call():
        return llk.block_norm(x["y"], x["h"], x["pre"], post_weight=x["post"], gate=x["gate"])

    want = [t.clone() for t in call()]
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        got = call()
    explicit = llk.block_norm(x["y"], x["h"], x["pre"], post_weight=x["post"], gate=x["gate"],
                              stream=side)
    gpu.cuda.synchronize()
    for a, b, c in zip(want, got, explicit):
        assert gpu.equal(a, b) and gpu.equal(a, c)
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph):
        out = call()
    for k in range(3):
        x["h"].mul_(1.5)
        want = [t.clone() for t in call()]
        for t in out:
            t.zero_()
        graph.replay()
        gpu.cuda.synchronize()
        for a, b in zip(want, out):
            assert gpu.equal(a, b), k


def test_rows_beyond_one_launch(llk, gpu):
    """2^26 rows and more of narrow ones: 2^32 threads at a wave to a row, more
    than a dimension of one launch takes."""
    M, N = (1 << 26) + 3, 2
    h = gpu.zeros((M, N), dtype=gpu.bfloat16, device="cuda")
    at = [0, 1, (1 << 24) - 1, 1 << 24, (1 << 25) - 1, 1 << 25, (1 << 26) - 1, 1 << 26, M - 1]
    for i, m in enumerate(at):
        h[m, 0], h[m, 1] = 1 + i, -0.5 * i
    w = gpu.tensor([1.0, 2.0], device="cuda").bfloat16()
    y = h * 2
    r, n = llk.block_norm(y, h, w)
    want_r, want_n, mr, mn = reference(y[at], h[at], w)
    close(r[at], want_r, mr, "residual")
    close(n[at], want_n, mn, "out")
    assert int((r != 0).sum()) == int((h != 0).sum()) == int((n != 0).sum())
