"""Rotary positions against their definition with angles in extended precision.

Bound.  The angle is kept to 2^-32 of a turn and rounded to fp32 (half of 2^-24 of
at most half a turn): within 2^-25.9 of a turn, 2^-23.2 rad.  sincospif is within 4
ulp of at most 1 (2^-22), times the factor one rounding of 2^-24, and the two
products and their sum three more: |error| <= (|a| + |b|) factor 2^-20.8, and the
result's rounding."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

STEP = {"bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}


def reference(x, pos, table, interleaved, inverse=False):
    """(result, bound before rounding) in float64."""
    x = x.double().cpu().numpy()
    p = pos.cpu().numpy().astype(np.longdouble)
    angle = p[:, None] * np.array(table.frequencies, np.longdouble)
    two_pi = np.longdouble("6.283185307179586476925286766559")
    angle = (angle - two_pi * np.rint(angle / two_pi)).astype(np.float64)[:, None]
    c, s = np.cos(angle), np.sin(angle) * (-1 if inverse else 1)
    rot, f = table.rotary_dim, table.attention_factor
    first = np.s_[..., 0:rot:2] if interleaved else np.s_[..., :rot // 2]
    second = np.s_[..., 1:rot:2] if interleaved else np.s_[..., rot // 2:rot]
    a, b = x[first], x[second]
    out, most = x.copy(), np.zeros_like(x)
    out[first], out[second] = (a * c - b * s) * f, (b * c + a * s) * f
    most[first] = most[second] = (np.abs(a) + np.abs(b)) * f * 2.0 ** -20.8
    return out, most


def check(got, want, most):
    step = STEP[str(got.dtype).split(".")[1]]
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= most * (1 + step) + step * np.abs(want) * (most > 0)).all(), err.max()


def make(torch, T, heads, dim, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, heads, dim, generator=gen, device="cuda").to(dtype)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,heads,kv,dim,rot", [
    (1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (3, 7, 7, 80, 22), (5, 4, 1, 64, 32), (17, 3, 2, 96, 34),
    (64, 8, 2, 256, 256), (130, 5, 5, 128, 64), (700, 2, 1, 128, 16), (1500, 3, 1, 64, 64),
    (2, 2, 2, 1024, 1024), (600, 1, 1, 18, 16), (9, 4, 4, 127, 64)])
def test_rotary(llk, gpu, T, heads, kv, dim, rot, interleaved):
    table = llk.RotaryTable(rot)
    rng = np.random.default_rng(T)
    pos = rng.integers(0, 1 << 20, T).astype(np.int32)
    pos[0] = 0
    pos = gpu.from_numpy(pos).cuda()
    for dtype in (gpu.bfloat16, gpu.float32):
        q, k = make(gpu, T, heads, dim, dtype, 1), make(gpu, T, kv, dim, dtype, 2)
        a, b = llk.rotary(q, k, pos, table, interleaved=interleaved)
        for got, x in ((a, q), (b, k)):
            want, most = reference(x, pos, table, interleaved)
            check(got, want, most)
            assert gpu.equal(got[..., rot:], x[..., rot:])
        assert gpu.equal(a[0], q[0]) and gpu.equal(b[0], k[0])  # position 0
        alone, none = llk.rotary(q, None, pos, table, interleaved=interleaved)
        assert none is None and gpu.equal(alone, a)
        llk.rotary(q, k, pos, table, interleaved=interleaved, q_out=q, k_out=k)  # in place
        assert gpu.equal(q, a) and gpu.equal(k, b)


def test_far_and_negative_positions(llk, gpu):
    table = llk.RotaryTable(64, base=10000.0)
    pos = gpu.tensor([2 ** 31 - 1, -2 ** 31, -1, 1, 131072, 1 << 20, 10 ** 9, -12345],
                     dtype=gpu.int32, device="cuda")
    q = make(gpu, 8, 3, 64, gpu.float32)
    for interleaved in (False, True):
        got, _ = llk.rotary(q, None, pos, table, interleaved=interleaved)
        check(got, *reference(q, pos, table, interleaved))


@pytest.mark.parametrize("scaling", ["linear", "base", "yarn", "bands"])
def test_scalings(llk, gpu, scaling):
    table = llk.RotaryTable(128, base=500000.0, scaling=scaling, factor=8.0, trained=8192)
    pos = gpu.arange(65000, 65050, dtype=gpu.int32, device="cuda")
    q = make(gpu, 50, 4, 128, gpu.float32)
    got, _ = llk.rotary(q, None, pos, table)
    check(got, *reference(q, pos, table, False))


def test_own_frequencies(llk, gpu):
    f = [1.0, -0.25, 7.5, 0.0, 1e-9, 3e4]
    table = llk.RotaryTable.from_frequencies(f, attention_factor=0.5)
    assert table.rotary_dim == 12
    pos = gpu.tensor([0, 5, 100000], dtype=gpu.int32, device="cuda")
    q = make(gpu, 3, 2, 16, gpu.float32)
    got, _ = llk.rotary(q, None, pos, table)
    check(got, *reference(q, pos, table, False))


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(llk, gpu, interleaved):
    """inverse=True is the transpose of the call without it (the formula, and
    differences of a linear map), and undoes it where the factor is 1."""
    T, heads, dim, rot = 5, 2, 24, 16
    pos = gpu.tensor([0, 1, 77, 4000, -3], dtype=gpu.int32, device="cuda")
    for kw in ({}, dict(scaling="yarn", factor=16.0, trained=2048)):
        table = llk.RotaryTable(rot, **kw)
        f = table.attention_factor
        x, g = make(gpu, T, heads, dim, gpu.float32, 1), make(gpu, T, heads, dim, gpu.float32, 2)
        back, _ = llk.rotary(g, None, pos, table, interleaved=interleaved, inverse=True)
        check(back, *reference(g, pos, table, interleaved, inverse=True))
        y, _ = llk.rotary(x, None, pos, table, interleaved=interleaved)
        # <g, R x> = <R^T g, x>; each side's terms are within 2^-20 of their size
        left, right = (g.double() * y.double()).sum(), (back.double() * x.double()).sum()
        size = (g.double().abs() * y.double().abs() + back.double().abs() * x.double().abs()).sum()
        assert abs(left - right) <= size * 2.0 ** -19 * max(f, 1)
        # central differences of the map along each pair's values: R e, an exact column
        one = gpu.zeros(T, heads, dim, device="cuda")
        for d in range(dim):
            one.zero_()
            one[..., d] = 1
            up, _ = llk.rotary(x + 0.5 * one, None, pos, table, interleaved=interleaved)
            down, _ = llk.rotary(x - 0.5 * one, None, pos, table, interleaved=interleaved)
            got = ((up - down).double() * g.double()).sum(-1)
            near = (x.abs().double().sum(-1) + dim) * g.abs().double().sum(-1) * f * 2.0 ** -19
            assert ((got - back[..., d].double()).abs() <= near).all(), d
        if f == 1:
            again, _ = llk.rotary(y, None, pos, table, interleaved=interleaved, inverse=True)
            assert (again - x).abs().max() <= 4 * x.abs().max() * 2.0 ** -20


def test_strides_and_alignment(llk, gpu):
    """q and k as slices of one product's rows, heads before tokens, odd offsets;
    results into slices, beside which nothing changes."""
    T, H, D, rot = 33, 4, 64, 48
    table = llk.RotaryTable(rot)
    pos = gpu.arange(T, dtype=gpu.int32, device="cuda") * 37
    for dtype in (gpu.bfloat16, gpu.float32):
        for interleaved in (False, True):
            big = make(gpu, T, 3 * H, D + 3, dtype)
            q, k = big[:, :H, 1:1 + D], big[:, H:2 * H, 2:2 + D]
            want = llk.rotary(q.contiguous(), k.contiguous(), pos, table, interleaved=interleaved)
            got = llk.rotary(q, k, pos, table, interleaved=interleaved)
            assert gpu.equal(got[0], want[0]) and gpu.equal(got[1], want[1])
            turned = q.transpose(0, 1).contiguous().transpose(0, 1)
            out = gpu.full((H, T, D + 5), 3.0, device="cuda").to(dtype)
            got, _ = llk.rotary(turned, None, pos, table, interleaved=interleaved,
                                q_out=out.transpose(0, 1)[..., 5:])
            assert gpu.equal(got, want[0]) and (out[..., :5] == 3).all()
            rest = big.clone()
            llk.rotary(q, k, pos, table, interleaved=interleaved, q_out=q, k_out=k)
            assert gpu.equal(q, want[0]) and gpu.equal(k, want[1])
            for part in (np.s_[:, 2 * H:], np.s_[:, :, :1], np.s_[:, :H, 1 + D:]):
                assert gpu.equal(big[part], rest[part])


def test_values_that_are_not_finite_stay_in_their_pair(llk, gpu):
    table = llk.RotaryTable(32)
    pos = gpu.tensor([5, 9], dtype=gpu.int32, device="cuda")
    q = make(gpu, 2, 3, 40, gpu.bfloat16)
    want, _ = llk.rotary(q, None, pos, table)
    q[1, 2, 3], q[0, 1, 39] = float("nan"), float("inf")
    got, _ = llk.rotary(q, None, pos, table)
    assert got[1, 2, 3].isnan() and got[1, 2, 19].isnan() and got[0, 1, 39] == float("inf")
    want[1, 2, 3], want[1, 2, 19], want[0, 1, 39] = 0, 0, 0
    got[1, 2, 3], got[1, 2, 19], got[0, 1, 39] = 0, 0, 0
    assert gpu.equal(got, want)


def test_empty_streams_and_graph(llk, gpu):
    table = llk.RotaryTable(64)
    q = make(gpu, 6, 4, 64, gpu.bfloat16)
    pos = gpu.arange(6, dtype=gpu.int32, device="cuda")
    got, _ = llk.rotary(q[:0], None, pos[:0], table)
    assert got.shape == (0, 4, 64)
    a, b = llk.rotary(q, q[:, :0], pos, table)
    assert b.shape == (6, 0, 64) and gpu.equal(a, llk.rotary(q, None, pos, table)[0])
    side = gpu.cuda.Stream()
    out = gpu.empty_like(q)
    gpu.cuda.synchronize()
    llk.rotary(q, None, pos, table, q_out=out, stream=side)
    side.synchronize()
    assert gpu.equal(out, a)
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        llk.rotary(q, None, pos, table, q_out=out)
    for _ in range(3):
        pos += 1000
        graph.replay()
        assert gpu.equal(out, llk.rotary(q, None, pos, table)[0])
