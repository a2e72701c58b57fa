"""4-bit weights with group scales against their definition in 64 bits.

Exact cases: X of integers to 3 and scales of powers of two from 1/8 to 2, with
which every product and sum is a multiple of 2^-7 below 4104 * 3 * 2 * 2 < 2^16, so
fp32 adds without rounding: fp32 results are equal, bf16 and fp16 ones equal after
one rounding.

Bound of the others: a group's two sums have at most 128 terms of |x| (1 + c / 16)
<= 2 |x| and are scaled by 16 s, and with the groups, the waves and the result at
most 128 + K / 32 + 32 roundings of 2^-24 each of what has been summed:
|error| <= (160 + K / 32) 2^-24 64 sum(s |x|) before the rounding to the result's
type."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def case(torch, M, K, N, group, zeros, scale_dtype, seed, exact):
    """x bf16, codes, scales, zeros on the device."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda")

    groups = -(-K // group)
    codes = ints(0, 16, K, N).to(torch.uint8)
    z = ints(0, 16, groups, N).to(torch.uint8) if zeros else None
    if exact:
        x = ints(-3, 4, M, K).to(torch.bfloat16)
        scales = torch.exp2(ints(-3, 2, groups, N).float()).to(scale_dtype)
    else:
        x = torch.randn(M, K, generator=gen, device="cuda").bfloat16()
        scales = (torch.randn(groups, N, generator=gen, device="cuda") * 0.02).to(scale_dtype)
    return x, codes, scales, z


def dense(codes, scales, z, group):
    """W in float64."""
    K = codes.shape[0]
    rows = np.arange(K) // group
    c = codes.cpu().numpy().astype(np.float64)
    zero = 8.0 if z is None else z.cpu().numpy().astype(np.float64)[rows]
    return (c - zero) * scales.double().cpu().numpy()[rows]


def f64(t):
    return t.double().cpu().numpy()


def bound(x, scales, group, K):
    rows = np.arange(K) // group
    return (160 + K / 32) * 2.0 ** -24 * 64 * (np.abs(f64(x)) @ np.abs(f64(scales))[rows])


STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11, "float32": 2.0 ** -24}
SIZES = [(1, 128, 16), (1, 1, 1), (1, 4104, 48), (2, 7, 17), (3, 31, 100), (4, 32, 15), (5, 33, 16),
         (8, 64, 33), (9, 127, 16), (13, 129, 40), (16, 200, 64), (17, 1000, 72), (33, 640, 130),
         (64, 256, 96), (65, 300, 257), (100, 2048, 64), (129, 384, 272), (300, 520, 80)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_exact_products(llk, gpu, M, K, N, group):
    for zeros, st in ((False, gpu.bfloat16), (True, gpu.float16)):
        x, codes, scales, z = case(gpu, M, K, N, group, zeros, st, M * K + N, True)
        w = llk.Q4Weights.from_codes(codes, scales, z, group=group)
        want = f64(x) @ dense(codes, scales, z, group)
        got = llk.q4_matmul(x, w)
        assert got.dtype == gpu.float32 and got.shape == (M, N)
        assert np.array_equal(f64(got), want), (zeros, np.abs(f64(got) - want).max())
        exact32 = gpu.from_numpy(want).float().cuda()
        for t in (gpu.bfloat16, gpu.float16):
            assert gpu.equal(llk.q4_matmul(x, w, out_dtype=t), exact32.to(t))
        acc = gpu.full((M, N), 0.5, device="cuda")
        assert llk.q4_matmul(x, w, out=acc, accumulate=True) is acc
        assert np.array_equal(f64(acc), want + 0.5)


@pytest.mark.parametrize("M,K,N,group", [(1, 4096, 512, 128), (1, 13824, 96, 32), (4, 1000, 200, 64),
                                         (7, 5120, 130, 128), (16, 2048, 64, 32), (40, 777, 96, 64),
                                         (130, 4096, 64, 128), (255, 1000, 300, 32)])
def test_products(llk, gpu, M, K, N, group):
    for zeros, st in ((False, gpu.float16), (True, gpu.bfloat16)):
        x, codes, scales, z = case(gpu, M, K, N, group, zeros, st, K + N, False)
        w = llk.Q4Weights.from_codes(codes, scales, z, group=group)
        want = f64(x) @ dense(codes, scales, z, group)
        most = bound(x, scales, group, K)
        for t in (gpu.float32, gpu.bfloat16, gpu.float16):
            got = f64(llk.q4_matmul(x, w, out_dtype=t))
            step = STEP[str(t).split(".")[1]]
            # (fp16 below its normal range: half its smallest step)
            assert (np.abs(got - want) <= most * (1 + step) + step * np.abs(want) + 2.0 ** -25).all()
        first = gpu.randn(M, N, device="cuda").bfloat16()
        got = f64(llk.q4_matmul(x, w, out=first.clone(), accumulate=True))
        total = want + f64(first)
        assert (np.abs(got - total) <= most * 1.01 + 2.0 ** -8 * np.abs(total) + 2.0 ** -22).all()


@pytest.mark.parametrize("M,K,N,group", [(1, 4096, 272, 128), (1, 100, 16, 32), (3, 640, 100, 64),
                                         (8, 1000, 48, 32), (16, 512, 65, 128), (17, 5120, 96, 32),
                                         (64, 300, 128, 128), (150, 1024, 136, 64)])
def test_swiglu(llk, gpu, M, K, N, group):
    for zeros in (False, True):
        x, *g = case(gpu, M, K, N, group, zeros, gpu.bfloat16, 7 * K + N, False)
        _, *u = case(gpu, M, K, N, group, zeros, gpu.bfloat16, 7 * K + N + 1, False)
        x = (x.float() * 0.5).bfloat16()
        wg, wu = (llk.Q4Weights.from_codes(*s, group=group) for s in (g, u))
        a, b = f64(x) @ dense(*g, group), f64(x) @ dense(*u, group)
        ea, eb = bound(x, g[1], group, K), bound(x, u[1], group, K)
        silu = a / (1 + np.exp(-a))
        # SiLU's slope is below 1.1; the activation itself within 4 ulp
        most = 1.1 * ea * (np.abs(b) + eb) + np.abs(silu) * eb + 2.0 ** -21 * np.abs(silu * b)
        for t, step in ((gpu.float32, 2.0 ** -24), (gpu.bfloat16, 2.0 ** -8)):
            got = f64(llk.q4_swiglu(x, wg, wu, out_dtype=t))
            assert (np.abs(got - silu * b) <= most * (1 + step) + step * np.abs(silu * b) + 1e-30).all()


@pytest.mark.parametrize("M", [1, 5, 16, 40, 130])
def test_strides_and_alignment(llk, gpu, M):
    """X at any row stride and element alignment, Y as a slice: what lies beside
    it stays; codes, scales and zeros as slices."""
    K, N, group = 328, 72, 64
    x, codes, scales, z = case(gpu, M, K, N, group, True, gpu.bfloat16, M, True)
    want = gpu.from_numpy(f64(x) @ dense(codes, scales, z, group)).float().cuda()

    def wider(t, left, right):
        big = gpu.full((t.shape[0], t.shape[1] + left + right), 99, device="cuda").to(t.dtype)
        big[:, left:left + t.shape[1]] = t
        return big[:, left:left + t.shape[1]]

    w = llk.Q4Weights.from_codes(wider(codes, 3, 2), wider(scales, 1, 4), wider(z, 5, 1), group=group)
    for left, right in ((1, 0), (3, 4), (8, 8)):
        big = gpu.full((M + 2, N + 7), 5.0, device="cuda")
        llk.q4_matmul(wider(x, left, right), w, out=big[1:-1, 2:2 + N])
        assert gpu.equal(big[1:-1, 2:2 + N], want)
        big[1:-1, 2:2 + N] = 5.0
        assert (big == 5.0).all()


def test_empty(llk, gpu):
    x, codes, scales, z = case(gpu, 4, 64, 32, 32, False, gpu.bfloat16, 1, True)
    w = llk.Q4Weights.from_codes(codes, scales, z, group=32)
    assert llk.q4_matmul(x[:0], w).shape == (0, 32)
    none = llk.Q4Weights.from_codes(codes[:0], scales[:0], group=32)
    for M in (4, 40):
        some = gpu.zeros(M, 0, dtype=gpu.bfloat16, device="cuda")
        assert (llk.q4_matmul(some, none) == 0).all()
        assert (llk.q4_swiglu(some, none, none) == 0).all()
        acc = gpu.ones(M, 32, device="cuda")
        assert (llk.q4_matmul(some, none, out=acc, accumulate=True) == 1).all()
    narrow = llk.Q4Weights.from_codes(codes[:, :0], scales[:, :0], group=32)
    assert llk.q4_matmul(x, narrow).shape == (4, 0)


@pytest.mark.parametrize("M", [1, 6, 16, 50, 140])
def test_non_finite_rows_stay_in_their_row(llk, gpu, M):
    K, N, group = 200, 40, 64
    x, codes, scales, z = case(gpu, M, K, N, group, True, gpu.bfloat16, 3, True)
    w = llk.Q4Weights.from_codes(codes, scales, z, group=group)
    want = llk.q4_matmul(x, w)
    for bad in (float("inf"), float("nan")):
        y = x.clone()
        y[M // 2, 77] = bad
        got = llk.q4_matmul(y, w)
        assert got[M // 2].isnan().all()
        rest = [m for m in range(M) if m != M // 2]
        assert gpu.equal(got[rest], want[rest])
    # a scale that is not finite stays in its column
    s = scales.clone()
    s[1, 7] = float("nan")
    got = llk.q4_matmul(x, llk.Q4Weights.from_codes(codes, s, z, group=group))
    assert got[:, 7].isnan().all()
    keep = [n for n in range(N) if n != 7]
    assert gpu.equal(got[:, keep], want[:, keep])


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantise(llk, gpu, group):
    """Codes, scales and zeros against the rule in fp32, value for value."""
    gen = gpu.Generator(device="cuda").manual_seed(group)
    for K, N in ((1, 1), (130, 257), (300, 70)):
        w = gpu.randn(K, N, generator=gen, device="cuda").bfloat16()
        w[:, 0] = 0
        w[K // 2, N // 2] = 40.0
        if N > 5:
            w[0, 3], w[0, 4], w[0, 5] = float("nan"), float("inf"), 3e38
        for zeros in (False, True):
            for t in (gpu.bfloat16, gpu.float16):
                codes, scales, z = llk.q4_quantise(w, group=group, zeros=zeros, scale_dtype=t)
                assert (z is None) == (not zeros)
                x = w.float().cpu().numpy()
                for g in range(-(-K // group)):
                    part = x[g * group:(g + 1) * group]
                    lo, hi = np.minimum(part.min(0), 0), np.maximum(part.max(0), 0)
                    f = np.float32
                    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
                        s = hi / f(15) - lo / f(15) if zeros else np.maximum(hi, -lo) / f(7)
                        s[~np.isfinite(part).all(0)] = np.nan
                        s = gpu.from_numpy(s).to(t).float().numpy()
                        some = (s > 0) & np.isfinite(s)
                        zero = np.full(N, 8, f) if not zeros else \
                            np.where(some, np.minimum(np.rint(-lo / s), 15), 0).astype(f)
                        c = np.where(some, np.clip(np.rint(part / s) + zero, 0, 15), zero)
                    assert np.array_equal(scales[g].float().cpu().numpy(), s, equal_nan=True)
                    assert np.array_equal(codes[g * group:(g + 1) * group].cpu().numpy(), c)
                    if zeros:
                        assert np.array_equal(z[g].cpu().numpy(), zero)


def test_quantised_weights(llk, gpu):
    """Weights through quantise() and back: each within half a step."""
    K, N, group = 256, 96, 64
    w = gpu.randn(K, N, device="cuda").bfloat16()
    eye = gpu.eye(K, device="cuda").bfloat16()
    for zeros in (False, True):
        codes, scales, z = llk.q4_quantise(w, group=group, zeros=zeros)
        got = f64(llk.q4_matmul(eye, llk.Q4Weights.quantise(w, group=group, zeros=zeros)))
        assert np.array_equal(got, dense(codes, scales, z, group))
        # half a step, the zero's rounding by half a step more at the ends (held to
        # 0..15), and the scale's by 2^-8 of at most 15 steps
        step = f64(scales)[np.arange(K) // group]
        assert (np.abs(got - f64(w)) <= step * (0.5 + 0.5 * zeros + 15 * 2.0 ** -8)).all()


def test_streams_and_graph(llk, gpu):
    """A captured product replays with new X; another stream gives the same."""
    for M in (1, 12, 70):
        x, codes, scales, z = case(gpu, M, 1000, 144, 128, True, gpu.float16, 5, False)
        w = llk.Q4Weights.from_codes(codes, scales, z, group=128)
        want = llk.q4_matmul(x, w)
        side = gpu.cuda.Stream()
        side.wait_stream(gpu.cuda.current_stream())
        with gpu.cuda.stream(side):
            assert gpu.equal(llk.q4_matmul(x, w), want)
        got = gpu.empty_like(want)
        gpu.cuda.synchronize()
        llk.q4_matmul(x, w, out=got, stream=side)
        side.synchronize()
        assert gpu.equal(got, want)
        graph = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(graph, stream=side):
            out = llk.q4_matmul(x, w)
            both = llk.q4_swiglu(x, w, w)
        for seed in range(3):
            x.copy_(gpu.randn(*x.shape, device="cuda"))
            graph.replay()
            assert gpu.equal(out, llk.q4_matmul(x, w)) and gpu.equal(both, llk.q4_swiglu(x, w, w))


@pytest.mark.parametrize("M,K,N", [(17, 1, 16), (20, 5, 33), (100, 7, 16), (1000, 3, 40), (17, 8, 16),
                                   (129, 9, 300)])
def test_many_rows_of_few_values(llk, gpu, M, K, N):
    for group in (32, 128):
        x, codes, scales, z = case(gpu, M, K, N, group, True, gpu.bfloat16, M + K, True)
        w = llk.Q4Weights.from_codes(codes, scales, z, group=group)
        want = f64(x) @ dense(codes, scales, z, group)
        assert np.array_equal(f64(llk.q4_matmul(x, w)), want)
        both = llk.q4_swiglu(x, w, w, out_dtype=gpu.float32)
        # exact sums: only the activation's 4 ulp, of its exponent's argument two
        # roundings of |sum| 2^-24, and its product
        with np.errstate(over="ignore"):
            silu = want / (1 + np.exp(-want))
        near = (np.abs(want) + 8) * 2.0 ** -23 * np.abs(silu * want) + 1e-30
        assert (np.abs(f64(both) - silu * want) <= near).all()


@pytest.mark.parametrize("M", [1, 12, 30, 200])
def test_sums_added_to_half_precision(llk, gpu, M):
    """One rounding of what is there plus the product (exact cases, so equal)."""
    K, N, group = 500, 48, 32
    x, codes, scales, z = case(gpu, M, K, N, group, False, gpu.bfloat16, M, True)
    w = llk.Q4Weights.from_codes(codes, scales, z, group=group)
    want = f64(x) @ dense(codes, scales, z, group)
    for t in (gpu.float16, gpu.bfloat16):
        acc = gpu.randint(-64, 64, (M, N), device="cuda").to(t)
        total = gpu.from_numpy(want + f64(acc)).float().cuda().to(t)
        assert gpu.equal(llk.q4_matmul(x, w, out=acc, accumulate=True), total)


@pytest.mark.parametrize("M,K,N,sides", [(5, 13824, 256, 1), (40, 4096, 512, 2), (300, 5000, 80, 1)])
def test_a_workspace_of_the_callers(llk, gpu, M, K, N, sides):
    """Split products in memory of the caller's, exactly as large as is asked for,
    with its neighbours untouched; one that is too small is refused."""
    x, codes, scales, z = case(gpu, M, K, N, 128, True, gpu.bfloat16, 1, False)
    w = llk.Q4Weights.from_codes(codes, scales, z, group=128)

    def call(**kw):
        return llk.q4_matmul(x, w, **kw) if sides == 1 else llk.q4_swiglu(x, w, w, **kw)

    need = llk.q4_scratch_size(M, N, K, sides)
    assert need > 0
    memory = gpu.full((need + 512,), 7, dtype=gpu.uint8, device="cuda")
    assert gpu.equal(call(scratch=memory[256:256 + need]), call())
    assert (memory[:256] == 7).all() and (memory[256 + need:] == 7).all()
    with pytest.raises(llk.LLKError):
        call(scratch=memory[256:need])


def test_rows_far_apart(llk, gpu):
    """Offsets of X and Y beyond 2^32 bytes."""
    K, N = 64, 32
    for M in (16, 40):
        step = (1 << 31) // (M - 4)
        x, codes, scales, z = case(gpu, M, K, N, 64, True, gpu.bfloat16, M, True)
        w = llk.Q4Weights.from_codes(codes, scales, z, group=64)
        far = gpu.empty(M * step, dtype=gpu.bfloat16, device="cuda").as_strided((M, K), (step, 1))
        far.copy_(x)
        out = gpu.empty(M * step, dtype=gpu.float32, device="cuda").as_strided((M, N), (step, 1))
        llk.q4_matmul(far, w, out=out)
        assert np.array_equal(f64(out), f64(x) @ dense(codes, scales, z, 64))


@pytest.mark.parametrize("M,K,N,sides", [(15, 5000, 13824, 1), (14, 5120, 12800, 2)])
def test_a_first_call_under_capture(llk, gpu, M, K, N, sides):
    """A launch with more than 64 KiB of LDS that nothing made before the capture."""
    x, codes, scales, z = case(gpu, M, K, N, 64, True, gpu.float16, 8, False)
    w = llk.Q4Weights.from_codes(codes, scales, z, group=64)
    scratch = gpu.empty(max(llk.q4_scratch_size(M, N, K, sides), 256), dtype=gpu.uint8, device="cuda")

    def call():
        return llk.q4_matmul(x, w, scratch=scratch) if sides == 1 else \
            llk.q4_swiglu(x, w, w, scratch=scratch)

    side = gpu.cuda.Stream()
    gpu.cuda.synchronize()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        out = call()
    for _ in range(3):
        x.copy_(gpu.randn(*x.shape, device="cuda"))
        graph.replay()
        gpu.cuda.synchronize()
        assert gpu.equal(out, call())


@pytest.mark.parametrize("zeros", [False, True])
def test_weights_made_on_a_stream_of_the_callers(llk, gpu, monkeypatch, zeros):
    """quantise(), q4_quantise() and from_codes() on a stream that is behind: what
    the current stream allocates and writes meanwhile is no memory of theirs."""
    from dslcompiler_amd import q4
    K, N, group = 1000, 1040, 64
    w = gpu.randn(K, N, device="cuda").bfloat16()
    want = llk.Q4Weights.quantise(w, group=group, zeros=zeros)
    want_parts = [t for t in llk.q4_quantise(w, group=group, zeros=zeros) if t is not None]
    parts = []
    quantise = llk.q4_quantise

    def noted(*args, **kw):
        out = quantise(*args, **kw)
        parts.extend((t.data_ptr(), t.numel() * t.element_size()) for t in out if t is not None)
        return out

    monkeypatch.setattr(q4, "q4_quantise", noted)
    big = [gpu.zeros(1 << 28, dtype=gpu.uint8, device="cuda") for _ in range(2)]
    side = gpu.cuda.Stream()
    gpu.cuda.synchronize()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        for n in range(400):  # about 40 ms of copies
            big[n % 2].copy_(big[1 - n % 2])
    got = llk.Q4Weights.quantise(w, group=group, zeros=zeros, stream=side)
    other = [gpu.full((size,), 0xff, dtype=gpu.uint8, device="cuda") for _, size in parts * 2]
    if not side.query():  # it has not packed yet
        for t in other:
            for at, size in parts:
                assert t.data_ptr() + t.numel() <= at or at + size <= t.data_ptr()
    made = llk.q4_quantise(w, group=group, zeros=zeros, stream=side)
    again = llk.Q4Weights.from_codes(*made, group=group, stream=side)
    gpu.cuda.synchronize()
    assert len(parts) == 2 + zeros
    for a, b in zip([t for t in made if t is not None], want_parts):
        assert gpu.equal(a, b)
    x = gpu.randn(5, K, device="cuda").bfloat16()
    first = llk.q4_matmul(x, want)
    assert gpu.equal(llk.q4_matmul(x, got), first) and gpu.equal(llk.q4_matmul(x, again), first)
    rows = np.arange(K) // group
    codes, scales, z = (None if t is None else f64(t) for t in made)
    dense64 = (codes - (8 if z is None else z[rows])) * scales[rows]
    most = bound(x, made[1], group, K)
    assert (np.abs(f64(first) - f64(x) @ dense64) <= most * (1 + 2.0 ** -24)).all()


def dense_on_device(torch, codes, scales, z, group):
    """W in float64, on the device."""
    rows = torch.arange(codes.shape[0], device="cuda") // group
    zero = 8.0 if z is None else z.double()[rows]
    return (codes.double() - zero) * scales.double()[rows]


# The kernel for few rows by column tiles to a workgroup and splits of K: 1 tile below
# 640 tiles of a product (400 of a SwiGLU), then 2, 4 for a SwiGLU from 800 on; 4 and a
# split K where 16-row blocks of X pass 256 units (640 for a wide SwiGLU).  The sizes
# leave no, one, two or three tiles, whole or not, to the last workgroup.
FEW_ROWS = [(M, 300, N, sides) for M in (1, 5, 9, 16)
            for N, sides in ((10240, 1), (10256, 1), (11000, 1), (6400, 2), (6424, 2), (12800, 2), (12840, 2))]
FEW_ROWS += [(16, 4096, 1040, 1), (9, 5000, 1072, 1), (13, 4096, 2000, 1), (1, 33000, 100, 1),
             (16, 4096, 11008, 2), (9, 5000, 1064, 2), (5, 8000, 1048, 2), (1, 33000, 40, 2),
             (16, 4096, 12840, 2), (9, 5120, 12824, 2), (14, 5120, 12872, 2)]


@pytest.mark.parametrize("M,K,N,sides", FEW_ROWS)
def test_few_rows_of_wide_weights(llk, gpu, M, K, N, sides):
    """Exact sums (the file's docstring; X to 1 for long K, whose sums then stay below
    33000 * 2 < 2^17): products equal, a SwiGLU within its activation's roundings."""
    group = (32, 64, 128)[(M + N) % 3]
    x, *g = case(gpu, M, K, N, group, True, gpu.bfloat16, M + N, True)
    if K > 4104:
        x.clamp_(-1, 1)
    a = x.double() @ dense_on_device(gpu, *g, group)
    wg = llk.Q4Weights.from_codes(*g, group=group)
    if sides == 1:
        assert gpu.equal(llk.q4_matmul(x, wg).double(), a)
        acc = gpu.full((M, N), 0.5, dtype=gpu.float32, device="cuda")
        assert gpu.equal(llk.q4_matmul(x, wg, out=acc, accumulate=True).double(), a + 0.5)
        return
    _, *u = case(gpu, M, K, N, group, False, gpu.float16, M + N + 1, True)
    b = x.double() @ dense_on_device(gpu, *u, group)
    wu = llk.Q4Weights.from_codes(*u, group=group)
    want = a / (1 + gpu.exp(-a)) * b
    # the activation's 4 ulp, of its exponent's argument two roundings of |a| 2^-24, and
    # its product
    near = (a.abs() + 8) * 2.0 ** -23 * want.abs() + 1e-30
    got = llk.q4_swiglu(x, wg, wu, out_dtype=gpu.float32).double()
    assert ((got - want).abs() <= near).all()


@pytest.mark.parametrize("M,K,N", [(14, 5120, 12872), (15, 4096, 12840)])
def test_a_captured_swiglu_against_its_sums(llk, gpu, M, K, N):
    """More than 64 KiB of LDS, captured and replayed, against 64 bits."""
    x, *g = case(gpu, M, K, N, 64, True, gpu.float16, 9, True)
    _, *u = case(gpu, M, K, N, 64, True, gpu.float16, 10, True)
    x.clamp_(-1, 1)
    dense_g, dense_u = (dense_on_device(gpu, *s, 64) for s in (g, u))
    wg, wu = (llk.Q4Weights.from_codes(*s, group=64) for s in (g, u))
    side = gpu.cuda.Stream()
    gpu.cuda.synchronize()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        out = llk.q4_swiglu(x, wg, wu, out_dtype=gpu.float32)
    for n in range(3):
        x.copy_(x.roll(n, 1))
        graph.replay()
        a, b = x.double() @ dense_g, x.double() @ dense_u
        want = a / (1 + gpu.exp(-a)) * b
        near = (a.abs() + 8) * 2.0 ** -23 * want.abs() + 1e-30
        assert ((out.double() - want).abs() <= near).all()
