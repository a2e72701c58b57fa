"""Library workspaces made while the default stream is busy: nothing of the default
stream's (a fill of the fresh memory, for one, which HIP would queue there) reaches into the
calls of the stream that the workspace belongs to."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def behind(llk, gpu, calls, rounds):
    """`rounds` calls on a stream of their own, the first of which makes its
    workspace, while the default stream has about 30 ms of copies queued."""
    big = [gpu.zeros(1 << 28, dtype=gpu.uint8, device="cuda") for _ in range(2)]
    side = gpu.cuda.Stream()
    gpu.cuda.synchronize()
    llk.workspace_trim()
    for n in range(300):
        big[n % 2].copy_(big[1 - n % 2])
    with gpu.cuda.stream(side):
        for n in range(rounds):
            calls(n)
    gpu.cuda.synchronize()
    llk.workspace_trim()


def test_split_products(llk, gpu):
    K, N, M, rounds = 13824, 5120, 5, 2000
    codes = gpu.randint(0, 16, (K, N), device="cuda").to(gpu.uint8)
    scales = (gpu.rand(K // 128, N, device="cuda") * 0.01).bfloat16()
    w = llk.Q4Weights.from_codes(codes, scales, group=128)
    assert llk.q4_scratch_size(M, N, K) > 0
    x = gpu.randn(M, K, device="cuda").bfloat16()
    want = llk.q4_matmul(x, w)
    out = gpu.zeros(rounds, M, N, device="cuda")
    behind(llk, gpu, lambda n: llk.q4_matmul(x, w, out=out[n]), rounds)
    assert (out == want).all()


def test_split_swiglu(llk, gpu):
    M, K, N, rounds = 8, 4096, 14336, 1000
    x = gpu.randn(M, K, device="cuda").bfloat16()
    wg, wu = (llk.PackedWeights.from_device((gpu.randn(K, N, device="cuda") * K ** -0.5).bfloat16())
              for _ in range(2))
    want = llk.fused_swiglu(x, wg, wu)
    out = gpu.zeros(rounds, M, N, dtype=want.dtype, device="cuda")
    behind(llk, gpu, lambda n: llk.fused_swiglu(x, wg, wu, out=out[n]), rounds)
    assert (out == want).all()


def test_kept_scores(llk, gpu):
    """64 sequences of a table of 65536 keys each: 512 MiB of scores."""
    D, size, sequences, heads, group, rounds = 64, 64, 64, 8, 4, 1000
    table = gpu.arange(sequences * 1024, device="cuda").int().view(sequences, 1024) % (sequences * 8)
    table[:, :8] = gpu.randperm(sequences * 8, device="cuda").int().view(sequences, 8)
    lens = gpu.randint(100, 8 * size + 1, (sequences,), device="cuda").int()
    cache = llk.kv4_cache(sequences * 8, heads, size, D)
    starts = gpu.cat([gpu.zeros(1, device="cuda"), lens.cumsum(0)]).int()
    kv = gpu.randn(int(lens.sum()), heads, D, device="cuda").bfloat16()
    llk.kv4_write(kv, kv.roll(1, 0), cache, table, lens, starts=starts)
    q = gpu.randn(sequences, heads * group, D, device="cuda").bfloat16()
    plan = llk.describe_kv4_attention(q, cache, table, lens, weigh=True)
    assert plan["workspace_bytes"] >= 512 << 20
    marks = gpu.zeros(sequences * 8, heads, size, device="cuda")
    first = llk.kv4_attention(q, cache, table, lens, weights=marks)
    want = marks.clone()
    out = gpu.zeros(rounds, *q.shape, dtype=gpu.bfloat16, device="cuda")
    same = gpu.zeros(rounds, dtype=gpu.bool, device="cuda")

    def call(n):
        llk.kv4_attention(q, cache, table, lens, weights=marks, decay=0.0, out=out[n])
        same[n] = (marks == want).all()

    behind(llk, gpu, call, rounds)
    assert (out.view(gpu.int16) == first.view(gpu.int16)).all() and same.all()
