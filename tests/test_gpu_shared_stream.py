"""Threads that call on one stream: the launches of a call whose second kernel
joins the partial results of the first stay together, so no call reads another's
partial results from the workspace they share."""
from __future__ import annotations

import threading

import numpy as np
import pytest

from test_gpu_kv4 import Case, _dev

pytestmark = pytest.mark.gpu


def together(torch, call, n, times):
    """call(i) `times` times in each of n threads at once on the current stream; their results."""
    stream = torch.cuda.current_stream()
    got, failed, start = [[] for _ in range(n)], [], threading.Barrier(n)

    def work(i):
        try:
            with torch.cuda.stream(stream):
                start.wait(30)
                for _ in range(times):
                    got[i].append(call(i))
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
        assert not t.is_alive()
    torch.cuda.synchronize()
    assert not failed, failed
    return got


def test_attention(llk, gpu):
    c = Case(gpu, [3000, 1200], [1, 1], 2, 128, 64, seed=3)
    pool, table, lens, _ = c.dev()
    q = [_dev(gpu, c.queries(8), gpu.bfloat16) for _ in range(4)]
    # the last thread's calls have other lengths, so other splits
    most = [0, 0, 0, 1500]
    assert llk.describe_kv4_attention(q[0], pool, table, lens)["launches"] == 2

    def call(i):
        return llk.kv4_attention(q[i], pool, table, lens, max_len=most[i])

    want = [call(i).clone() for i in range(4)]
    for i, outs in enumerate(together(gpu, call, 4, 200)):
        assert len(outs) == 200 and all(gpu.equal(o, want[i]) for o in outs), i


def test_swiglu(llk, gpu):
    M, K, N = 8, 4096, 2000
    gen = gpu.Generator(device="cuda").manual_seed(5)

    def rnd(*shape):
        return gpu.randn(*shape, generator=gen, device="cuda").bfloat16()

    x = [rnd(M, K) for _ in range(3)]
    wg, wu = (llk.PackedWeights.from_device(rnd(K, N) * K ** -0.5) for _ in range(2))
    old = llk.get_tunable("decode_splits")
    llk.set_tunable("decode_splits", 3)
    try:
        assert llk.describe_launch("fused_swiglu", M, N, K)["workspace_bytes"] > 0

        def call(i):
            return llk.fused_swiglu(x[i], wg, wu)

        want = [call(i).clone() for i in range(3)]
        assert np.isfinite(want[0].float().cpu().numpy()).all()
        for i, outs in enumerate(together(gpu, call, 3, 200)):
            assert len(outs) == 200 and all(gpu.equal(o, want[i]) for o in outs), i
    finally:
        llk.set_tunable("decode_splits", old)
