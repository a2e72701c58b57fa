"""What the 4-bit weights refuse, before any device work, and their sizes."""
from __future__ import annotations

import pytest

FAKE = 1 << 20  # an aligned address


@pytest.fixture()
def L(llk):
    return llk.lib()


def _t(rows, cols, stride=None, data=FAKE, one=1):
    from dslcompiler_amd._lib import Tensor2D
    return Tensor2D(data, rows, cols, cols if stride is None else stride, one)


def _w(K=256, N=64, group=64, codes=FAKE, scales=FAKE):
    from dslcompiler_amd._lib import Q4WeightsC
    return Q4WeightsC(codes, scales, K, N, group)


def test_sizes(L):
    assert L.llk_q4_code_bytes(128, 16) == 1024
    assert L.llk_q4_code_bytes(129, 17) == 4 * 1024
    assert L.llk_q4_code_bytes(4096, 14336) == 4096 * 14336 // 2
    assert L.llk_q4_scale_bytes(128, 16, 32) == 4 * 64
    assert L.llk_q4_scale_bytes(129, 1, 128) == 2 * 64
    assert L.llk_q4_code_bytes(0, 16) == 0 and L.llk_q4_code_bytes(-1, 16) == 0
    for group in (0, 16, 48, 256, -32):
        assert L.llk_q4_scale_bytes(128, 16, group) == 0, group


BAD_WEIGHTS = [(dict(group=48), -2), (dict(group=0), -2), (dict(K=-1), -2), (dict(N=1 << 40), -2),
               (dict(K=1 << 40), -2), (dict(codes=None), -1), (dict(scales=None), -1),
               (dict(codes=FAKE + 8), -4), (dict(scales=FAKE + 4), -4)]


def test_product_refusals(L):
    x, y = _t(4, 256), _t(4, 64)
    for bad, code in BAD_WEIGHTS:
        assert L.llk_q4_gemm(x, _w(**bad), y, 0, 0, None) == code, bad
        assert L.llk_q4_swiglu(x, _w(**bad), _w(), y, 0, None) == code, bad
        assert L.llk_q4_swiglu(x, _w(), _w(**bad), y, 0, None) == code, bad
        assert L.llk_last_error()
    assert L.llk_q4_gemm(x, None, y, 0, 0, None) == -1
    assert L.llk_q4_gemm(None, _w(), y, 0, 0, None) == -1
    assert L.llk_q4_gemm(x, _w(), None, 0, 0, None) == -1
    assert L.llk_q4_swiglu(x, _w(), None, y, 0, None) == -1
    for bad, code in [(_t(4, 255), -2), (_t(-1, 256), -2), (_t(1 << 25, 256), -2),
                      (_t(4, 256, stride=255), -4), (_t(4, 256, one=2), -4),
                      (_t(4, 256, data=FAKE + 1), -4), (_t(4, 256, data=None), -1)]:
        rows = bad.dim0
        assert L.llk_q4_gemm(bad, _w(), _t(rows, 64), 0, 0, None) == code, (bad.dim0, bad.dim1)
    for bad, code in [(_t(4, 63), -2), (_t(3, 64), -2), (_t(4, 64, stride=63), -4),
                      (_t(4, 64, one=3), -4), (_t(4, 64, data=None), -1)]:
        assert L.llk_q4_gemm(x, _w(), bad, 0, 0, None) == code
    assert L.llk_q4_gemm(x, _w(), _t(4, 64, data=FAKE + 2), 2, 0, None) == -4
    assert L.llk_q4_gemm(x, _w(), y, 5, 0, None) == -3
    assert L.llk_q4_swiglu(x, _w(), _w(), y, 1, None) == -3  # no fp16 result, as llk_swiglu_bf16
    assert L.llk_q4_swiglu(x, _w(), _w(N=32), y, 0, None) == -2
    assert L.llk_q4_swiglu(x, _w(), _w(group=128), y, 0, None) == -2
    big = 1 << 24  # more workgroups than a launch takes
    assert L.llk_q4_gemm(_t(big, 256), _w(N=1 << 16), _t(big, 1 << 16), 0, 0, None) == -2
    assert b"too many" in L.llk_last_error()
    assert L.llk_q4_scratch_size(1, 4096, 4096, 1) == 0
    assert L.llk_q4_scratch_size(16, 4096, 13824, 1) % (16 * 4096 * 4) == 0
    assert L.llk_q4_scratch_size(17, 4096, 4096, 1) % (17 * 4096 * 4) == 0
    assert L.llk_q4_scratch_size(17, 16, 0, 2) == 0
    assert L.llk_q4_scratch_size(-1, 4096, 4096, 1) == 0 and L.llk_q4_scratch_size(17, 16, 16, 3) == 0
    # nothing to do
    assert L.llk_q4_gemm(_t(0, 256), _w(), _t(0, 64), 0, 0, None) == 0
    assert L.llk_q4_gemm(x, _w(N=0), _t(4, 0), 0, 0, None) == 0


@pytest.mark.parametrize("sides", [1, 2])
@pytest.mark.parametrize("M,N,K", [(16, 0, 4096), (1, 0, 65535 * 32), (3, 0, 65535 * 32), (17, 0, 4096),
                                   (0, 4096, 4096), (0, 0, 4096), (16, 0, 0), (0, 0, 0)])
def test_workspace_of_an_empty_product(L, M, N, K, sides):
    """Also where X alone would not fit a workgroup, so that K would be split by
    the number of columns."""
    assert L.llk_q4_scratch_size(M, N, K, sides) == 0


def test_pack_and_quantise_refusals(L):
    codes, scales = _t(256, 64), _t(4, 64)
    for bad, code in BAD_WEIGHTS:
        K, N = bad.get("K", 256), bad.get("N", 64)
        assert L.llk_q4_pack(_t(K, N), _t(4, N), 0, None, _w(**bad), None) == code, bad
    assert L.llk_q4_pack(codes, scales, 0, None, None, None) == -1
    assert L.llk_q4_pack(None, scales, 0, None, _w(), None) == -1
    assert L.llk_q4_pack(codes, None, 0, None, _w(), None) == -1
    assert L.llk_q4_pack(codes, scales, 2, None, _w(), None) == -3
    assert L.llk_q4_pack(codes, _t(5, 64), 0, None, _w(), None) == -2
    assert L.llk_q4_pack(codes, _t(4, 64, data=FAKE + 1), 0, None, _w(), None) == -4
    assert L.llk_q4_pack(codes, scales, 0, _t(4, 63), _w(), None) == -2
    assert L.llk_q4_pack(_t(256, 64, stride=10), scales, 0, None, _w(), None) == -4
    w = _t(256, 64)
    assert L.llk_q4_quantise(w, 64, codes, scales, 0, None, None) != 0  # no device here
    assert L.llk_q4_quantise(None, 64, codes, scales, 0, None, None) == -1
    assert L.llk_q4_quantise(w, 63, codes, scales, 0, None, None) == -2
    assert L.llk_q4_quantise(w, 64, codes, scales, 2, None, None) == -3
    assert L.llk_q4_quantise(w, 64, _t(255, 64), scales, 0, None, None) == -2
    assert L.llk_q4_quantise(w, 64, codes, _t(3, 64), 0, None, None) == -2
    assert L.llk_q4_quantise(w, 64, codes, scales, 0, _t(4, 1), None) == -2
    assert L.llk_q4_quantise(_t(256, 64, data=None), 64, codes, scales, 0, None, None) == -1
    assert L.llk_q4_quantise(_t(0, 64), 64, _t(0, 64), _t(0, 64), 0, None, None) == 0


def test_python_refusals(llk):
    import torch
    w = torch.zeros(128, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        llk.q4_quantise(w)
    with pytest.raises(ValueError, match="CUDA"):
        llk.Q4Weights.from_codes(w.to(torch.uint8), w[:1])
    with pytest.raises(ValueError, match="Q4Weights"):
        llk.q4_matmul(w.T, w)
    with pytest.raises(ValueError, match="Q4Weights"):
        llk.q4_swiglu(w.T, w, w)


@pytest.mark.parametrize("zeros", [False, True])
def test_quantise_keeps_its_temporaries_for_the_stream(llk, monkeypatch, zeros):
    """The codes, scales and zeros that quantise() makes and drops are the stream's
    until it has packed them: the allocator is told of it before it gets them back."""
    from dslcompiler_amd import q4

    class Part:
        streams = ()

        def record_stream(self, stream):
            self.streams += (stream,)

    parts = (Part(), Part(), Part() if zeros else None)
    monkeypatch.setattr(q4, "q4_quantise", lambda w, **kw: parts)
    monkeypatch.setattr(q4.Q4Weights, "from_codes",
                        classmethod(lambda cls, *p, **kw: [t.streams for t in p if t is not None]))
    stream = object()
    seen = llk.Q4Weights.quantise(None, zeros=zeros, stream=stream)
    assert seen == [(stream,)] * (2 + zeros)
    for t in parts:
        if t is not None:
            t.streams = ()
    # they are of the current stream's memory, which takes them in its order
    assert llk.Q4Weights.quantise(None, zeros=zeros) == [()] * (2 + zeros)
