"""Weights in 4 bits with group scales, on torch tensors.

- :func:`q4_quantise`: bf16 weights to codes, scales and zeros;
- :class:`Q4Weights`: such weights in the kernels' order;
- :func:`q4_matmul` and :func:`q4_swiglu`: products with them, as
  :func:`~dslcompiler_amd.matmul` and :func:`~dslcompiler_amd.fused_swiglu` are
  with bf16 ones.

    W[k, n] = scale[k // group, n] * (code[k, n] - zero[k // group, n])

with codes and zeros 0..15; the last group is as long as K leaves it.
"""
from __future__ import annotations

from . import _lib
from ._lib import LLK_BF16, LLK_FP16, LLK_FP32, check, lib
from .decoder import _begin, _context, _kind, _rows
from .ops import _torch

_BF16 = _BYTES = _SCALES = _SUMS = _OUT = None  # torch dtype -> llk_dtype (0 for bytes)


def _start() -> int:
    """The current device; the tables of types on the first call."""
    global _BF16, _BYTES, _SCALES, _SUMS, _OUT
    if _OUT is None:  # the one that is set last: a second thread finds all of them, or none
        torch = _torch()
        _BF16, _BYTES = {torch.bfloat16: LLK_BF16}, {torch.uint8: 0}
        _SCALES = {torch.bfloat16: LLK_BF16, torch.float16: LLK_FP16}
        _SUMS = {torch.bfloat16: LLK_BF16, torch.float32: LLK_FP32}
        _OUT = {**_SCALES, torch.float32: LLK_FP32}
    return _begin()


def _matrix(t, name: str, dev: int, kinds):
    """(descriptor, kind) of a 2-D operand."""
    kind = _kind(t, name, dev, kinds)
    return _rows(t, name), kind


def _result(x, m: int, n: int, dtype, kinds):
    """An uninitialised [m, n] result beside x, its descriptor and its kind."""
    kind = kinds.get(dtype)
    if kind is None:
        raise ValueError(f"out_dtype {dtype} unsupported; expected one of {tuple(kinds)}")
    out = x.new_empty((m, n), dtype=dtype)
    return out, _lib.Tensor2D(out.data_ptr(), m, n, n, 1), kind


def q4_quantise(w, *, group: int = 128, zeros: bool = False, scale_dtype=None, stream=None):
    """(codes uint8 [K, N], scales [groups, N], zeros uint8 [groups, N] or None)
    of bf16 weights [K, N] on the current device.

    Without zeros a group's scale is its largest magnitude / 7; with them it is
    (largest - smallest of its values and 0) / 15.  The scale is rounded to
    scale_dtype (bf16 or fp16; bf16 if none is given), then each value to the
    nearest code.  A group with an infinity or a NaN gets the scale NaN."""
    dev, torch = _start(), _torch()
    wd, _ = _matrix(w, "w", dev, _BF16)
    if group not in (32, 64, 128):
        raise ValueError(f"group must be 32, 64 or 128, not {group}")
    shape = (-(-wd.dim0 // group), wd.dim1)
    codes = torch.empty((wd.dim0, wd.dim1), dtype=torch.uint8, device=w.device)
    scales = torch.empty(shape, dtype=scale_dtype or torch.bfloat16, device=w.device)
    z = torch.empty(shape, dtype=torch.uint8, device=w.device) if zeros else None
    check(lib().llk_q4_quantise(wd, group, _rows(codes, "codes"), _rows(scales, "scales"),
                                _kind(scales, "scales", dev, _SCALES),
                                None if z is None else _rows(z, "zeros"), _context(dev, stream)))
    return codes, scales, z


class Q4Weights:
    """4-bit weights [K, N] in the kernels' order, on the current device."""

    def __init__(self, K: int, N: int, group: int, device):
        torch = _torch()
        self.K, self.N, self.group = K, N, group
        codes, scales = lib().llk_q4_code_bytes(K, N), lib().llk_q4_scale_bytes(K, N, group)
        if codes == 0 and K * N != 0 or scales == 0 and (K * N != 0 or group not in (32, 64, 128)):
            raise ValueError(f"no 4-bit weights of ({K}, {N}) in groups of {group}")
        self._memory = (torch.empty(max(codes, 16), dtype=torch.uint8, device=device),
                        torch.empty(max(scales, 16), dtype=torch.uint8, device=device))
        self.device_index = self._memory[0].get_device()
        self.c = _lib.Q4WeightsC(self._memory[0].data_ptr(), self._memory[1].data_ptr(), K, N, group)

    @property
    def device_bytes(self) -> int:
        return sum(m.numel() for m in self._memory)

    @classmethod
    def from_codes(cls, codes, scales, zeros=None, *, group: int = 128, stream=None) -> "Q4Weights":
        """Codes uint8 [K, N], scales bf16 or fp16 [ceil(K / group), N] and zeros
        uint8 of the same shape (None: 8 everywhere)."""
        dev = _start()
        cd, _ = _matrix(codes, "codes", dev, _BYTES)
        sd, kind = _matrix(scales, "scales", dev, _SCALES)
        zd = None if zeros is None else _matrix(zeros, "zeros", dev, _BYTES)[0]
        w = cls(cd.dim0, cd.dim1, group, codes.device)
        check(lib().llk_q4_pack(cd, sd, kind, zd, w.c, _context(dev, stream)))
        return w

    @classmethod
    def quantise(cls, w, *, group: int = 128, zeros: bool = False, scale_dtype=None,
                 stream=None) -> "Q4Weights":
        """:func:`q4_quantise` of bf16 weights [K, N], packed."""
        parts = q4_quantise(w, group=group, zeros=zeros, scale_dtype=scale_dtype, stream=stream)
        if stream is not None:
            # dropped as this returns, when the stream may not have packed them yet: until
            # then their memory is not to be given to the current stream's next allocations
            for t in parts:
                if t is not None:
                    t.record_stream(stream)
        return cls.from_codes(*parts, group=group, stream=stream)


def _packed(w, name: str, dev: int) -> _lib.Q4WeightsC:
    if not isinstance(w, Q4Weights):
        raise ValueError(f"{name} must be Q4Weights")
    if w.device_index != dev:
        raise ValueError(f"{name} is on cuda:{w.device_index}, the current device is cuda:{dev}")
    return w.c


def q4_matmul(x, w: Q4Weights, *, out=None, out_dtype=None, accumulate: bool = False, stream=None,
              scratch=None):
    """X W, x bf16 [M, K], to bf16, fp16 or fp32 (the default, as of matmul);
    with accumulate=True, out += X W, out being required.  Sums in fp32, weights
    as they are.  A row of X with an infinity or a NaN gives NaN."""
    dev = _start()
    wc = _packed(w, "w", dev)
    xd, _ = _matrix(x, "x", dev, _BF16)
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs `out`, the accumulator")
        out, od, kind = _result(x, xd.dim0, w.N, out_dtype or _torch().float32, _OUT)
    else:
        od, kind = _matrix(out, "out", dev, _OUT)
    check(lib().llk_q4_gemm(xd, wc, od, kind, accumulate,
                            _context(dev, stream, scratch)))
    return out


def q4_swiglu(x, wg: Q4Weights, wu: Q4Weights, *, out=None, out_dtype=None, stream=None,
              scratch=None):
    """SiLU(X Wg) * (X Wu), x bf16 [M, K], to bf16 (the default) or fp32; weights
    of one shape and group."""
    dev = _start()
    gc, uc = _packed(wg, "wg", dev), _packed(wu, "wu", dev)
    xd, _ = _matrix(x, "x", dev, _BF16)
    if out is None:
        out, od, kind = _result(x, xd.dim0, wg.N, out_dtype or _torch().bfloat16, _SUMS)
    else:
        od, kind = _matrix(out, "out", dev, _SUMS)
    check(lib().llk_q4_swiglu(xd, gc, uc, od, kind, _context(dev, stream, scratch)))
    return out


def q4_scratch_size(M: int, N: int, K: int, sides: int = 1) -> int:
    """Bytes of `scratch` that q4_matmul (sides 1) and q4_swiglu (sides 2) need."""
    return int(lib().llk_q4_scratch_size(M, N, K, sides))
