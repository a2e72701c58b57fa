"""examples/decoder_layer.py: a prompt and decoded tokens through two layers,
against the same layers in float64 on the host with the cache's own values, and
token by token against the prompt at once.

Bound.  The kernels round to bf16 where the framework's types say so: q, k, v,
attention, MLP intermediate and each block's result, the residual sum after each
block and each norm.  That is 10 roundings of at most 2^-8 a layer, most of them
of a block that enters the residual with a weight of 1/2, and a norm that keeps
their relative size: rel-L2 within 2 layers * 10 * 2^-9 (their rms) < 2^-4.6.
A code of the cache may come out otherwise where k or v lies within a rounding
of a tie, so both sides read the kernels' cache."""
from __future__ import annotations

import importlib.util
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]


def example():
    spec = importlib.util.spec_from_file_location("decoder_layer",
                                                  ROOT / "examples" / "decoder_layer.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def make(gpu, monkeypatch, **kw):
    """A model, and its matrices as float64."""
    mod = example()
    plain = []
    pack = mod.llk.PackedWeights.from_device

    def keep(w):
        plain.append(w.double().cpu().numpy())
        return pack(w)

    monkeypatch.setattr(mod.llk.PackedWeights, "from_device", keep)
    model = mod.Model(**kw)
    monkeypatch.undo()
    names = ("qkv", "o", "gate", "up", "down")
    mats = [dict(zip(names, plain[5 * i:5 * i + 5])) for i in range(len(model.layers))]
    return model, mats


def reference(model, mats, x, table, lens, starts):
    """forward() in float64, the attention over the cache as it is."""
    def f64(t):
        return t.double().cpu().numpy()

    def norm(v, w):
        return v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6) * f64(w)

    h = f64(x)
    n = norm(h, model.layers[0].attention_norm)
    for i, (layer, w) in enumerate(zip(model.layers, mats)):
        D, H = layer.head_dim, layer.heads
        q = (n @ w["qkv"])[:, :H * D].reshape(-1, H, D)
        pool = layer.cache.cpu().numpy()
        out, _ = ref.attention(q, pool, table, lens, starts, D ** -0.5, model.window, model.sinks)
        y = out.reshape(len(h), -1) @ w["o"]
        h = h + model.scale * norm(y, layer.attention_post)
        n = norm(h, layer.mlp_norm)
        g = n @ w["gate"]
        y = (g / (1 + np.exp(-g)) * (n @ w["up"])) @ w["down"]
        h = h + model.scale * norm(y, layer.mlp_post)
        last = i + 1 == len(model.layers)
        n = norm(h, model.final_norm if last else model.layers[i + 1].attention_norm)
    return n


def test_prompt_and_tokens(llk, gpu, monkeypatch):
    model, mats = make(gpu, monkeypatch, hidden=256, inner=512, heads=4, kv_heads=2, head_dim=64,
                       pages=16, page_size=16, window=40, sinks=3)
    gen = gpu.Generator(device="cuda").manual_seed(3)
    prompts = [70, 21]
    x = gpu.randn(sum(prompts), 256, generator=gen, device="cuda").bfloat16()
    table = gpu.randperm(16, generator=gen, device="cuda").int().view(2, 8)
    lens = gpu.tensor(prompts, dtype=gpu.int32, device="cuda")
    starts = gpu.tensor([0, 70, 91], dtype=gpu.int32, device="cuda")
    out = model.forward(x, table, lens, starts)
    t, n, s = (v.cpu().numpy() for v in (table, lens, starts))

    def rel(got, want):
        got = got.double().cpu().numpy()
        return np.linalg.norm(got - want) / np.linalg.norm(want)

    bound = 2 * 10 * 2.0 ** -9
    assert rel(out, reference(model, mats, x, t, n, s)) <= bound
    token = gpu.randn(2, 256, generator=gen, device="cuda").bfloat16()
    for _ in range(3):
        lens += 1
        got = model.forward(token, table, lens)
        assert rel(got, reference(model, mats, token, t, lens.cpu().numpy(), None)) <= bound
        token = got


def test_runs_as_a_program():
    for more in ([], ["--graph"]):
        r = subprocess.run([sys.executable, str(ROOT / "examples" / "decoder_layer.py"),
                            "--prompt", "60", "--tokens", "3", *more],
                           capture_output=True, text=True, timeout=100)
        assert r.returncode == 0, r.stdout + r.stderr
        assert "lengths [63, 23]" in r.stdout
        assert "nan" not in r.stdout


def test_program_gives_the_same_with_a_graph():
    """Lengths and the last token after the same steps, eager and replayed
    (the step before the capture changes both, from which they are restored)."""
    said = []
    for more in ([], ["--graph"]):
        r = subprocess.run([sys.executable, str(ROOT / "examples" / "decoder_layer.py"),
                            "--prompt", "300", "--tokens", "5", *more],
                           capture_output=True, text=True, timeout=100)
        assert r.returncode == 0, r.stdout + r.stderr
        said.append(r.stdout.split("us a step")[0].rsplit(",", 1)[0])
    assert said[0] == said[1] and "lengths [305, 105]" in said[0]


def test_captured_steps(llk, gpu, monkeypatch):
    """A decoded token's step captured once: each replay, with new lengths and
    tokens, equals the eager step bit by bit and the layers in 64 bits."""
    model, mats = make(gpu, monkeypatch, hidden=256, inner=512, heads=4, kv_heads=2, head_dim=64,
                       pages=16, page_size=16, window=40, sinks=3)
    gen = gpu.Generator(device="cuda").manual_seed(4)
    table = gpu.randperm(16, generator=gen, device="cuda").int().view(2, 8)
    lens = gpu.tensor([45, 60], dtype=gpu.int32, device="cuda")
    starts = gpu.tensor([0, 45, 105], dtype=gpu.int32, device="cuda")
    x = gpu.randn(105, 256, generator=gen, device="cuda").bfloat16()
    model.forward(x, table, lens, starts)
    token = gpu.randn(2, 256, generator=gen, device="cuda").bfloat16()
    lens += 1
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        model.forward(token, table, lens)
    gpu.cuda.synchronize()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        out = model.forward(token, table, lens)
    bound = 2 * 10 * 2.0 ** -9
    for n in range(4):
        graph.replay()
        got = out.clone()
        want = reference(model, mats, token, table.cpu().numpy(), lens.cpu().numpy(), None)
        assert np.linalg.norm(got.double().cpu().numpy() - want) <= bound * np.linalg.norm(want), n
        assert gpu.equal(model.forward(token, table, lens), got), n
        token.copy_(got)
        lens += 1


def test_token_by_token_against_the_prompt_at_once(llk, gpu, monkeypatch):
    """The same 75 tokens through pages of their own.

    Bound.  Each pass is within b = 20 * 2^-9 of the layers over its own cache, and
    the caches differ where a code comes out otherwise.  Layer 1 quantises the same
    keys and values but for rare roundings.  Those of layer 2 differ by at most b / 2
    of their size; a code's step is at most 0.63 of a block's rms (the scale is at
    most 2 / 7 of the largest of 32, about 2.2 rms, and steps are 1 or less below 4),
    so the quantised ones by sqrt(0.63 * b / 2) = 0.11 of it, and attention by as much
    through the values and as much through the scores: 0.16.  With the layer's weight
    of 1/2 in the residual, twice (attention, and the MLP behind it): 0.16 * 0.5 *
    sqrt(2) = 0.11.  In all 2 b + 0.11 < 0.19."""
    model, _ = make(gpu, monkeypatch, hidden=256, inner=512, heads=4, kv_heads=2, head_dim=64,
                    pages=16, page_size=16, window=40, sinks=3)
    gen = gpu.Generator(device="cuda").manual_seed(6)
    n = 75
    x = gpu.randn(n, 256, generator=gen, device="cuda").bfloat16()
    table = gpu.randperm(16, generator=gen, device="cuda").int().view(2, 8)
    starts = gpu.tensor([0, n], dtype=gpu.int32, device="cuda")
    lens = gpu.tensor([n], dtype=gpu.int32, device="cuda")
    whole = model.forward(x, table[:1], lens, starts).double()
    for i in range(n):
        lens.fill_(i + 1)
        got = model.forward(x[i:i + 1], table[1:], lens).double()
        assert (got - whole[i]).norm() <= 0.19 * whole[i].norm(), i
