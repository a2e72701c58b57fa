"""examples/decoder_layer.py on 4-bit weights, with rotary positions and a bounded
cache: a prompt and decoded tokens, eager and captured, against the same layers in
float64 over the cache and marks that each step left.

Bound of the outputs: as for the layers on bf16 weights (test_gpu_decoder_layer), two
roundings to bf16 more a layer, of q and of k: within 2 layers * 12 * 2^-9.  The
weights in 4 bits are not rounded further, so the reference has their exact values."""
from __future__ import annotations

import subprocess
import sys

import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_decoder_layer import ROOT, example
from test_gpu_kv4_evict import moved, plan

pytestmark = pytest.mark.gpu

BOUND = 2 * 12 * 2.0 ** -9


def make(llk, gpu, monkeypatch, **kw):
    """A model, and its matrices as float64."""
    mod = example()
    plain = []
    quantise = llk.Q4Weights.quantise

    def keep(w, *, group):
        codes, scales, _ = llk.q4_quantise(w, group=group)
        rows = np.arange(w.shape[0]) // group
        plain.append((codes.double().cpu().numpy() - 8) * scales.double().cpu().numpy()[rows])
        return quantise(w, group=group)

    monkeypatch.setattr(mod.llk.Q4Weights, "quantise", keep)
    model = mod.Model(bits=4, rotary=True, **kw)
    monkeypatch.undo()
    names = ("qkv", "o", "gate", "up", "down")
    return model, [dict(zip(names, plain[5 * i:5 * i + 5])) for i in range(len(model.layers))]


def f64(t):
    return t.double().cpu().numpy()


def reference(model, mats, x, table, lens, starts, at, pools):
    """forward() in float64 over the layers' caches as they were before evictions."""
    def norm(v, w):
        return v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6) * f64(w)

    h = f64(x)
    n = norm(h, model.layers[0].attention_norm)
    for i, (layer, w) in enumerate(zip(model.layers, mats)):
        D, H = layer.head_dim, layer.heads
        q = (n @ w["qkv"])[:, :H * D].reshape(-1, H, D)
        angle = (f64(at)[:, None] * np.array(model.turn.frequencies))[:, None]
        a, b = q[..., :D // 2], q[..., D // 2:]
        q = np.concatenate([a * np.cos(angle) - b * np.sin(angle),
                            b * np.cos(angle) + a * np.sin(angle)], -1)
        window = (0, 0) if model.keep else (model.window, model.sinks)
        out, _ = ref.attention(q, pools[i], table, lens, starts, D ** -0.5, *window)
        h = h + model.scale * norm(out.reshape(len(h), -1) @ w["o"], layer.attention_post)
        n = norm(h, layer.mlp_norm)
        g = n @ w["gate"]
        h = h + model.scale * norm((g / (1 + np.exp(-g)) * (n @ w["up"])) @ w["down"], layer.mlp_post)
        last = i + 1 == len(model.layers)
        n = norm(h, model.final_norm if last else model.layers[i + 1].attention_norm)
    return n


def rel(got, want):
    return np.linalg.norm(f64(got) - want) / np.linalg.norm(want)


SMALL = dict(hidden=256, inner=512, heads=4, kv_heads=2, head_dim=64, pages=16, page_size=16,
             window=40, sinks=3)


def start(gpu, seed):
    gen = gpu.Generator(device="cuda").manual_seed(seed)
    x = gpu.randn(91, 256, generator=gen, device="cuda").bfloat16()
    table = gpu.randperm(16, generator=gen, device="cuda").int().view(2, 8)
    lens = gpu.tensor([70, 21], dtype=gpu.int32, device="cuda")
    starts = gpu.tensor([0, 70, 91], dtype=gpu.int32, device="cuda")
    at = gpu.cat([gpu.arange(70), gpu.arange(21)]).int().cuda()
    token = gpu.randn(2, 256, generator=gen, device="cuda").bfloat16()
    return x, table, lens, starts, at, token


def test_rotary_on_4_bit_weights(llk, gpu, monkeypatch):
    model, mats = make(llk, gpu, monkeypatch, **SMALL)
    x, table, lens, starts, at, token = start(gpu, 3)

    def pools():
        return [n.cache.cpu().numpy() for n in model.layers]

    out = model.forward(x, table, lens, starts, at=at)
    t = table.cpu().numpy()
    assert rel(out, reference(model, mats, x, t, lens.cpu().numpy(), starts.cpu().numpy(), at,
                              pools())) <= BOUND
    at = lens.clone()
    for _ in range(3):
        lens += 1
        got = model.forward(token, table, lens, at=at)
        assert rel(got, reference(model, mats, token, t, lens.cpu().numpy(), None, at, pools())) <= BOUND
        token = got
        at += 1


def test_bounded_cache(llk, gpu, monkeypatch):
    """Before each eviction: the outputs, and that the weights of a head's slots add
    up to what its rows gave.  After it: the cache and marks that sorting gives."""
    keep = 40
    model, mats = make(llk, gpu, monkeypatch, keep=keep, **SMALL)
    x, table, lens, starts, at, token = start(gpu, 4)
    before = []
    evict = type(model.layers[0]).evict

    def watched(layer, table, lens, *args):
        before.append([f.cpu().numpy() for f in (layer.cache, *layer.marks, lens)])
        evict(layer, table, lens, *args)

    monkeypatch.setattr(type(model.layers[0]), "evict", watched)
    t = table.cpu().numpy()
    held = np.zeros((2, 2, 2))  # weight left by a step, of layer, sequence, head
    for step in range(5):
        before.clear()
        new = np.array([70, 21]) if step == 0 else np.array([1, 1])
        asked, begin = (x, starts) if step == 0 else (token, None)
        out = model.forward(asked, table, lens, begin, max_len=100, at=at)
        n = before[0][3]
        want = reference(model, mats, asked, t, n, None if begin is None else begin.cpu().numpy(), at,
                         [b[0] for b in before])
        assert rel(out, want) <= BOUND
        for i, (layer, (pool, weights, positions, _)) in enumerate(zip(model.layers, before)):
            for s in range(2):
                j = np.arange(n[s])
                w = weights[t[s, j // 16], :, j % 16].astype(np.float64).sum(0)
                # fp32 sums of weights that are within 2^-18 and their scores' errors
                # ((64 + 16) 2^-22 of S, which stays below 40 here)
                assert np.allclose(w, held[i, s] + 2 * new[s], rtol=2.0 ** -9, atol=0), (step, i, s)
            cut, source = plan(weights, positions, t, n, keep, keep // 4, 3)
            want_pool, marks = moved(pool, t, source, keep, 16, 64, [weights, positions])
            assert np.array_equal(layer.cache.cpu().numpy(), want_pool)
            for got, m in zip(layer.marks, marks):
                assert np.array_equal(got.cpu().numpy(), m)
            assert np.array_equal(lens.cpu().numpy(), cut)
            for s in range(2):
                j = np.arange(cut[s])
                held[i, s] = marks[0][t[s, j // 16], :, j % 16].astype(np.float64).sum(0)
                p = marks[1][t[s, j // 16], :, j % 16]  # [slot, head]
                newest = (69 if s == 0 else 20) + step
                for h in range(2):
                    assert len(set(p[:, h])) == cut[s] and p[:, h].max() == newest
                    kept = set(p[:, h])
                    assert kept >= set(range(newest - min(keep // 4, newest) + 1, newest + 1))
                    assert kept >= {0, 1, 2}
        at = gpu.tensor([70, 21], dtype=gpu.int32, device="cuda") + step
        lens += 1
        token = out[-2:].contiguous() if step == 0 else out


def test_captured_steps_of_a_bounded_cache(llk, gpu, monkeypatch):
    """The step captured once: replays give the eager steps' outputs, caches and marks."""
    model, _ = make(llk, gpu, monkeypatch, keep=40, **SMALL)
    x, table, lens, starts, at, token = start(gpu, 5)
    model.forward(x, table, lens, starts, max_len=100, at=at)
    at = gpu.tensor([70, 21], dtype=gpu.int32, device="cuda")

    def step():
        lens.add_(1)
        token.copy_(model.forward(token, table, lens, max_len=100, at=at))
        at.add_(1)

    state = [token, lens, at] + [t for n in model.layers for t in (n.cache, *n.marks)]
    first = [t.clone() for t in state]
    eager = []
    for _ in range(4):
        step()
        eager.append([t.clone() for t in state])
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        step()
    gpu.cuda.synchronize()
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph, stream=side):
        step()
    for t, was in zip(state, first):
        t.copy_(was)
    for want in eager:
        graph.replay()
        for got, w in zip(state, want):
            assert gpu.equal(got, w)


def test_runs_as_a_program():
    for more in (["--bits", "4"], ["--rotary", "--keep", "32"],
                 ["--bits", "4", "--rotary", "--keep", "32", "--graph"]):
        r = subprocess.run([sys.executable, str(ROOT / "examples" / "decoder_layer.py"),
                            "--prompt", "60", "--tokens", "3", *more],
                           capture_output=True, text=True, timeout=100)
        assert r.returncode == 0, r.stdout + r.stderr
        assert ("lengths [32, 23]" if "--keep" in more else "lengths [63, 23]") in r.stdout
        assert "nan" not in r.stdout
