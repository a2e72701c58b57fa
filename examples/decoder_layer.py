"""A decoder layer on the gfx950 kernels: norms, projections, a 4-bit paged
cache, attention and the SwiGLU MLP, for a prompt and then token by token.

    python examples/decoder_layer.py [--layers 2] [--prompt 300] [--tokens 8] [--graph]
                                     [--bits 4] [--rotary] [--keep 256]

Random weights, two sequences of different lengths, a window of 256 positions
with 4 first tokens that stay visible.  Every step of a decoded token is one
fixed list of launches, so with --graph the step is captured once and replayed.

--bits 4 keeps the weights in 4 bits.  --rotary turns queries and keys by their
positions.  --keep bounds the cache, in place of the window: after every step
each head keeps that many tokens, the newest quarter and the first 4 among them
and otherwise those that attention gave the most weight.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
import dslcompiler_amd as llk  # noqa: E402


class Layer:
    """Weights of one layer (norms before and after each block, bf16) and its
    cache: one slice of the model's pool."""

    def __init__(self, gen, hidden, inner, heads, kv_heads, head_dim, cache, bits=16, marks=None):
        def weight(k, n):
            w = torch.randn(k, n, generator=gen, device="cuda") * k ** -0.5
            if bits == 4:
                return llk.Q4Weights.quantise(w.bfloat16(), group=64)
            return llk.PackedWeights.from_device(w.bfloat16())

        def norm():
            return (1 + 0.1 * torch.randn(hidden, generator=gen, device="cuda")).bfloat16()

        self.heads, self.kv_heads, self.head_dim, self.cache = heads, kv_heads, head_dim, cache
        self.qkv = weight(hidden, (heads + 2 * kv_heads) * head_dim)
        self.o = weight(heads * head_dim, hidden)
        self.gate, self.up, self.down = (weight(hidden, inner), weight(hidden, inner),
                                         weight(inner, hidden))
        self.attention_norm, self.attention_post = norm(), norm()
        self.mlp_norm, self.mlp_post = norm(), norm()
        self.matmul = llk.q4_matmul if bits == 4 else llk.matmul
        self.bits, self.marks = bits, marks  # marks: weights and positions of the cache's slots

    def attend(self, x, table, lens, starts, window, sinks, max_len, turn=None, at=None):
        """Projections, cache and attention of the new tokens x [tokens, hidden],
        at positions `at`."""
        qkv = self.matmul(x, self.qkv, out_dtype=torch.bfloat16)
        qkv = qkv.unflatten(1, (self.heads + 2 * self.kv_heads, self.head_dim))
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 1)
        if turn is not None:
            q, k = llk.rotary(q, k, at, turn, q_out=q, k_out=k)
        if self.marks is None:
            llk.kv4_write(k, v, self.cache, table, lens, starts=starts)
            out = llk.kv4_attention(q, self.cache, table, lens, starts=starts, window=window,
                                    sinks=sinks, max_len=max_len)
        else:  # a slot is no position once others were evicted: no window
            weights, positions = self.marks
            llk.kv4_write(k, v, self.cache, table, lens, starts=starts, weights=weights,
                          positions=positions, at=at)
            out = llk.kv4_attention(q, self.cache, table, lens, starts=starts, max_len=max_len,
                                    weights=weights)
        return self.matmul(out.flatten(1), self.o, out_dtype=torch.bfloat16)

    def mlp(self, x):
        if self.bits == 4:
            return self.matmul(llk.q4_swiglu(x, self.gate, self.up), self.down,
                               out_dtype=torch.bfloat16)
        return llk.mlp(x, self.gate, self.up, self.down)[1]

    def evict(self, table, lens, keep, sinks, max_len):
        """Bounds the cache; the lengths stay as they are, for the other layers."""
        weights, positions = self.marks
        _, source = llk.kv4_evict_plan(weights, table, lens, keep, positions=positions,
                                       recent=keep // 4, first=sinks, max_len=max_len)
        llk.kv4_evict(self.cache, table, source, head_dim=self.head_dim, weights=weights,
                      positions=positions)


class Model:
    def __init__(self, layers=2, hidden=1024, inner=2752, heads=16, kv_heads=4, head_dim=64,
                 pages=64, page_size=32, window=256, sinks=4, seed=0, bits=16, rotary=False,
                 keep=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        pool = llk.kv4_cache(pages * layers, kv_heads, page_size, head_dim)
        pool = pool.unflatten(0, (pages, layers))  # a page of every layer together
        marks = [None] * layers
        if keep:
            every = [m.unflatten(0, (pages, layers))
                     for m in llk.kv4_marks(pages * layers, kv_heads, page_size)]
            marks = [tuple(m[:, n] for m in every) for n in range(layers)]
        self.layers = [Layer(gen, hidden, inner, heads, kv_heads, head_dim, pool[:, n], bits,
                             marks[n]) for n in range(layers)]
        self.turn = llk.RotaryTable(head_dim) if rotary else None
        self.keep = keep
        self.final_norm = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
        self.page_size, self.window, self.sinks = page_size, window, sinks
        self.scale = (2 * layers) ** -0.5  # of each block's contribution

    def forward(self, x, table, lens, starts=None, max_len=None, at=None):
        """The last layer's normed output for the new tokens x [tokens, hidden]
        (bf16); lens counts them.  at: their positions, int32 [tokens], where the
        model turns by them or bounds its cache (lens is then cut to its bound)."""
        first = self.layers[0]
        h, n = llk.block_norm(None, x, first.attention_norm)
        for i, layer in enumerate(self.layers):
            y = layer.attend(n, table, lens, starts, self.window, self.sinks, max_len, self.turn, at)
            h, n = llk.block_norm(y, h, layer.mlp_norm, post_weight=layer.attention_post,
                                  scale=self.scale)
            y = layer.mlp(n)
            following = self.layers[i + 1].attention_norm if i + 1 < len(self.layers) else \
                self.final_norm
            h, n = llk.block_norm(y, h, following, post_weight=layer.mlp_post, scale=self.scale)
        if self.keep:
            for layer in self.layers:
                layer.evict(table, lens, self.keep, self.sinks, max_len)
            lens.clamp_(max=self.keep)
        return n


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--tokens", type=int, default=8)
    ap.add_argument("--graph", action="store_true")
    ap.add_argument("--bits", type=int, default=16, choices=(4, 16))
    ap.add_argument("--rotary", action="store_true")
    ap.add_argument("--keep", type=int, default=0)
    a = ap.parse_args()
    prompts = [a.prompt, max(1, a.prompt // 3)]
    most = a.prompt + a.tokens
    model = Model(layers=a.layers, pages=2 * -(-most // 32), bits=a.bits, rotary=a.rotary,
                  keep=a.keep)
    table = torch.randperm(2 * -(-most // 32), device="cuda").int().view(2, -1)
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, prompts[0], sum(prompts)], dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(sum(prompts), 1024, generator=gen, device="cuda").bfloat16()
    at = torch.cat([torch.arange(n, dtype=torch.int32, device="cuda") for n in prompts])
    out = model.forward(x, table, lens, starts, max_len=max(prompts), at=at)
    at = torch.tensor(prompts, dtype=torch.int32, device="cuda")  # of the next tokens
    token = out[(starts[1:] - 1).long()].contiguous()  # stands for the next token's embedding

    def step():
        lens.add_(1)
        token.copy_(model.forward(token, table, lens, max_len=most, at=at))
        at.add_(1)

    replay = step
    if a.graph:
        changed = [token, lens, at]
        if a.keep:  # the cache and its marks, which an eviction moves
            changed += [t for n in model.layers for t in (n.cache, *n.marks)]
        held = [t.clone() for t in changed]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())  # for what the step changes, copied above
        with torch.cuda.stream(side):  # the library's workspace of this stream
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for t, was in zip(changed, held):
            t.copy_(was)
        replay = graph.replay
    torch.cuda.synchronize()
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for _ in range(a.tokens):
        replay()
    end.record()
    torch.cuda.synchronize()
    print(f"{a.layers} layers, prompts {prompts}, {a.tokens} tokens: lengths {lens.tolist()}, "
          f"last token begins {[round(v, 4) for v in token[:, :3].flatten().tolist()]}, "
          f"{begin.elapsed_time(end) / a.tokens * 1e3:.1f} us a step")


if __name__ == "__main__":
    main()
