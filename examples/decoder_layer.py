"""A decoder layer on the gfx950 kernels: norms, projections, a 4-bit paged
cache, attention and the SwiGLU MLP, for a prompt and then token by token.

    python examples/decoder_layer.py [--layers 2] [--prompt 300] [--tokens 8] [--graph]

Random weights, two sequences of different lengths, a window of 256 positions
with 4 first tokens that stay visible.  Every step of a decoded token is one
fixed list of launches, so with --graph the step is captured once and replayed.
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

    def __init__(self, gen, hidden, inner, heads, kv_heads, head_dim, cache):
        def weight(k, n):
            w = torch.randn(k, n, generator=gen, device="cuda") * k ** -0.5
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

    def attend(self, x, table, lens, starts, window, sinks, max_len):
        """Projections, cache and attention of the new tokens x [tokens, hidden]."""
        qkv = llk.matmul(x, self.qkv, out_dtype=torch.bfloat16)
        qkv = qkv.unflatten(1, (self.heads + 2 * self.kv_heads, self.head_dim))
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 1)
        llk.kv4_write(k, v, self.cache, table, lens, starts=starts)
        out = llk.kv4_attention(q, self.cache, table, lens, starts=starts, window=window,
                                sinks=sinks, max_len=max_len)
        return llk.matmul(out.flatten(1), self.o, out_dtype=torch.bfloat16)


class Model:
    def __init__(self, layers=2, hidden=1024, inner=2752, heads=16, kv_heads=4, head_dim=64,
                 pages=64, page_size=32, window=256, sinks=4, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        pool = llk.kv4_cache(pages * layers, kv_heads, page_size, head_dim)
        pool = pool.unflatten(0, (pages, layers))  # a page of every layer together
        self.layers = [Layer(gen, hidden, inner, heads, kv_heads, head_dim, pool[:, n])
                       for n in range(layers)]
        self.final_norm = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
        self.page_size, self.window, self.sinks = page_size, window, sinks
        self.scale = (2 * layers) ** -0.5  # of each block's contribution

    def forward(self, x, table, lens, starts=None, max_len=None):
        """The last layer's normed output for the new tokens x [tokens, hidden]
        (bf16); lens counts them."""
        first = self.layers[0]
        h, n = llk.block_norm(None, x, first.attention_norm)
        for i, layer in enumerate(self.layers):
            y = layer.attend(n, table, lens, starts, self.window, self.sinks, max_len)
            h, n = llk.block_norm(y, h, layer.mlp_norm, post_weight=layer.attention_post,
                                  scale=self.scale)
            _, y = llk.mlp(n, layer.gate, layer.up, layer.down)
            following = self.layers[i + 1].attention_norm if i + 1 < len(self.layers) else \
                self.final_norm
            h, n = llk.block_norm(y, h, following, post_weight=layer.mlp_post, scale=self.scale)
        return n


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--tokens", type=int, default=8)
    ap.add_argument("--graph", action="store_true")
    a = ap.parse_args()
    prompts = [a.prompt, max(1, a.prompt // 3)]
    most = a.prompt + a.tokens
    model = Model(layers=a.layers, pages=2 * -(-most // 32))
    table = torch.randperm(2 * -(-most // 32), device="cuda").int().view(2, -1)
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, prompts[0], sum(prompts)], dtype=torch.int32, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(sum(prompts), 1024, generator=gen, device="cuda").bfloat16()
    out = model.forward(x, table, lens, starts, max_len=max(prompts))
    token = out[(starts[1:] - 1).long()].contiguous()  # stands for the next token's embedding

    def step():
        lens.add_(1)
        token.copy_(model.forward(token, table, lens, max_len=most))

    replay = step
    if a.graph:
        held = token.clone(), lens.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())  # for what the step changes, copied above
        with torch.cuda.stream(side):  # the library's workspace of this stream
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        token.copy_(held[0])
        lens.copy_(held[1])
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
