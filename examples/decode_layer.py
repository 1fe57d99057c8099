"""A decoder answering token by token on NVFP4 weights: the decode-side operators together, as a serving loop uses them.

Each layer of a step takes one new token of every sequence through

    norm -> fp4_cached_gemv (QKV) -> append_qkv (head norms, rotation, cache write) -> decode_attention
         -> fp4_cached_gemv (output) -> norm -> fp4_cached_gemv (gate, up) -> SiLU -> fp4_cached_gemv (down)

and the last one's logits choose the next token.  Weights are random (there is nothing to say); the layer sizes are those of
the repository's decoder-stack benchmark.  The step is captured once in a CUDA graph and replayed: positions, slots and
lengths advance on the GPU.

    python examples/decode_layer.py [--layers 2] [--batch 4] [--steps 64] [--cache nvfp4|fp8|bf16]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp4-gemm-blackwell_b200"))
import fp4_decode  # noqa: E402
import fp4_gemm  # noqa: E402

EPS = 1e-6


def rms_norm(x, weight):
    y = x.float()
    return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.float()).to(torch.bfloat16)


class Layer:
    """One decoder layer: NVFP4 linears, BF16 norms, a paged key-value cache of its own."""

    def __init__(self, hidden, q_heads, kv_heads, head_dim, inner, pages, page_size, cache, gen, device):
        def weight(n, k):
            return torch.randn(n, k, generator=gen, device=device, dtype=torch.bfloat16) * k ** -0.5

        def ones(n):
            return (1 + 0.1 * torch.randn(n, generator=gen, device=device)).to(torch.bfloat16)

        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.weights = {"qkv": weight((q_heads + 2 * kv_heads) * head_dim, hidden), "out": weight(hidden, q_heads * head_dim),
                        "gate_up": weight(2 * inner, hidden), "down": weight(hidden, inner)}
        self.linears = {name: fp4_gemm.fp4_quantize(w, global_scale=True) for name, w in self.weights.items()}
        self.norm1, self.norm2, self.q_norm, self.k_norm = ones(hidden), ones(hidden), ones(head_dim), ones(head_dim)
        self.cache = fp4_decode.PagedKVCache(pages, page_size, kv_heads, head_dim, cache, device=device)

    def step(self, x, positions, slots, table, lens, rope):
        """x [B, hidden]: each sequence's new token; its key and value go to `slots`, and are seen by it (lens counts it)."""
        b = x.shape[0]
        qkv = fp4_gemm.fp4_cached_gemv(rms_norm(x, self.norm1), self.linears["qkv"])
        heads = qkv.view(b, self.q_heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = heads.split([self.q_heads, self.kv_heads, self.kv_heads], dim=1)
        q = self.cache.append_qkv(q, k, v, positions, slots, rope, self.q_norm, self.k_norm, eps=EPS)
        seen = fp4_decode.decode_attention(q, self.cache, table, lens)
        x = x + fp4_gemm.fp4_cached_gemv(seen.view(b, -1), self.linears["out"])
        gate, up = fp4_gemm.fp4_cached_gemv(rms_norm(x, self.norm2), self.linears["gate_up"]).chunk(2, dim=1)
        return x + fp4_gemm.fp4_cached_gemv(torch.nn.functional.silu(gate) * up, self.linears["down"])


class Decoder:
    def __init__(self, layers=2, batch=4, room=256, hidden=2880, q_heads=64, kv_heads=8, head_dim=64, inner=7680, vocab=4096,
                 page_size=16, cache="nvfp4", device="cuda", seed=0):
        device = torch.device(device, torch.cuda.current_device())
        gen = torch.Generator(device).manual_seed(seed)
        wide = -(-room // page_size)
        self.layers = [Layer(hidden, q_heads, kv_heads, head_dim, inner, batch * wide, page_size, cache, gen, device) for _ in range(layers)]
        self.embed = torch.randn(vocab, hidden, generator=gen, device=device, dtype=torch.bfloat16)
        self.head = fp4_gemm.fp4_quantize(torch.randn(vocab, hidden, generator=gen, device=device, dtype=torch.bfloat16) * hidden ** -0.5,
                                          global_scale=True)
        self.norm = torch.ones(hidden, dtype=torch.bfloat16, device=device)
        self.rope = fp4_decode.rope_table(room, head_dim, device=device)
        self.page_size, self.room = page_size, room
        # every sequence's pages, strewn over the cache
        self.table = torch.randperm(batch * wide, generator=gen, device=device).to(torch.int32).view(batch, wide).contiguous()
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.tokens = torch.randint(0, vocab, (batch,), generator=gen, device=device)

    def logits(self):
        """The next token's logits after self.tokens, which become part of the sequences."""
        positions = self.lens.clone()
        page = self.table.gather(1, (positions // self.page_size).long().unsqueeze(1)).squeeze(1)
        slots = page * self.page_size + positions % self.page_size
        self.lens += 1
        x = self.embed[self.tokens]
        for layer in self.layers:
            x = layer.step(x, positions, slots, self.table, self.lens, self.rope)
        return fp4_gemm.fp4_cached_gemv(rms_norm(x, self.norm), self.head)

    def step(self):
        self.tokens.copy_(self.logits().argmax(dim=-1))


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--cache", choices=sorted(fp4_decode.KV_KINDS), default="nvfp4")
    a = ap.parse_args()
    model = Decoder(a.layers, a.batch, room=a.steps + 4, cache=a.cache)
    model.step()  # sizes what is sized once
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.step()
    said = [model.tokens.clone()]
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(a.steps):
        graph.replay()
        said.append(model.tokens.clone())
    torch.cuda.synchronize()
    took = (time.perf_counter() - began) / a.steps
    print(f"{a.layers} layers, {a.batch} sequences, {a.cache} cache: {took * 1e6:.0f} us a step")
    print("first sequence:", torch.stack(said)[:, 0].tolist()[:16], "...")
    if fp4_gemm.device_error():
        raise SystemExit("a kernel found an index out of range")


if __name__ == "__main__":
    main()
