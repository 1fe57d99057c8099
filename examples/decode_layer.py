"""A decoder answering token by token on NVFP4 weights: the decode-side operators together, as a serving loop uses them.

Each layer of a step takes one new token of every sequence through

    fp4_cached_gemv (QKV) -> append_qkv (head norms, rotation, cache write) -> decode_attention -> fp4_cached_gemv (output)
         -> block_norm (residual, norm) -> fp4_cached_gemv (gate, up) -> SiLU -> fp4_cached_gemv (down) -> block_norm

and the next tokens are drawn from the last one's logits by sample.  With a prompt, which is read once and shared by all
sequences, shared_prefix_attention takes decode_attention's place.  Weights are random (there is nothing to say); the layer
sizes are those of the repository's decoder-stack benchmark.  The step is captured once in a CUDA graph and replayed:
positions, slots and lengths advance on the GPU.

    python examples/decode_layer.py [--layers 2] [--batch 4] [--steps 64] [--cache nvfp4|fp8|bf16] [--prompt 0] [--temperature 0.8]
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

    def step(self, h, x, positions, slots, attend, rope):
        """A new token of every sequence: h [B, hidden] its normed residual x.  Its key and value go to `slots`; attend(q,
        cache) is its attention over what it sees, them included.  Returns (the layer's output, x)."""
        b = h.shape[0]
        qkv = fp4_gemm.fp4_cached_gemv(h, self.linears["qkv"])
        heads = qkv.view(b, self.q_heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = heads.split([self.q_heads, self.kv_heads, self.kv_heads], dim=1)
        q = self.cache.append_qkv(q, k, v, positions, slots, rope, self.q_norm, self.k_norm, eps=EPS)
        seen = attend(q, self.cache)
        h, x = fp4_decode.block_norm(fp4_gemm.fp4_cached_gemv(seen.view(b, -1), self.linears["out"]), x, self.norm2, eps=EPS)
        gate, up = fp4_gemm.fp4_cached_gemv(h, self.linears["gate_up"]).chunk(2, dim=1)
        return fp4_gemm.fp4_cached_gemv(torch.nn.functional.silu(gate) * up, self.linears["down"]), x


class Decoder:
    def __init__(self, layers=2, batch=4, room=256, hidden=2880, q_heads=64, kv_heads=8, head_dim=64, inner=7680, vocab=4096,
                 page_size=16, cache="nvfp4", device="cuda", seed=0, prompt=0, temperature=0.0, top_p=1.0):
        device = torch.device(device, torch.cuda.current_device())
        gen = torch.Generator(device).manual_seed(seed)
        wide, shared = -(-room // page_size), -(-prompt // page_size)
        self.layers = [Layer(hidden, q_heads, kv_heads, head_dim, inner, batch * wide + shared, page_size, cache, gen, device) for _ in range(layers)]
        self.embed = torch.randn(vocab, hidden, generator=gen, device=device, dtype=torch.bfloat16)
        self.head = fp4_gemm.fp4_quantize(torch.randn(vocab, hidden, generator=gen, device=device, dtype=torch.bfloat16) * hidden ** -0.5,
                                          global_scale=True)
        self.norm = torch.ones(hidden, dtype=torch.bfloat16, device=device)
        self.rope = fp4_decode.rope_table(prompt + room, head_dim, device=device)
        self.page_size, self.room = page_size, room
        # every sequence's pages, strewn over the cache
        pages = torch.randperm(batch * wide + shared, generator=gen, device=device).to(torch.int32)
        self.table = pages[: batch * wide].view(batch, wide).contiguous()
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.tokens = torch.randint(0, vocab, (batch,), generator=gen, device=device)
        self.temperature, self.top_p = temperature, top_p
        self.u = torch.rand(batch, generator=gen, device=device)  # what the next tokens are drawn by
        self.prompt = None
        if prompt:
            self.prompt = torch.randint(0, vocab, (prompt,), generator=gen, device=device)
            self.prefix_table, self.prefix_lens = pages[batch * wide:].view(1, shared).contiguous(), torch.zeros(1, dtype=torch.int32, device=device)
            for token in self.prompt.view(-1, 1):  # read once, a token at a time
                self._forward(token, self.prefix_table, self.prefix_lens, lambda q, cache: fp4_decode.decode_attention(q, cache, self.prefix_table, self.prefix_lens))

    def _forward(self, tokens, table, lens, attend, before=0):
        """The logits after `tokens`, which become part of the sequences of `table` and `lens`, behind `before` shared ones."""
        page = table.gather(1, (lens // self.page_size).long().unsqueeze(1)).squeeze(1)
        slots = page * self.page_size + lens % self.page_size
        positions = lens + before
        lens += 1
        h, x = fp4_decode.block_norm(None, self.embed[tokens], self.layers[0].norm1, eps=EPS)
        for layer, norm in zip(self.layers, [layer.norm1 for layer in self.layers[1:]] + [self.norm]):
            y, x = layer.step(h, x, positions, slots, attend, self.rope)
            h, x = fp4_decode.block_norm(y, x, norm, eps=EPS)
        return fp4_gemm.fp4_cached_gemv(h, self.head)

    def logits(self):
        """The next token's logits after self.tokens, which become part of the sequences."""
        if self.prompt is None:
            return self._forward(self.tokens, self.table, self.lens, lambda q, cache: fp4_decode.decode_attention(q, cache, self.table, self.lens))
        return self._forward(self.tokens, self.table, self.lens, lambda q, cache: fp4_decode.shared_prefix_attention(
            q, cache, self.prefix_table, self.prefix_lens, self.table, self.lens), before=len(self.prompt))

    def step(self):
        self.tokens.copy_(fp4_decode.sample(self.logits(), self.u, self.temperature, top_p=self.top_p))


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--batch", type=int, default=4)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--cache", choices=sorted(fp4_decode.KV_KINDS), default="nvfp4")
    ap.add_argument("--prompt", type=int, default=0, help="tokens of a prompt that all sequences share")
    ap.add_argument("--temperature", type=float, default=0.0)
    a = ap.parse_args()
    model = Decoder(a.layers, a.batch, room=a.steps + 4, cache=a.cache, prompt=a.prompt, temperature=a.temperature, top_p=0.95)
    model.step()  # sizes what is sized once
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.step()
    said = [model.tokens.clone()]
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(a.steps):
        model.u.uniform_()
        graph.replay()
        said.append(model.tokens.clone())
    torch.cuda.synchronize()
    took = (time.perf_counter() - began) / a.steps
    print(f"{a.layers} layers, {a.batch} sequences, {a.cache} cache, {a.prompt} shared tokens: {took * 1e6:.0f} us a step")
    print("first sequence:", torch.stack(said)[:, 0].tolist()[:16], "...")
    if fp4_gemm.device_error():
        raise SystemExit("a kernel found an index out of range")


if __name__ == "__main__":
    main()
