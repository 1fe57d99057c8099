"""The decode-side operators together: examples/decode_layer.py against the same decoder in plain torch operations, on the
weights that its caches stand for."""
import os
import sys

import pytest
import torch

from tests.conftest import ROOT
from tests.test_gpu_decode import weight_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(cuda):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_layer
    return decode_layer


def plain_logits(model, example, history, kind):
    """Logits of every step in fp32: all tokens at once under a causal mask, keys and values rounded to the cache's format."""
    from tests.test_gpu_decode import stored
    from tests import decode_reference as R

    def norm(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + example.EPS) * w.float()

    def kept(x):
        codes, scales = stored(x.to(torch.bfloat16), kind)
        return R.cache_values(codes, scales, kind).to(x.device, torch.float32)

    def linear(x, cache):
        return x @ weight_values(cache).float().T

    x = model.embed[history].float()  # [B, T, hidden]
    b, t, _ = x.shape
    positions = torch.arange(t, device=x.device)
    for layer in model.layers:
        hq, hk, d = layer.q_heads, layer.kv_heads, layer.head_dim
        heads = linear(norm(x, layer.norm1), layer.linears["qkv"]).view(b * t, hq + 2 * hk, d)
        q, k, v = heads.split([hq, hk, hk], dim=1)
        at = positions.repeat(b)
        q = R.norm_rope(q, layer.q_norm, at, model.rope, example.EPS, False).float().view(b, t, hk, hq // hk, d)
        k = kept(R.norm_rope(k, layer.k_norm, at, model.rope, example.EPS, False).float()).view(b, t, hk, d)
        v = kept(v).view(b, t, hk, d)
        s = torch.einsum("bihgd,bjhd->bhgij", q, k) * d ** -0.5
        s = s.masked_fill(positions[None, :] > positions[:, None], float("-inf"))
        o = torch.einsum("bhgij,bjhd->bihgd", s.softmax(-1), v).reshape(b, t, hq * d)
        x = x + linear(o, layer.linears["out"])
        gate, up = linear(norm(x, layer.norm2), layer.linears["gate_up"]).chunk(2, dim=-1)
        x = x + linear(torch.nn.functional.silu(gate) * up, layer.linears["down"])
    return linear(norm(x, model.norm), model.head)


@pytest.mark.parametrize("kind", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("sizes", [dict(hidden=256, q_heads=4, kv_heads=2, head_dim=64, inner=320, vocab=500, batch=3),
                                   dict(hidden=384, q_heads=3, kv_heads=1, head_dim=128, inner=200, vocab=130, batch=5)])
def test_decoder_step_by_step(example, fp4, kind, sizes):
    steps = 37
    model = example.Decoder(layers=2, room=40, page_size=8, cache=kind, **sizes)
    history, got = [], []
    for _ in range(steps):
        history.append(model.tokens.clone())
        logits = model.logits()
        got.append(logits)
        model.tokens.copy_(logits.argmax(-1))
    got, history = torch.stack(got, 1).float(), torch.stack(history, 1)
    want = plain_logits(model, example, history, kind)
    # Activations are rounded to BF16 about ten times a layer (2^-9 of their size each, at random), and a key near a boundary
    # of its format may fall to the other side: 3 % of the logits' size in all for BF16 and fp8 and 6 % for nvfp4 is ample.
    rel = (got - want).norm() / want.norm()
    assert rel < {"bf16": 0.03, "fp8": 0.03, "nvfp4": 0.06}[kind], rel
    assert fp4.device_error() == 0


def test_captured_decoder_says_the_same(example, fp4):
    sizes = dict(layers=2, batch=3, room=64, hidden=256, q_heads=4, kv_heads=2, head_dim=64, inner=320, vocab=500, cache="nvfp4")
    eager, captured = example.Decoder(**sizes), example.Decoder(**sizes)
    said = []
    for _ in range(20):
        eager.step()
        said.append(eager.tokens.clone())
    captured.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for i in range(1, 20):
        graph.replay()
        assert torch.equal(captured.tokens, said[i]), i
    assert fp4.device_error() == 0
