"""What closes a decoding step, together with the rest of it: examples/decode_layer.py with a prompt that all sequences share and
tokens drawn from given numbers, against the same decoder in plain torch operations."""
import os
import sys

import pytest
import torch

from tests import sample_reference as S
from tests.conftest import ROOT
from tests.test_gpu_decode_layer import plain_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(cuda):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import decode_layer
    return decode_layer


SIZES = dict(hidden=256, q_heads=4, kv_heads=2, head_dim=64, inner=320, vocab=500, batch=3)


@pytest.mark.parametrize("kind", ["bf16", "fp8", "nvfp4"])
@pytest.mark.parametrize("prompt", [1, 21])
def test_decoder_behind_a_shared_prompt(example, fp4, kind, prompt):
    steps = 15
    model = example.Decoder(layers=2, room=20, page_size=8, cache=kind, prompt=prompt, **SIZES)
    history, got = [], []
    for _ in range(steps):
        history.append(model.tokens.clone())
        logits = model.logits()
        got.append(logits)
        model.tokens.copy_(logits.argmax(-1))
    got = torch.stack(got, 1).float()
    history = torch.cat((model.prompt.expand(SIZES["batch"], -1), torch.stack(history, 1)), 1)
    want = plain_logits(model, example, history, kind)[:, prompt:]
    # the bounds of test_decoder_step_by_step, for the same reasons
    rel = (got - want).norm() / want.norm()
    assert rel < {"bf16": 0.03, "fp8": 0.03, "nvfp4": 0.06}[kind], rel
    assert fp4.device_error() == 0


@pytest.mark.parametrize("prompt", [0, 33])
def test_captured_decoder_draws_the_same(example, fp4, prompt):
    sizes = dict(SIZES, layers=2, room=64, cache="nvfp4", prompt=prompt, temperature=0.9, top_p=0.95)
    eager, captured = example.Decoder(**sizes), example.Decoder(**sizes)
    numbers = torch.rand(20, SIZES["batch"], generator=torch.Generator().manual_seed(1)).to(eager.u.device)
    said = []
    for u in numbers:
        eager.u.copy_(u)
        eager.step()
        said.append(eager.tokens.clone())
    captured.u.copy_(numbers[0])
    captured.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for i in range(1, 20):
        captured.u.copy_(numbers[i])
        graph.replay()
        assert torch.equal(captured.tokens, said[i]), i
    assert fp4.device_error() == 0


def test_tokens_are_the_logits_own(example, fp4):
    model, twin = (example.Decoder(layers=1, room=20, cache="bf16", prompt=9, temperature=0.8, top_p=0.9, **SIZES) for _ in range(2))
    for _ in range(5):
        logits = twin.logits().double().cpu().numpy()
        want = [S.draw(logits[i], float(model.u[i]), float(torch.tensor(0.8)), 0, float(torch.tensor(0.9)), 0.0)[0] for i in range(SIZES["batch"])]
        model.step()
        assert model.tokens.tolist() == want
        twin.tokens.copy_(model.tokens)
        model.u.uniform_()
