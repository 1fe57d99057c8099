"""fp4_decode.sample on a B200 against tests/sample_reference.py: the tokens have to be the same, the shares within fp32's
rounding (2^-24) and one unit of the kernel's weights."""
import math

import numpy as np
import pytest
import torch

from tests import sample_reference as R

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
LAST = 1.0 - 2.0 ** -24


@pytest.fixture(scope="module")
def dec(cuda):
    import fp4_decode
    return fp4_decode


def per_row(v, b):
    return v.cpu().double().reshape(-1).tolist() if isinstance(v, torch.Tensor) else [float(np.float32(v))] * b


def check(dec, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, what=""):
    tokens, probs = dec.sample(logits, u, temperature, top_k, top_p, min_p, return_prob=True)
    assert tokens.dtype == torch.int64 and probs.dtype == torch.float32
    assert torch.equal(tokens, dec.sample(logits, u, temperature, top_k, top_p, min_p))
    b = logits.shape[0]
    rows, settings = logits.double().cpu().numpy(), [per_row(x, b) for x in (u, temperature, top_k, top_p, min_p)]
    for i in range(b):
        uu, t, k, p, m = (x[i] for x in settings)
        want, share = R.draw(rows[i], uu, t, int(k), p, m)
        assert int(tokens[i]) == want, (what, i, int(tokens[i]), want, uu, t, k, p, m)
        # the weight and the sum are whole multiples of 2^-44 or less (of a largest weight of 1), the share is rounded to fp32
        assert abs(float(probs[i]) - share) <= 2.0 ** -23 * share + 2.0 ** -40, (what, i, float(probs[i]), share)
    return tokens


def settings(b, g, cuda):
    def between(lo, hi):
        return lo + (hi - lo) * torch.rand(b, generator=g, device=cuda)

    i = torch.arange(b, device=cuda)
    t = torch.where(i % 7 == 6, torch.zeros(b, device=cuda), between(0.2, 1.5))
    k = torch.where(i % 2 == 0, torch.randint(1, 500, (b,), generator=g, device=cuda), torch.zeros_like(i)).int()
    p = torch.where(i % 3 != 1, between(0.3, 0.99), torch.ones(b, device=cuda))
    m = torch.where(i % 4 == 3, between(0.001, 0.2), torch.zeros(b, device=cuda))
    return t, k, p, m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,v", [(1, 1), (3, 2), (5, 7), (9, 100), (33, 1000), (64, 4097), (2, 20000), (1, 50001), (300, 2048), (5, 131072), (2, 300001)])
def test_mixed_settings(dec, cuda, dtype, b, v):
    g = torch.Generator(cuda).manual_seed(b * 1000 + v)
    logits = (3.0 * torch.randn(b, v, generator=g, device=cuda)).to(dtype)
    u = torch.rand(b, generator=g, device=cuda)
    check(dec, logits, u, *settings(b, g, cuda))
    check(dec, logits, u, 0.8)
    check(dec, logits, u, 1.0, 3, 0.9, 0.01)


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_logits_go_by_index(dec, cuda, dtype):
    # all weights are 1: token j is drawn for u in [j / V, (j + 1) / V), p keeps p * V, k the first k
    v = 256
    for value in (0.0, -0.0, 3.5, -7.0, 1e-7, -60000.0):
        u = torch.arange(v, device=cuda).float() / v
        logits = torch.full((v, v), value, device=cuda).to(dtype)
        logits[:, 3::5] *= -1.0 if value == 0 else 1.0
        assert check(dec, logits, u).tolist() == list(range(v))
        assert check(dec, logits, u, top_p=0.5).tolist() == [j // 2 for j in range(v)]
        assert check(dec, logits, u, top_k=64).tolist() == [j // 4 for j in range(v)]
        assert check(dec, logits, u, top_k=64, top_p=0.25).tolist() == [j // 16 for j in range(v)]
        assert check(dec, logits, u, top_k=1).tolist() == [0] * v
        assert check(dec, logits, u, min_p=1.0).tolist() == list(range(v))
        assert check(dec, logits, u, temperature=0.0).tolist() == [0] * v


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [70, 5000, 40000])
def test_ties_at_every_border(dec, cuda, dtype, v):
    # few levels, many equal logits: k, p and u all end among equals
    g = torch.Generator(cuda).manual_seed(v)
    b = 48
    logits = torch.randint(-3, 4, (b, v), generator=g, device=cuda).to(dtype)
    u = torch.rand(b, generator=g, device=cuda)
    k = torch.randint(1, v, (b,), generator=g, device=cuda).int()
    p = torch.rand(b, generator=g, device=cuda)
    check(dec, logits, u, 1.3, k, 1.0, 0.0)
    check(dec, logits, u, 0.9, 0, p, 0.0)
    check(dec, logits, u, 2.0, k, p, 0.02)


@pytest.mark.parametrize("dtype", TYPES)
def test_masks_and_what_is_no_number(dec, cuda, dtype):
    v, inf, nan = 700, math.inf, math.nan
    g = torch.Generator(cuda).manual_seed(1)
    low = torch.finfo(dtype).min
    logits = torch.randn(12, v, generator=g, device=cuda).to(dtype)
    logits[0] = -inf                      # a mask that leaves nothing
    logits[1] = -inf
    logits[1, 699] = -3.0                 # one token
    logits[2] = nan
    logits[3] = nan
    logits[3, 5] = 2.0
    logits[4, 100:110] = inf              # ten that are infinitely likely
    logits[5] = low                       # the type's lowest value as a mask that leaves nothing: all alike
    logits[6] = low
    logits[6, [3, 77]] = 1.0
    logits[7, ::2] = -inf
    logits[7, 1::4] = nan
    logits[8] = inf
    logits[9] = torch.finfo(dtype).max
    logits[10, :300] = low
    logits[11] = torch.finfo(dtype).tiny * torch.randint(-3, 4, (v,), generator=g, device=cuda)
    for at in (0.0, 0.3, 0.77, LAST):
        u = torch.full((12,), at, device=cuda)
        for args in ((1.0,), (0.5, 20), (1.0, 0, 0.6), (1.5, 0, 1.0, 0.1), (0.7, 50, 0.9, 0.05), (0.0,)):
            tokens = check(dec, logits, u, *args, what=f"u {at} {args}")
            assert tokens[0] == -1 and tokens[2] == -1 and tokens[1] == 699 and tokens[3] == 5


@pytest.mark.parametrize("dtype", TYPES)
def test_settings_at_their_ends(dec, cuda, dtype):
    g = torch.Generator(cuda).manual_seed(2)
    b, v = 6, 3001
    logits = (2.0 * torch.randn(b, v, generator=g, device=cuda)).to(dtype)
    u = torch.tensor([0.0, 1e-30, 0.5, LAST, 1.0, 7.0], device=cuda)
    for t in (1e-30, 1e-3, 0.05, 1.0, 50.0, 1e30, math.inf):
        check(dec, logits, u, t, what=f"T {t}")
    for t in (math.nan, -1.0):  # as 0 (known on the GPU only)
        assert torch.equal(dec.sample(logits, u, torch.full((b,), t, device=cuda)), logits.float().argmax(1))
    for p in (0.0, -1.0, 1e-30, 1e-3, LAST, 1.0, 2.0):
        check(dec, logits, u, 1.0, 0, p, what=f"p {p}")
    for k in (-5, 0, 1, 2, v - 1, v, v + 1, 2 ** 31 - 1):
        check(dec, logits, u, 1.0, k, what=f"k {k}")
        check(dec, logits, u, 1.0, torch.full((b,), k, dtype=torch.int32, device=cuda), 0.9, what=f"k {k}")
    for m in (-1.0, 0.0, 1e-30, 0.5, 1.0, 3.0):
        check(dec, logits, u, 1.0, 0, 1.0, m, what=f"min-p {m}")
    nan = torch.full((b,), math.nan, device=cuda)
    assert torch.equal(dec.sample(logits, u, 1.0, 0, nan, nan), dec.sample(logits, u, 1.0))
    assert torch.equal(dec.sample(logits, nan, 1.0), dec.sample(logits, torch.zeros(b, device=cuda), 1.0))
    assert torch.equal(dec.sample(logits, -u, 1.0), dec.sample(logits, torch.zeros(b, device=cuda), 1.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread,shift", [(1e-6, 0.0), (1e-3, 20.0), (0.3, -40.0), (100.0, 0.0), (3000.0, -5000.0)])
def test_logits_of_any_size(dec, cuda, dtype, spread, shift):
    # near zero (where the bins end), far from it, all close together, far apart
    g = torch.Generator(cuda).manual_seed(3)
    b, v = 12, 9000
    logits = (spread * torch.randn(b, v, generator=g, device=cuda) + shift).to(dtype)
    u = torch.rand(b, generator=g, device=cuda)
    check(dec, logits, u, 1.0, 0, 0.9)
    check(dec, logits, u, spread, 700, 0.95, 0.01)
    check(dec, logits, u, 20.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b", [1, 40, 700])
def test_rows_of_any_stride_and_start(dec, cuda, dtype, b):
    g = torch.Generator(cuda).manual_seed(b)
    v = 5003
    wide = torch.randn(b, v + 13, generator=g, device=cuda).to(dtype)
    u = torch.rand(b, generator=g, device=cuda)
    for at in (0, 1, 3, 8, 13):
        part = wide[:, at: at + v]
        assert torch.equal(dec.sample(part, u, 0.9, 100, 0.9), dec.sample(part.clone(memory_format=torch.contiguous_format), u, 0.9, 100, 0.9))
    check(dec, wide[:7, 1: 1 + v], u[:7], 0.9, 0, 0.9)
    turned = torch.randn(30, 20, generator=g, device=cuda).to(dtype).t()
    assert torch.equal(dec.sample(turned, u.new_full((20,), 0.4)), dec.sample(turned.contiguous(), u.new_full((20,), 0.4)))
    one = wide[:1].expand(9, v + 13)  # one row for all
    assert torch.equal(dec.sample(one, u.new_full((9,), 0.4)), dec.sample(one.contiguous(), u.new_full((9,), 0.4)))


def test_captured_with_other_streams_beside_it(dec, cuda):
    g = torch.Generator(cuda).manual_seed(5)
    logits, u = torch.randn(8, 30000, generator=g, device=cuda).bfloat16(), torch.rand(8, generator=g, device=cuda)
    t = torch.full((8,), 0.7, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dec.sample(logits, u, t, 40, 0.9)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, probs = dec.sample(logits, u, t, 40, 0.9, return_prob=True)
    for seed in range(3):
        logits.copy_(torch.randn(8, 30000, generator=g, device=cuda))
        u.copy_(torch.rand(8, generator=g, device=cuda))
        graph.replay()
        with torch.cuda.stream(side):
            other = dec.sample(logits, u, t, 40, 0.9)
        want = dec.sample(logits, u, t, 40, 0.9, return_prob=True)
        torch.cuda.synchronize()
        assert torch.equal(tokens, want[0]) and torch.equal(probs, want[1]) and torch.equal(other, want[0])


def test_shares_are_drawn_as_often(dec, cuda):
    # u over an even grid of 2^16 numbers: each token as often as its share says, to within one at each end
    g = torch.Generator(cuda).manual_seed(6)
    n = 1 << 16
    logits = torch.randn(1, 50, generator=g, device=cuda)
    u = (torch.arange(n, device=cuda).float() + 0.5) / n
    tokens = dec.sample(logits.expand(n, 50), u)
    share = torch.softmax(logits[0].double(), 0)
    assert ((torch.bincount(tokens, minlength=50) - share * n).abs() <= 1.0 + 1e-6).all()


def test_nothing_to_do_and_refusals(dec, cuda):
    logits, u = torch.zeros(2, 5, device=cuda), torch.zeros(2, device=cuda)
    assert dec.sample(logits[:0], u[:0]).shape == (0,)
    for bad in (dict(logits=logits[0]), dict(logits=logits.double()), dict(logits=logits.cpu()), dict(logits=logits[:, :0]), dict(u=u[:1]),
                dict(u=u.double()), dict(u=u.cpu()), dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=u[:1]), dict(top_k=u.cpu()),
                dict(top_p=torch.zeros(3, device=cuda)), dict(min_p=torch.zeros(2))):
        with pytest.raises(ValueError):
            dec.sample(**{**dict(logits=logits, u=u), **bad})
