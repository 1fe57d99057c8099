"""fp4_decode.block_norm on a B200 against its formula in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8  # of BF16


@pytest.fixture(scope="module")
def dec(cuda):
    import fp4_decode
    return fp4_decode


def formula(x, residual, weight, post_weight, gate, scale, eps):
    """(normed, r, what was added to the residual, 1 / root of its mean square) in 64 bits."""
    r, f = residual.double(), None
    if x is not None:
        f = x.double()
        if post_weight is not None:
            f = f / torch.sqrt(f.square().mean(-1, keepdim=True) + eps) * post_weight.double()
        if gate is not None:
            f = f * gate.double()
        f = f * scale
        r = r + f
    factor = 1.0 / torch.sqrt(r.square().mean(-1, keepdim=True) + eps)
    return r * factor * weight.double(), r, torch.zeros_like(r) if f is None else f, factor


def check(dec, x, residual, weight, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    normed, out = dec.block_norm(x, residual, weight, post_weight, gate, scale, eps)
    assert normed.dtype == torch.bfloat16 and normed.shape == residual.shape and out.dtype == residual.dtype and out.shape == residual.shape
    want, r, f, factor = formula(x, residual, weight, post_weight, gate, scale, eps)
    # fp32: a sum of squares is off by 2^-24 for each of a thread's up to 64 terms and the 10 steps of joining, half of that
    # behind the root, whose reciprocal is off by 2^-22; five products by 2^-24 each: 2^-18 of a factor in all.
    added = 2.0 ** -18 * f.abs() + 2.0 ** -24 * r.abs()
    half = 2.0 ** -24 if residual.dtype == torch.float32 else HALF
    tiny = 2.0 ** -133  # half a step of the smallest BF16
    if x is None:
        assert out is residual
    else:
        bad = (out.double() - r).abs() > half * r.abs() + added + tiny
        assert not bad.any(), (int(bad.sum()), (out.double() - r).abs().max().item())
    tol = HALF * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -18 * want.abs() + added * factor * weight.double().abs() + tiny
    bad = (normed.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), (normed.double() - want).abs().max().item())
    return normed, out


def inputs(t, h, cuda, kind, seed=0):
    g = torch.Generator(cuda).manual_seed(seed + t + h)

    def randn(*s):
        return torch.randn(*s, generator=g, device=cuda)

    residual = (3 * randn(t, h)).to(kind)
    weights = [(1 + 0.2 * randn(h)).bfloat16() for _ in range(2)]
    return randn(t, h).bfloat16(), residual, weights, [None, (1 + 0.3 * randn(h)).bfloat16(), torch.sigmoid(randn(t, h)).bfloat16()]


WIDTHS = [1, 2, 6, 7, 8, 31, 64, 255, 256, 264, 1000, 1001, 2880, 4096, 4097, 5003, 5118, 5120, 5122, 8192, 8193, 16384, 16392, 20001, 32750, 32760, 32767, 32768]


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("h", WIDTHS)
def test_every_part(dec, cuda, kind, h):
    for t in (1, 5):
        x, residual, (w, post), gates = inputs(t, h, cuda, kind)
        for gate in gates:
            check(dec, x, residual, w, None, gate, 0.5)
            check(dec, x, residual, w, post, gate, -1.25, 1e-3)
        check(dec, None, residual, w)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,h", [(1021, 520), (70000, 24), (300, 2880), (4099, 129)])
def test_many_rows(dec, cuda, kind, t, h):
    x, residual, (w, post), gates = inputs(t, h, cuda, kind)
    check(dec, x, residual, w, post, gates[2], 0.22)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_rows_of_any_stride_and_start(dec, cuda, kind):
    t, h = 6, 264
    x, residual, (w, post), gates = inputs(t, h, cuda, kind)
    want = dec.block_norm(x, residual, w, post, gates[2])
    for pad, at in ((8, 0), (8, 8), (5, 0), (9, 3), (16, 1)):
        def skew(v):
            wide = torch.zeros(*v.shape[:-1], h + pad + at, dtype=v.dtype, device=cuda)
            wide[..., at: at + h] = v
            return wide[..., at: at + h]
        got = check(dec, skew(x), skew(residual), skew(w), skew(post), skew(gates[2]))
        # (other threads add other parts of a sum: the same to fp32's rounding, rarely another BF16)
        assert all(((a.double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 2.0 ** -20).all() for a, b in zip(got, want))
    check(dec, x.t().contiguous().t(), residual.t().contiguous().t(), w, post, gates[2].t().contiguous().t())
    check(dec, x[:1].expand(t, h), residual[:1].expand(t, h), w)
    check(dec, x.view(2, 3, h), residual.view(2, 3, h), w, post, gates[2].view(2, 3, h))
    check(dec, x.view(2, 3, h), residual.view(2, 3, h), w, post, gates[1])
    check(dec, x.view(2, 3, h).transpose(0, 1), residual.view(2, 3, h).transpose(0, 1), w)
    check(dec, x[0], residual[0], w)


def test_values_that_cancel_and_extremes(dec, cuda):
    h = 520
    x, residual, (w, post), _ = inputs(4, h, cuda, torch.float32)
    residual = -x.float() * (1 + 2.0 ** -20)
    check(dec, x, residual, w)
    zero = torch.zeros_like(x)
    check(dec, zero, zero.float(), w, post)  # rows of zeros: 1 / root of eps, zeros
    check(dec, x * 2.0 ** 40, residual * 2.0 ** -40, w, post)
    check(dec, x * 2.0 ** -60, residual * 2.0 ** -60, w, post, eps=1e-12)
    bad = x.clone()
    bad[1, 3] = float("nan")
    bad[2, 5] = float("inf")
    normed, out = dec.block_norm(bad, residual, w, post)
    good = dec.block_norm(x, residual, w, post)
    assert torch.isnan(normed[1]).all() and torch.isnan(out[2, 5])  # a row's own
    assert all(torch.equal(a[[0, 3]], b[[0, 3]]) for a, b in zip((normed, out), good))


def test_other_types_are_cast(dec, cuda):
    x, residual, (w, post), gates = inputs(3, 200, cuda, torch.bfloat16)
    want = dec.block_norm(x, residual, w, post, gates[1])
    got = dec.block_norm(x.float(), residual.half().float().bfloat16(), w.float(), post.double(), gates[1].float())
    assert torch.equal(got[1], want[1]) and torch.equal(got[0], want[0])
    assert dec.block_norm(x, residual.half(), w)[1].dtype == torch.bfloat16


def test_captured(dec, cuda):
    x, residual, (w, post), gates = inputs(33, 2880, cuda, torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = dec.block_norm(x, residual, w, post, gates[1])
    x.mul_(-2.0)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, dec.block_norm(x, residual, w, post, gates[1])))


def test_nothing_to_do_and_refusals(dec, cuda):
    x, residual, (w, post), gates = inputs(3, 64, cuda, torch.bfloat16)
    normed, out = dec.block_norm(x[:0], residual[:0], w)
    assert normed.shape == (0, 64) and out.shape == (0, 64)
    for bad in (dict(x=x[:2]), dict(x=x.cpu()), dict(weight=w[:63]), dict(weight=w.cpu()), dict(post_weight=post[:5]), dict(gate=gates[2][:2]),
                dict(gate=gates[2][:, :1]), dict(x=None, gate=gates[1]), dict(x=None, post_weight=post), dict(residual=residual.cpu()),
                dict(residual=residual[:, :0], x=x[:, :0])):
        with pytest.raises(ValueError):
            dec.block_norm(**{**dict(x=x, residual=residual, weight=w), **bad})
    for bad in (dict(scale=float("inf")), dict(eps=-1.0), dict(eps=float("nan"))):
        with pytest.raises(RuntimeError):
            dec.block_norm(**{**dict(x=x, residual=residual, weight=w), **bad})
    with pytest.raises(ValueError):
        dec.block_norm(None, torch.zeros(1, 32769, device=cuda), torch.zeros(32769, device=cuda))
