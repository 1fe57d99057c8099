"""fp4_decode.shared_prefix_attention on a B200 against tests/shared_reference.py."""
import math

import pytest
import torch

from tests import decode_reference as R
from tests import shared_reference as S

pytestmark = pytest.mark.gpu
KINDS = ["bf16", "fp8", "nvfp4"]


@pytest.fixture(scope="module")
def dec(cuda):
    import fp4_decode
    return fp4_decode


def case(dec, cuda, kind, d, hq, hk, page, shared, mine, seed=0, spread=1.5, width=None, shared_width=None):
    """(q, cache, prefix_table, prefix_lens, page_table, lens) of prefixes of `shared` keys and sequences with `mine` of their own."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in [*shared, *mine]]
    pages = max(1, sum(need)) + 2
    cache = dec.PagedKVCache(pages, page, hk, d, kind, device=cuda)
    k, v = ((torch.randn(pages * page, hk, d, generator=g) * s).to(torch.bfloat16).to(cuda) for s in (spread, 1.0))
    cache.append(k, v, torch.arange(pages * page, device=cuda))
    order = torch.randperm(pages, generator=g).to(torch.int32)

    def table(lens, at, wide):
        t = torch.full((len(lens), max([1] + [-(-n // page) for n in lens]) if wide is None else wide), -7, dtype=torch.int32)
        for i, n in enumerate(lens):
            n = -(-n // page)
            t[i, :n] = order[at: at + n]
            at += n
        return t.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)

    q = (torch.randn(len(mine), hq, d, generator=g) * spread).to(torch.bfloat16).to(cuda)
    return (q, cache, *table(shared, 0, shared_width), *table(mine, sum(need[: len(shared)]), width))


def check(dec, q, cache, prefix_table, prefix_lens, table, lens, sinks=None, scale=None):
    args = (q, cache, prefix_table, prefix_lens, table, lens)
    out, lse = dec.shared_prefix_attention(*args, scale=scale, sinks=sinks, return_lse=True)
    k, v = R.cache_values(cache.k_pages, cache.k_scales, cache.dtype), R.cache_values(cache.v_pages, cache.v_scales, cache.dtype)
    by = q.shape[-1] ** -0.5 if scale is None else scale
    want, wlse, mag = S.attention(q, k, v, prefix_table, prefix_lens, table, lens, cache.page_size, by, sinks)
    # Beside the output's rounding: a score is a sum of D products in fp32 and its exponential is off by 2^-22 of itself, a
    # weight by 2^-16 (bf16; less otherwise), the sums by 2^-24 for each term, as decode_attention's.
    n = float(prefix_lens.max() + (lens.max() if lens.numel() else 0))
    err = (out.double() - want).abs()
    bad = err > 2.0 ** -8 * want.abs() + 2.0 ** -10 * mag + n * 2.0 ** -25 * v.abs().max()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {err.max().item()}"
    smax = (q.double().norm(dim=-1).max() * k.norm(dim=-1).max() * abs(by)).item()
    both = torch.isfinite(wlse)
    assert torch.equal(torch.isfinite(lse), both)
    assert (lse.double() - wlse)[both].abs().max().item() <= 2.0 ** -18 * (1 + smax) if both.any() else True
    assert torch.equal(out, dec.shared_prefix_attention(*args, scale=scale, sinks=sinks)), "not the same twice"
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shared,mine", [([1], [0]), ([64], [1, 0]), ([128], [5] * 2), ([127], [0, 3, 16]), ([129], [40] * 5), ([1000], [0] * 4), ([4097], [33, 0, 2])])
def test_one_prefix(dec, cuda, fp4, kind, d, shared, mine):
    check(dec, *case(dec, cuda, kind, d, 8, 2, 16, shared, mine))
    assert fp4.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,hq,hk", [(64, 64, 8), (64, 5, 1), (128, 32, 8), (128, 16, 16), (256, 20, 4), (64, 48, 1), (256, 3, 3)])
@pytest.mark.parametrize("each", [1, 3, 16, 37])
def test_rows_of_every_number(dec, cuda, fp4, kind, d, hq, hk, each):
    # rows of a key head: below, at and beyond one tile of 128
    mine = [(i * 37) % 90 for i in range(each)]
    check(dec, *case(dec, cuda, kind, d, hq, hk, 32, [700], mine, seed=each))
    assert fp4.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 2, 8, 16, 64, 256, 1024])
def test_pages_of_every_size(dec, cuda, fp4, kind, d, page):
    check(dec, *case(dec, cuda, kind, d, 8, 4, page, [1500, 333], [20, 0, 300, 7], seed=page))
    assert fp4.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shared", [[0], [0, 0, 0], [300, 0, 1], [1, 2, 3, 64, 65, 128, 129, 1000], [0, 20000, 0, 0, 31, 0], [5] * 40])
def test_prefixes_of_uneven_lengths(dec, cuda, fp4, kind, d, shared):
    for each in (1, 2):
        mine = [(i * 53) % 70 if i % 3 else 0 for i in range(each * len(shared))]
        check(dec, *case(dec, cuda, kind, d, 6, 2, 16, shared, mine, seed=len(shared)))
    assert fp4.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_more_prefixes_than_a_warp_and_units_than_ctas(dec, cuda, fp4, kind):
    shared = [(i * 97) % 400 for i in range(75)]
    check(dec, *case(dec, cuda, kind, 64, 8, 4, 16, shared, [i % 20 for i in range(150)]))
    assert fp4.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_sinks_scale_and_nothing_at_all(dec, cuda, fp4, kind, d):
    args = case(dec, cuda, kind, d, 8, 2, 16, [260, 0], [12, 0, 0, 40])
    sinks = torch.randn(8, device=cuda) * 3
    check(dec, *args, sinks=sinks)
    check(dec, *args, sinks=sinks, scale=0.3)
    check(dec, *args, scale=-0.05)
    check(dec, *args, scale=0.0)
    out, lse = dec.shared_prefix_attention(*args, return_lse=True)
    assert (out[2] == 0).all() and (lse[2] == -math.inf).all()  # neither prefix nor own keys
    assert fp4.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_same_as_over_whole_tables(dec, cuda, kind, d):
    # the prefix's pages before each sequence's own (the prefix ends with its page): decode_attention sees the same keys
    q, cache, pt, pl, table, lens = case(dec, cuda, kind, d, 8, 2, 16, [320, 64], [30, 0, 111, 5])
    out, lse = dec.shared_prefix_attention(q, cache, pt, pl, table, lens, return_lse=True)
    whole = [torch.cat((pt[i // 2][: int(pl[i // 2]) // 16], table[i])) for i in range(4)]
    width = max(len(w) for w in whole)
    whole = torch.stack([torch.nn.functional.pad(w, (0, width - len(w)), value=-1) for w in whole])
    want, wlse = dec.decode_attention(q, cache, whole, lens + pl.repeat_interleave(2), return_lse=True)
    k, v = (R.cache_values(p, s, kind) for p, s in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)))
    assert ((out.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 2.0 ** -10 * v.abs().max()).all()
    assert ((lse - wlse).abs() <= 2.0 ** -16 * (1 + wlse.abs())).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_values_that_nearly_cancel(dec, cuda, kind, d):
    # as test_attention_of_values_that_nearly_cancel: +-t in turn under scores within 2^-6 of each other; the output shows how
    # many bits the weights hold (22 for fp8 and nvfp4, 16 for bf16), scores, exponentials and joining 64 terms of 2^-24
    n, hk, hq, page = 96, 2, 8, 16
    g = torch.Generator().manual_seed(d)
    cache = dec.PagedKVCache(n // page, page, hk, d, kind, device=cuda)
    k = torch.randn(n, hk, d, generator=g)
    v = torch.tensor([1.0, -1.0]).repeat(n // 2).reshape(-1, 1, 1) * (torch.randint(0, 2, (hk, d), generator=g) * 2.0 - 1.0)
    cache.append(k.to(torch.bfloat16).to(cuda), v.to(torch.bfloat16).to(cuda), torch.arange(n, device=cuda))
    q = torch.randn(3, hq, d, generator=g).to(torch.bfloat16).to(cuda)
    pages = torch.arange(n // page, dtype=torch.int32, device=cuda)
    args = (q, cache, pages[None, :4], torch.tensor([64], dtype=torch.int32, device=cuda), pages[None, 4:].expand(3, 2),
            torch.tensor([0, 2, 30], dtype=torch.int32, device=cuda))
    scale = 2.0 ** -8 * d ** -0.5
    out = dec.shared_prefix_attention(*args, scale=scale)
    rows = [R.cache_values(p, s, kind) for p, s in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales))]
    want, _, mag = S.attention(q, *rows, *args[2:], page, scale, None)
    err = (out.double() - want).abs()
    bad = err > 2.0 ** -8 * want.abs() + (160 * 2.0 ** -24 + (2.0 ** -16 if kind == "bf16" else 0.0)) * mag
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {(err / mag)[bad].max().item()} of the terms"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rising", [True, False])
def test_scores_that_rise_and_fall(dec, cuda, fp4, kind, d, rising):
    # the reference moves in many tiles (or in the first alone): sums and outputs are scaled on the way
    n, page = 1500, 16
    g = torch.Generator().manual_seed(d)
    cache = dec.PagedKVCache(-(-n // page) + 3, page, 2, d, kind, device=cuda)
    at = torch.arange(cache.num_pages * page)
    size = (at.float() / n * 4).reshape(-1, 1, 1)
    size = size if rising else size.flip(0)
    k = torch.ones(len(at), 2, d) * size + 0.1 * torch.randn(len(at), 2, d, generator=g)
    v = torch.randn(len(at), 2, d, generator=g) * torch.exp2(4 * torch.randn(len(at), 1, 1, generator=g))
    cache.append(k.to(torch.bfloat16).to(cuda), v.to(torch.bfloat16).to(cuda), at.to(cuda))
    q = (torch.randn(5, 8, d, generator=g) + torch.tensor([3.0, -3.0, 0.0, 1.0, -1.0]).reshape(5, 1, 1)).to(torch.bfloat16).to(cuda)
    pages = torch.arange(cache.num_pages, dtype=torch.int32, device=cuda)
    table = pages[None, -3:].expand(5, 3)
    check(dec, q, cache, pages[None], torch.tensor([n], dtype=torch.int32, device=cuda), table, torch.tensor([0, 40, 17, 48, 1], dtype=torch.int32, device=cuda))
    assert fp4.device_error() == 0


def test_bad_pages_and_lengths(dec, cuda, fp4):
    for kind in KINDS:
        q, cache, pt, pl, table, lens = case(dec, cuda, kind, 64, 8, 2, 16, [500, 130], [30, 0, 111, 5])
        bad = pt.clone()
        bad[0, 3], bad[0, 20], bad[1, 0] = -1, cache.num_pages, 1 << 30
        check(dec, q, cache, bad, pl, table, lens)
        assert fp4.device_error() == 13
        own = table.clone()
        own[2, 1] = -5
        check(dec, q, cache, pt, pl, own, lens)
        assert fp4.device_error() == 13
        want = dec.shared_prefix_attention(q, cache, pt[:, :5], torch.tensor([80, 80], dtype=torch.int32, device=cuda), table, lens)
        assert fp4.device_error() == 0
        assert torch.equal(dec.shared_prefix_attention(q, cache, pt[:, :5], torch.tensor([81, 1 << 30], dtype=torch.int32, device=cuda), table, lens), want)
        assert fp4.device_error() == 13
        none = dec.shared_prefix_attention(q, cache, pt, torch.tensor([-1, -500], dtype=torch.int32, device=cuda), table, lens)
        assert fp4.device_error() == 13
        assert torch.equal(none, dec.shared_prefix_attention(q, cache, pt[:, :0], torch.zeros(2, dtype=torch.int32, device=cuda), table, lens))
        assert fp4.device_error() == 0
        assert torch.equal(none, dec.decode_attention(q, cache, table, lens))
        no_own = torch.zeros(4, dtype=torch.int32, device=cuda)
        assert torch.equal(dec.shared_prefix_attention(q, cache, pt, pl, table[:, :0], no_own), dec.shared_prefix_attention(q, cache, pt, pl, table, no_own))
        assert fp4.device_error() == 0


def test_tensors_of_any_strides(dec, cuda):
    q, cache, pt, pl, table, lens = case(dec, cuda, "nvfp4", 64, 8, 2, 16, [500, 130], [30, 0, 111, 5])
    want = dec.shared_prefix_attention(q, cache, pt, pl, table, lens)
    wide = torch.zeros(4, 12, 64, dtype=torch.bfloat16, device=cuda)
    wide[:, 2:10] = q
    tables = torch.zeros(2, pt.shape[1] + 3, dtype=torch.int32, device=cuda)
    tables[:, 1: 1 + pt.shape[1]] = pt
    assert torch.equal(dec.shared_prefix_attention(wide[:, 2:10], cache, tables[:, 1: 1 + pt.shape[1]], pl.repeat_interleave(2)[::2], table.t().contiguous().t(), lens), want)
    assert torch.equal(dec.shared_prefix_attention(q.float(), cache, pt, pl, table, lens), want)
    one = dec.shared_prefix_attention(q, cache, pt[:1].expand(2, -1), pl[:1].expand(2), table, lens)
    assert torch.equal(one, dec.shared_prefix_attention(q, cache, pt[:1].repeat(2, 1), pl[:1].repeat(2), table, lens))


@pytest.mark.parametrize("kind", KINDS)
def test_captured_beside_other_calls(dec, cuda, kind):
    a = case(dec, cuda, kind, 64, 64, 8, 64, [3000], [100] * 8, seed=1)
    b = case(dec, cuda, kind, 128, 16, 4, 16, [700, 0, 90], [10, 50, 0, 3, 200, 64], seed=2)
    wants = [dec.shared_prefix_attention(*x) for x in (a, b)]
    graphs, outs = [], []
    for x in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(dec.shared_prefix_attention(*x))
        graphs.append(graph)
    sides = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for graph, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                graph.replay()
        with torch.cuda.stream(sides[2]):
            third = dec.shared_prefix_attention(*a)
        fourth = dec.shared_prefix_attention(*b)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1], wants[1]) and torch.equal(third, wants[0]) and torch.equal(fourth, wants[1])
    # lengths change between replays, as they do in a decoding loop
    a[3].fill_(2900), a[5].fill_(90)
    graphs[0].replay()
    assert torch.equal(outs[0], dec.shared_prefix_attention(*a))


def test_other_calls_on_the_same_workspace(dec, cuda):
    a = case(dec, cuda, "fp8", 64, 8, 2, 16, [900], [300] * 4, seed=3)
    want, plain = dec.shared_prefix_attention(*a), dec.decode_attention(a[0], a[1], a[4], a[5])
    for _ in range(3):
        assert torch.equal(dec.decode_attention(a[0], a[1], a[4], a[5]), plain)
        assert torch.equal(dec.shared_prefix_attention(*a), want)


def test_nothing_to_do_and_refusals(dec, cuda):
    q, cache, pt, pl, table, lens = case(dec, cuda, "bf16", 64, 8, 2, 16, [50, 60], [3, 0, 1, 2])
    good = dict(q=q, cache=cache, prefix_table=pt, prefix_lens=pl, page_table=table, seq_lens=lens)
    assert dec.shared_prefix_attention(q[:0], cache, pt, pl, table[:0], lens[:0]).shape == (0, 8, 64)
    for bad in (dict(q=q[:3], page_table=table[:3], seq_lens=lens[:3]), dict(prefix_lens=pl[:0], prefix_table=pt[:0]), dict(prefix_lens=pl.long()),
                dict(prefix_lens=pl.cpu()), dict(prefix_table=pt[:1]), dict(prefix_table=pt.long()), dict(prefix_table=pt[0]), dict(page_table=table[:2]),
                dict(seq_lens=lens.long()), dict(q=q[:, :7]), dict(q=q[..., :32]), dict(sinks=torch.zeros(3, device=cuda)), dict(prefix_lens=pl.reshape(2, 1))):
        with pytest.raises(ValueError):
            dec.shared_prefix_attention(**{**good, **bad})
    with pytest.raises(RuntimeError):
        dec.shared_prefix_attention(**good, scale=math.nan)
