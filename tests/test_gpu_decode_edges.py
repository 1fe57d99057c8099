"""The decode-side operators on a B200 where they can go wrong unseen: slices that just fit, tensors that share or skew their
memory, weights that nearly cancel.  Against the 64-bit restatements of tests/decode_reference.py, with the tolerances of
tests/test_gpu_decode.py or ones derived beside the test."""
import pytest
import torch

from tests import decode_reference as R
from tests.test_gpu_decode import KINDS, attention_case, close, heads, raw, stored, weight_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec(cuda):
    import fp4_decode
    return fp4_decode


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(8, 2), (16, 1)])
def test_attention_of_values_that_nearly_cancel(dec, cuda, kind, d, hq, hk):
    # Values of +-t in turn under scores within about 2^-6 of each other: the output is a sum of differences of nearly equal
    # weights, and shows how many bits those hold.  Beside its rounding to BF16 it may be off by 2^-24 of sum(p |v|) for each
    # of the n terms of the sums in fp32 and 64 times that for the rest: the scores (D * 2^-24 of sum |q k| scale < 2^-4, and
    # their factors), the exponential (2^-22), the weights (22 bits for fp8 and nvfp4; 16 for bf16, that is 2^-16 more),
    # value scales, joining and division.
    lens, page = [2, 16, 34, 60], 16
    g = torch.Generator().manual_seed(d + hq)
    n = 64
    cache = dec.PagedKVCache(len(lens) * n // page, page, hk, d, kind, device=cuda)
    k = torch.randn(len(lens) * n, hk, d, generator=g)
    sign = torch.tensor([1.0, -1.0]).repeat(len(lens) * n // 2).reshape(-1, 1, 1)
    v = sign * (torch.randint(0, 2, (hk, d), generator=g) * 2.0 - 1.0)
    cache.append(k.to(torch.bfloat16).to(cuda), v.to(torch.bfloat16).to(cuda), torch.arange(len(lens) * n, device=cuda))
    q = torch.randn(len(lens), hq, d, generator=g).to(torch.bfloat16).to(cuda)
    table = torch.arange(len(lens) * n // page, dtype=torch.int32, device=cuda).reshape(len(lens), -1)
    seq = torch.tensor(lens, dtype=torch.int32, device=cuda)
    scale = 2.0 ** -8 * d ** -0.5
    out = dec.decode_attention(q, cache, table, seq, scale=scale)
    rows = [R.cache_values(p, s, kind) for p, s in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales))]
    want, _, mag = R.attention(q, *rows, table, seq, page, scale, 0, None)
    terms = (seq.double().reshape(-1, 1, 1) + 64) * 2.0 ** -24 + (2.0 ** -16 if kind == "bf16" else 0.0)
    err = (out.double() - want).abs()
    bad = err > 2.0 ** -8 * want.abs() + terms * mag
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {(err / mag)[bad].max().item()} of the terms"


@pytest.mark.parametrize("m,n,k", [(3, 20480, 32768), (5, 12800, 32768), (6, 19072, 16384), (7, 28672, 9344), (9, 15360, 14464), (9, 16384, 14400),
                                   (10, 14336, 16384), (12, 12288, 16384), (13, 12416, 12288), (13, 14336, 12288), (14, 10240, 16384),
                                   (11, 15360, 11904), (25, 12288, 16384)])
def test_gemv_where_a_slice_only_just_fits(cuda, fp4, m, n, k):
    # rows whose bytes a step do not divide what a CTA holds of x: the longest slice has to fit, its last row to its end
    g = torch.Generator(cuda).manual_seed(m + k)
    w = torch.randn(n, k, generator=g, device=cuda, dtype=torch.bfloat16) * 0.02
    x = torch.randn(m, k, generator=g, device=cuda, dtype=torch.bfloat16)
    cache = fp4.FP4WeightCache(w, global_scale=True)
    del w
    y = fp4.fp4_cached_gemv(x, cache)
    assert torch.equal(y, fp4.fp4_cached_gemv(x, cache)), "not the same twice"
    wv = weight_values(cache)
    close(y, x.double() @ wv.T, x.double().abs() @ wv.abs_().T, 64, f"gemv {m}x{n}x{k}")
    cache.free()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_over_page_tables_of_any_strides(dec, cuda, fp4, kind):
    # one prefix for all sequences (rows shared by expand), rows that overlap, a column, a turned table
    q, cache, _, _ = attention_case(dec, cuda, kind, 64, 8, 2, 16, [300] * 5, seed=3)
    flat = torch.randperm(cache.num_pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).to(cuda)
    lens = torch.tensor([100, 3, 0, 112, 57], dtype=torch.int32, device=cuda)
    forms = [flat[:7].view(1, 7).expand(5, 7), flat[:1].view(1, 1).expand(5, 7), flat.as_strided((5, 7), (3, 1)), flat[:70].view(7, 10)[:, :5].t(),
             flat[:70].view(5, 14)[:, ::2], flat[:70].view(10, 7)[::2]]
    for table in forms:
        want = dec.decode_attention(q, cache, table.clone(memory_format=torch.contiguous_format), lens)
        assert torch.equal(dec.decode_attention(q, cache, table, lens), want)
    short = torch.clamp(lens, max=16)
    for table in (flat[:50].view(5, 10)[:, 4:5], flat[:1].view(1, 1).expand(5, 1)):
        want = dec.decode_attention(q, cache, table.clone(memory_format=torch.contiguous_format), short)
        assert torch.equal(dec.decode_attention(q, cache, table, short), want)
    one = flat[:21].view(7, 3).t()[1:2]
    assert torch.equal(dec.decode_attention(q[:1], cache, one, lens[:1]), dec.decode_attention(q[:1], cache, one.clone(memory_format=torch.contiguous_format), lens[:1]))
    assert fp4.device_error() == 0


def skewed(x):
    """Views of x's values that torch calls contiguous (or nearly) and whose rows start anywhere."""
    t, h, d = x.shape
    for at in (1, 2, 3, 5):
        flat = torch.empty(x.numel() + at, dtype=x.dtype, device=x.device)
        flat[at:] = x.reshape(-1)
        yield flat[at:].view(t, h, d)
    padded = torch.empty(t, h, d + 5, dtype=x.dtype, device=x.device)
    for at in (0, 4, 5):
        padded[..., at: at + d] = x
        yield padded[..., at: at + d]


@pytest.mark.parametrize("t,hq", [(1, 1), (1, 4), (3, 1), (5, 2)])
def test_rows_that_start_anywhere(dec, cuda, t, hq):
    q, k, v, (wq, wk), pos = (x.contiguous() if isinstance(x, torch.Tensor) else x for x in heads(t, hq, 1, 64, t, cuda))
    table = dec.rope_table(500, 64, device=cuda)
    slots = torch.arange(t, device=cuda) + 3
    want = dec.qk_norm_rope(q, k, pos, table, wq, wk)
    for kind in KINDS:
        ref = dec.PagedKVCache(2, 16, 1, 64, kind, device=cuda)
        ref.append(k, v, slots)
        pages, lens = torch.zeros(t, 1, dtype=torch.int32, device=cuda), torch.full((t,), 3 + t, dtype=torch.int32, device=cuda)
        seen = dec.decode_attention(q, ref, pages, lens)
        for a, b, c in zip(skewed(q), skewed(k), skewed(v)):
            assert all(torch.equal(x, y) for x, y in zip(dec.qk_norm_rope(a, b, pos, table, wq, wk), want))
            cache = dec.PagedKVCache(2, 16, 1, 64, kind, device=cuda)
            cache.append(b, c, slots)
            assert torch.equal(raw(cache.k_pages), raw(ref.k_pages)) and torch.equal(raw(cache.v_pages), raw(ref.v_pages))
            assert torch.equal(cache.append_qkv(a, b, c, pos, slots, table, wq, wk), want[0])
            assert torch.equal(dec.decode_attention(a, ref, pages, lens), seen)


@pytest.mark.parametrize("m,n,k", [(70000, 200, 256), (70001, 120, 4100), (1000, 16384, 16384), (300, 16384, 2880)])
def test_gemv_of_more_rows_than_a_launch(cuda, fp4, m, n, k):
    # a row's result does not depend on the rows beside it (from a tile of 16 on): many at once equal 160 at a time
    g = torch.Generator(cuda).manual_seed(m)
    cache = fp4.FP4WeightCache(torch.randn(n, k, generator=g, device=cuda, dtype=torch.bfloat16) * 0.02, global_scale=True)
    wide = torch.randn(m, k + 8, generator=g, device=cuda, dtype=torch.bfloat16)
    x = wide[:, :k]
    y = fp4.fp4_cached_gemv(x, cache)
    for at in [*range(0, m, max(160, m // 8000 * 800)), m - 16, 65440, 65520]:
        if 0 <= at < m:
            part = x[at: at + 160] if m - at >= 16 else x[m - 16:]
            want = fp4.fp4_cached_gemv(part, cache)
            assert torch.equal(y[at: at + len(part)], want[-len(y[at: at + len(part)]):]), at
    cache.free()


def nvfp4_of_fp32(y):
    """(codes, scale bytes) of fp32 rows y [..., D] by the codec's definition: the oracle's scale of absmax / 6, then the
    nearest of the levels of y / scale, the lower one at a midpoint."""
    from oracle import nvfp4_oracle as O
    lib = O.lib()
    b = y.reshape(-1, 16)
    sixth = b.abs().amax(-1) / torch.full((b.shape[0],), 6.0)
    bytes_ = torch.tensor([lib.oracle_ue4m3_encode(max(s, 2.0 ** -9)) for s in sixth.tolist()], dtype=torch.uint8)
    x = b * (torch.ones(b.shape[0]) / torch.tensor([lib.oracle_ue4m3_decode(c) for c in bytes_.tolist()])).unsqueeze(-1)
    code = torch.bucketize(x.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])).to(torch.uint8) | ((x < 0).to(torch.uint8) << 3)
    code = code.reshape(y.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), bytes_.reshape(*y.shape[:-1], -1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("part,interleaved", [(1, False), (2, False), (1, True)])
def test_append_qkv_stores_fp32_keys_to_the_byte(dec, cuda, kind, d, part, interleaved):
    # A table of factors c with sines of zero makes each key x * c rounded to fp32, nothing else, and so known to the bit: with
    # c at, just below and just above every absmax where a scale changes (6 times the midpoints of the scales, the powers of
    # two of the subnormal ones), and anywhere between.  What the cache holds has to be its format's of that number.
    g = torch.Generator().manual_seed(d)
    levels = torch.tensor(R.UE4M3[1:128], dtype=torch.float64)
    edges = torch.cat((levels, (levels[1:] + levels[:-1]) / 2)) * 6.0
    edges = edges.float()
    up, down = torch.full_like(edges, float("inf")), torch.zeros_like(edges)
    c = torch.cat((edges, torch.nextafter(edges, up), torch.nextafter(edges, down), torch.exp2(torch.rand(300, generator=g) * 46 - 18)))
    t, h, rot = len(c), 2, d // part
    table = torch.cat((c.unsqueeze(1).expand(t, rot // 2), torch.zeros(t, rot // 2)), dim=1).contiguous()
    k = (torch.rand(t, h, d, generator=g) * 2 - 1).to(torch.bfloat16)
    k[..., torch.arange(0, d, 16) + torch.randint(0, 16, (d // 16,), generator=g)] = 1.0  # each block's largest
    k[:, 1] = -k[:, 1]
    y = k.float().clone()
    y[..., :rot] *= c.reshape(-1, 1, 1)
    q, v = (torch.randn(t, n, d, generator=g).to(torch.bfloat16) for n in (1, h))
    cache = dec.PagedKVCache(-(-t // 16), 16, h, d, kind, device=cuda)
    slots = torch.randperm(cache.num_pages * 16, generator=g)[:t]
    cache.append_qkv(q.to(cuda), k.to(cuda), v.to(cuda), torch.arange(t, device=cuda), slots.to(cuda), table.to(cuda), interleaved=interleaved)
    for got, scales, want in ((cache.k_pages, cache.k_scales, nvfp4_of_fp32(y) if kind == "nvfp4" else stored(y, kind)),
                              (cache.v_pages, cache.v_scales, stored(v, kind))):
        assert torch.equal(raw(got).cpu()[slots // 16, :, slots % 16], raw(want[0]))
        if scales is not None:
            assert torch.equal(scales.cpu()[slots // 16, :, slots % 16], want[1])


def test_cleanup_frees_the_attention_workspaces(dec, cuda, fp4):
    case = attention_case(dec, cuda, "nvfp4", 64, 8, 2, 16, [600, 50], seed=6)
    want = dec.decode_attention(*case)
    assert any(key[0] == cuda.index for key in dec._WORKSPACES)
    fp4.cleanup()
    assert not any(key[0] == cuda.index for key in dec._WORKSPACES)
    assert torch.equal(dec.decode_attention(*case), want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("factor", [-(2.0 ** 80), -(2.0 ** 100), -(2.0 ** 116), 2.0 ** 116])
def test_attention_of_scores_of_any_size(dec, cuda, kind, factor):
    # Scores all of one sign and of any finite size, further apart than fp32 can blur: each head sees its largest alone.
    n, d = 90, 64
    cache = dec.PagedKVCache(6, 16, 1, d, kind, device=cuda)
    g = torch.Generator().manual_seed(3)
    order = torch.randperm(n, generator=g)
    k = torch.exp2(order.float() / n * 5).reshape(n, 1, 1).expand(n, 1, d)  # each row its one number, apart by 4 %
    k = k * torch.where(torch.arange(d) < 16, 1.0, 2.0 ** -6)  # (its first block, in nvfp4 a few of them alike)
    v = torch.randn(n, 1, d, generator=g)
    cache.append(k.to(torch.bfloat16).to(cuda), v.to(torch.bfloat16).to(cuda), torch.arange(n, device=cuda))
    q = torch.full((1, 4, d), factor).to(torch.bfloat16).to(cuda)
    table, lens = torch.arange(6, dtype=torch.int32, device=cuda).reshape(1, 6), torch.tensor([n], dtype=torch.int32, device=cuda)
    out, lse = dec.decode_attention(q, cache, table, lens, return_lse=True)
    keys, values = (R.cache_values(p, s, kind).permute(0, 2, 1, 3).reshape(-1, d)[:n] for p, s in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)))
    s = keys.sum(-1) * q[0, 0, 0].double() * d ** -0.5
    top = s == s.max()
    want = values[top].mean(0)
    assert torch.isfinite(lse).all() and ((lse.double() - s.max()).abs() <= 2.0 ** -18 * s.abs().max()).all()
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * values[top].abs().mean(0)).all()
