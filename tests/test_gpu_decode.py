"""The decode-side operators on a B200 against 64-bit restatements of their formulas (tests/decode_reference.py).

Tolerances, from the arithmetic: a result rounded once to BF16 is off by at most 2^-9 of itself (2^-8 is allowed: the
64-bit value may lie just across a rounding boundary from the fp32 one), below the normal numbers by half of their
spacing 2^-133; fp32 sums of n terms by n * 2^-24 of the terms'
magnitudes (2^-22 * n allowed with the products' and factors' own roundings); attention weights are held in 11 bits or
more next to fp32 sums, so its results may be off by 2^-10 of sum(p |v|), and by 2^-25 for each key too small for that."""
import math

import pytest
import torch

from tests import decode_reference as R
from tests import workloads as W

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec(cuda):
    import fp4_decode
    return fp4_decode


def close(got, want, terms, n, what):
    """|got - want| <= 2^-8 |want| + 2^-133 + n 2^-22 terms, non-finite places alike."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    err = (got - want).abs()
    bad = (err > 2.0 ** -8 * want.abs() + 2.0 ** -133 + n * 2.0 ** -22 * terms) & torch.isfinite(want)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {err[bad].max().item()}"


# ------------------------------------------------------------------------------------------------------ matrix-vector

def weight_values(cache):
    """The cached weight [N, K] in 64 bits."""
    sd = cache.state_dict()
    n, k = cache.N, cache.K
    vals = R.e2m1_values(sd["fp4"]).reshape(n, k // 16, 16)
    atoms = R.ue4m3_values(sd["sf"]).reshape(n // 128, k // 64, 32, 4, 4)
    scales = atoms.permute(0, 3, 2, 1, 4).reshape(n, k // 16)
    return (vals * scales.unsqueeze(-1)).reshape(n, k)[: cache.N_orig, : cache.K_orig] / cache.global_scale


def gemv_check(cuda, fp4, m, n, k, bias=True, global_scale=False, x=None):
    x0, w, b = W.cached_linear_inputs(m, n, k, seed=m + n + k)
    cache = fp4.FP4WeightCache(w.to(cuda), b.to(cuda) if bias else None, global_scale=global_scale)
    x = x0.to(cuda) if x is None else x
    y = fp4.fp4_cached_gemv(x, cache)
    wv = weight_values(cache)
    want = x.double() @ wv.T
    terms = x.double().abs() @ wv.abs().T
    if bias:
        want, terms = want + b.to(cuda).double(), terms + b.to(cuda).double().abs()
    assert y.dtype == torch.bfloat16 and y.shape == (m, n)
    # a chain of sums in fp32 is at most K long; partial sums over lanes and blocks make it a root of that or so
    close(y, want, terms, min(k, 64), f"gemv {m}x{n}x{k}")
    cache.free()


@pytest.mark.parametrize("m", [1, 2, 3, 7, 8, 9, 15, 16, 17, 33])
def test_gemv_rows(cuda, fp4, m):
    gemv_check(cuda, fp4, m, 200, 400)


@pytest.mark.parametrize("n,k", [(1, 1), (1, 16), (7, 15), (8, 17), (31, 127), (32, 128), (33, 129), (127, 64), (128, 1000),
                                 (129, 2880), (2880, 2880), (1000, 4097), (96, 16384)])
@pytest.mark.parametrize("m", [1, 5, 16])
def test_gemv_sizes(cuda, fp4, m, n, k):
    gemv_check(cuda, fp4, m, n, k, bias=(n + k) % 2 == 0, global_scale=n % 2 == 1)


@pytest.mark.parametrize("m,k", [(1, 20000), (16, 9000), (12, 16400), (40, 5000)])
def test_gemv_long_rows(cuda, fp4, m, k):
    gemv_check(cuda, fp4, m, 300, k)


@pytest.mark.parametrize("m,n,k", [(16, 7200, 16384), (11, 9700, 15999), (5, 19000, 16000), (17, 7300, 16384)])
def test_gemv_many_rows_of_a_long_k(cuda, fp4, m, n, k):
    g = torch.Generator(cuda).manual_seed(m)
    w = torch.randn(n, k, generator=g, device=cuda, dtype=torch.bfloat16) * 0.02
    x = torch.randn(m, k, generator=g, device=cuda, dtype=torch.bfloat16)
    bias = torch.randn(n, generator=g, device=cuda, dtype=torch.bfloat16)
    cache = fp4.FP4WeightCache(w, bias, global_scale=True)
    y = fp4.fp4_cached_gemv(x, cache)
    assert torch.equal(y, fp4.fp4_cached_gemv(x, cache)), "not the same twice"
    del w
    wv = weight_values(cache)
    want, terms = x.double() @ wv.T + bias.double(), x.double().abs() @ wv.abs_().T + bias.double().abs()
    close(y, want, terms, 64, f"gemv {m}x{n}x{k}")
    cache.free()


@pytest.mark.parametrize("m,n,k", [(1, 28500, 2050), (5, 28500, 2051), (8, 28416, 2100), (2, 14400, 4200), (16, 15360, 2880), (20, 7000, 6000)])
def test_gemv_many_rows(cuda, fp4, m, n, k):
    gemv_check(cuda, fp4, m, n, k, bias=k % 2 == 0)


def test_gemv_strided_batched_and_cast_rows(cuda, fp4):
    m, n, k = 6, 384, 650
    x, w, _ = W.cached_linear_inputs(m, n, k, seed=3, bias=False)
    cache = fp4.FP4WeightCache(w.to(cuda))
    want = fp4.fp4_cached_gemv(x.to(cuda), cache)
    wide = torch.full((m, 1001), float("nan"), dtype=torch.bfloat16, device=cuda)
    for at in (0, 1, 3, 8):  # every alignment of a row
        wide[:, at: at + k] = x.to(cuda)
        assert torch.equal(fp4.fp4_cached_gemv(wide[:, at: at + k], cache), want)
    assert torch.equal(fp4.fp4_cached_gemv(x.to(cuda).reshape(2, 3, k), cache), want.reshape(2, 3, n))
    assert torch.equal(fp4.fp4_cached_gemv(x.to(cuda).t().contiguous().t(), cache), want)
    assert torch.equal(fp4.fp4_cached_gemv(x.to(cuda).float(), cache), want)
    assert torch.equal(fp4.fp4_cached_gemv(x.to(cuda)[0], cache), want[0])
    assert fp4.fp4_cached_gemv(x.to(cuda)[:0], cache).shape == (0, n)
    cache.free()


def test_gemv_shard_and_fp32_bias(cuda, fp4):
    m, n, k = 4, 512, 384
    x, w, b = W.cached_linear_inputs(m, n, k, seed=8)
    x = x.to(cuda)
    cache = fp4.FP4WeightCache(w.to(cuda))
    whole = fp4.fp4_cached_gemv(x, cache)
    part = fp4.fp4_cached_gemv(x, cache.shard(128, 256))
    assert torch.equal(part, whole[:, 128:384])
    other = fp4.FP4WeightCache(w.to(cuda), b.to(cuda).float())
    y = fp4.fp4_cached_gemv(x, other)
    assert y.dtype == torch.float32 and torch.equal(y, whole + b.to(cuda).float())


@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -60, 1e-3, 1e4, 2.0 ** 100])
def test_gemv_magnitudes(cuda, fp4, scale):
    # activations of any size, one row far from the next: each row keeps its own precision
    m, n, k = 3, 160, 512
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(1)).to(cuda)
    x[1] *= scale
    x[2, 5:] *= 2.0 ** -20
    gemv_check(cuda, fp4, m, n, k, bias=False, x=x.to(torch.bfloat16))


def test_gemv_non_finite_activations_stay_in_their_row(cuda, fp4):
    m, n, k = 4, 256, 512
    x, w, _ = W.cached_linear_inputs(m, n, k, seed=2, bias=False)
    x = x.to(cuda)
    cache = fp4.FP4WeightCache(w.to(cuda))
    good = fp4.fp4_cached_gemv(x, cache)
    x[1, 7], x[2, 300] = float("nan"), float("inf")
    y = fp4.fp4_cached_gemv(x, cache)
    assert torch.equal(y[[0, 3]], good[[0, 3]])
    assert torch.isnan(y[1]).all()
    wv = weight_values(cache)[:, 300]
    assert torch.isnan(y[2][wv == 0]).all() and torch.isinf(y[2][wv != 0]).all()


def test_gemv_refusals(cuda, fp4):
    _, w, b = W.cached_linear_inputs(1, 128, 128, seed=0)
    cache = fp4.FP4WeightCache(w.to(cuda), b[:100].to(cuda))
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="doesn't match weight K"):
        fp4.fp4_cached_gemv(x[:, :64], cache)
    with pytest.raises(ValueError, match="bias has 100"):
        fp4.fp4_cached_gemv(x, cache)
    with pytest.raises(AssertionError, match="CUDA device"):
        fp4.fp4_cached_gemv(x.cpu(), cache)
    cache.free()
    with pytest.raises(RuntimeError, match="freed"):
        fp4.fp4_cached_gemv(x, cache)


# ------------------------------------------------------------------------------------------------------ norm + rotation

def heads(t, hq, hk, d, seed, cuda, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(t, (hq + 2 * hk) * d, generator=g) * spread).to(torch.bfloat16).to(cuda)
    q, k, v = qkv.split([hq * d, hk * d, hk * d], dim=1)
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(torch.bfloat16).to(cuda) for _ in range(2)]
    pos = torch.randint(0, 500, (t,), generator=g).to(cuda)
    return q.unflatten(1, (hq, d)), k.unflatten(1, (hk, d)), v.unflatten(1, (hk, d)), w, pos


@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("t,hq,hk", [(1, 1, 1), (1, 64, 8), (5, 3, 1), (67, 8, 2)])
def test_norm_rope_sizes(dec, cuda, d, t, hq, hk):
    q, k, _, (wq, wk), pos = heads(t, hq, hk, d, d + t, cuda)
    for rot in sorted({d, d // 2, 8, 24}):
        for interleaved in (False, True):
            for norm in (True, False):
                table = dec.rope_table(500, rot, device=cuda)
                got = dec.qk_norm_rope(q, k, pos, table, wq if norm else None, wk if norm else None, interleaved=interleaved)
                for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
                    want = R.norm_rope(x, w if norm else None, pos, table, 1e-6, interleaved)
                    terms = R.norm_rope(x, w if norm else None, pos, None, 1e-6, interleaved).abs().amax(-1, keepdim=True)
                    close(y, want, terms, 4, f"d {d} rot {rot} interleaved {interleaved} norm {norm}")


def test_norm_rope_layouts_types_and_none(dec, cuda):
    q, k, _, (wq, wk), pos = heads(9, 4, 2, 64, 1, cuda)
    table = dec.rope_table(500, 64, device=cuda)
    want = dec.qk_norm_rope(q, k, pos, table, wq, wk)
    for a in (lambda x: x.contiguous(), lambda x: x.transpose(0, 1).contiguous().transpose(0, 1), lambda x: x.float(),
              lambda x: torch.nn.functional.pad(x, (3, 2))[..., 3:-2]):
        got = dec.qk_norm_rope(a(q), a(k), pos.to(torch.int32), table, wq.float(), wk)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    plain = dec.qk_norm_rope(q, k, None, None)
    assert torch.equal(plain[0], q) and torch.equal(plain[1], k)
    none = dec.qk_norm_rope(q[:0], k[:0], pos[:0], table, wq, wk)
    assert none[0].shape == (0, 4, 64)
    only = dec.qk_norm_rope(q, k, pos, table, wq, None)
    assert torch.equal(only[0], want[0]) and not torch.equal(only[1], want[1])


def test_norm_rope_zero_rows_and_non_finite(dec, cuda):
    q, k, _, (wq, wk), pos = heads(6, 4, 2, 128, 2, cuda)
    table = dec.rope_table(500, 128, device=cuda)
    q, k = q.clone(), k.clone()
    good = dec.qk_norm_rope(q, k, pos, table, wq, wk)
    q[2, 1] = 0
    k[3, 0, 5] = float("nan")
    got = dec.qk_norm_rope(q, k, pos, table, wq, wk)
    assert not got[0][2, 1].any()
    assert torch.isnan(got[1][3, 0]).all()
    good[0][2, 1], got[1][3, 0] = 0, good[1][3, 0]
    assert torch.equal(got[0], good[0]) and torch.equal(got[1], good[1])


def test_norm_rope_position_outside_the_table(dec, cuda, fp4):
    q, k, _, (wq, wk), _ = heads(4, 2, 1, 64, 3, cuda)
    table = dec.rope_table(16, 64, device=cuda)
    fp4.device_error()
    for bad in (16, -1, 2 ** 40):
        pos = torch.tensor([0, bad, 15, 3], device=cuda)
        got = dec.qk_norm_rope(q, k, pos, table, wq, wk)[0]
        assert fp4.device_error() == 12
        pos[1] = 1
        want = dec.qk_norm_rope(q, k, pos, table, wq, wk)[0]
        assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]]) and fp4.device_error() == 0


def test_rope_table(dec, cuda):
    table = dec.rope_table(300, 16, base=500.0, device=cuda).cpu()
    for p in (0, 1, 77, 299):
        for i in range(8):
            a = p * 500.0 ** (-2 * i / 16)
            assert abs(table[p, i] - math.cos(a)) < 2.0 ** -24 and abs(table[p, 8 + i] - math.sin(a)) < 2.0 ** -24
    with pytest.raises(ValueError):
        dec.rope_table(0, 16, device=cuda)


def test_norm_rope_refusals(dec, cuda):
    q, k, _, (wq, wk), pos = heads(4, 2, 1, 64, 3, cuda)
    table = dec.rope_table(500, 64, device=cuda)
    for args, match in (((q[0], k, pos, table), "tokens, heads"), ((q, k[:2], pos, table), "other tokens"), ((q, k, pos[:2], table), "positions"),
                        ((q, k, pos.float(), table), "positions"), ((q, k, pos, table.double()), "rope"), ((q, k, pos, table[:, :12]), "rope"),
                        ((q, k, pos, table[:, :12].contiguous()), "multiple of 8"), ((q, k, pos, table, wq[:8]), "q_weight"),
                        ((q.cpu(), k, pos, table), "CUDA"), ((q, k.cpu(), pos, table), "CUDA")):
        with pytest.raises(ValueError, match=match):
            dec.qk_norm_rope(*args)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        dec.qk_norm_rope(q[..., :40], k[..., :40], pos, None)


# ------------------------------------------------------------------------------------------------------ the cache

KINDS = ["bf16", "fp8", "nvfp4"]


def stored(x, kind):
    """(codes, scales) of rows x [..., D] by the formats' definitions, on the CPU in fp32."""
    x = x.float().cpu()
    if kind == "bf16":
        return x.to(torch.bfloat16), None
    if kind == "fp8":
        amax = x.abs().amax(-1).clamp(min=2.0 ** -100)
        top = torch.full_like(amax, 448.0)
        return (x * (top / amax).unsqueeze(-1)).clamp(-448, 448).to(torch.float8_e4m3fn), amax / top
    from oracle import nvfp4_oracle as O
    rows = x.reshape(-1, x.shape[-1])
    q, s = O.quantize(O.bf16_bits(rows.to(torch.bfloat16)))
    n, d = rows.shape
    np_, kp = O.round_up(n, 128), O.round_up(d, 128)
    codes = torch.from_numpy(q).reshape(np_, kp // 2)[:n, : d // 2]
    atoms = torch.from_numpy(s).reshape(np_ // 128, kp // 64, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(np_, kp // 16)
    return codes.reshape(*x.shape[:-1], d // 2), atoms[:n, : d // 16].reshape(*x.shape[:-1], d // 16)


def raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 8, 64])
def test_append_and_read(dec, cuda, kind, d, page):
    h, pages = 3, 90 // page + 2
    for t in (1, 2, 37, 90):
        g = torch.Generator().manual_seed(t + d)
        k, v = ((torch.randn(t, h, d, generator=g) * 3).to(torch.bfloat16) for _ in range(2))
        k[t // 2, 1] = 0                                     # a row of zeros
        v[0, 0, ::7] = 400.0                                 # outliers
        v[-1, 2] = (v[-1, 2].float() * 2.0 ** -12).to(torch.bfloat16)  # scales in the subnormal range
        k[0, 2, :16] = torch.tensor([0.75, 1.75, 3.5, -0.75, -1.75, -3.5, 2.5, 5.0, -5.0, 6.0, 0.25, -0.25, 1.25, -0.0, 0.0, -2.5])
        slots = torch.randperm(pages * page, generator=g)[:t]
        cache = dec.PagedKVCache(pages, page, h, d, kind, device=cuda)
        before = [None if x is None else raw(x).clone() for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)]
        cache.append(k.to(cuda), v.to(cuda), slots.to(cuda))
        for x, pages_, scales_, b0, b1 in ((k, cache.k_pages, cache.k_scales, before[0], before[2]),
                                           (v, cache.v_pages, cache.v_scales, before[1], before[3])):
            codes, scales = stored(x, kind)
            want = b0.cpu()
            want[slots // page, :, slots % page] = raw(codes)
            assert torch.equal(raw(pages_).cpu(), want)
            if scales is not None:
                want = b1.cpu()
                want[slots // page, :, slots % page] = scales
                assert torch.equal(scales_.cpu(), want)
        kr, vr = cache.read(slots.to(torch.int32).to(cuda))
        for got, pages_, scales_ in ((kr, cache.k_pages, cache.k_scales), (vr, cache.v_pages, cache.v_scales)):
            want = R.cache_values(pages_, scales_, kind).cpu()[slots // page, :, slots % page]
            if kind == "fp8":
                close(got.cpu(), want, want.abs(), 1, "fp8 read")
            else:
                assert torch.equal(got.cpu().double(), want)  # exact in BF16
    assert "tokens" in repr(cache)


def test_nvfp4_extreme_blocks_equal_the_quantizer(dec, cuda):
    # subnormal scales, huge, infinite and NaN elements: the bytes of the weight quantizer
    x = torch.randn(40, 2, 64, generator=torch.Generator().manual_seed(0))
    x[::5] *= 1e12
    x[1::5] *= 2.0 ** -14
    x[2, 0, 3], x[3, 1, 20], x[4, 0, 40], x[6, 0] = float("inf"), float("-inf"), float("nan"), float("nan")
    x[7, 0, :16] = torch.tensor([2.0 ** 30, -2.0 ** 29] * 8)
    x = x.to(torch.bfloat16)
    cache = dec.PagedKVCache(5, 8, 2, 64, "nvfp4", device=cuda)
    slots = torch.arange(40)
    cache.append(x.to(cuda), x.to(cuda), slots.to(cuda))
    codes, scales = stored(x, "nvfp4")
    assert torch.equal(cache.k_pages.cpu()[slots // 8, :, slots % 8], codes)
    assert torch.equal(cache.v_scales.cpu()[slots // 8, :, slots % 8], scales)


def test_nvfp4_scale_of_every_absmax(dec, cuda):
    # one block for each positive BF16 number, as its absmax: the scale bytes and codes of the weight quantizer
    amax = torch.arange(1, 0x7F80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    n = -(-len(amax) // 8)
    x = torch.zeros(n * 8, 16, dtype=torch.bfloat16)
    x[: len(amax)] = (amax.float().unsqueeze(1) * torch.linspace(-1, 1, 16)).to(torch.bfloat16)
    x = x.reshape(n, 1, 128)
    cache = dec.PagedKVCache(-(-n // 64), 64, 1, 128, "nvfp4", device=cuda)
    slots = torch.arange(n)
    cache.append(x.to(cuda), x.to(cuda), slots.to(cuda))
    codes, scales = stored(x, "nvfp4")
    assert torch.equal(cache.k_scales.cpu()[slots // 64, :, slots % 64], scales)
    assert torch.equal(cache.v_pages.cpu()[slots // 64, :, slots % 64], codes)


def test_fp8_extreme_rows(dec, cuda):
    x = torch.randn(6, 1, 64, generator=torch.Generator().manual_seed(0))
    x[1] *= 2.0 ** -120
    x[2] *= 2.0 ** 120
    x[3, 0, 5] = float("nan")
    x[4, 0, 6] = float("inf")
    x = x.to(torch.bfloat16)
    cache = dec.PagedKVCache(1, 8, 1, 64, "fp8", device=cuda)
    cache.append(x.to(cuda), x.to(cuda), torch.arange(6, device=cuda))
    k, _ = cache.read(torch.arange(6, device=cuda))
    for i in (0, 2, 5):
        assert ((k[i].cpu().double() - x[i].double()).abs() <= 2.0 ** -4 * x[i].double().abs() + x[i].double().abs().max() * 2.0 ** -17).all()
    assert (k[1].cpu().double() - x[1].double()).abs().max() <= 2.0 ** -100
    assert torch.isnan(k[3]).all() and torch.isnan(k[4]).all()  # a row with no absmax is poisoned as a whole, its neighbours are not


@pytest.mark.parametrize("kind", KINDS)
def test_append_qkv_is_norm_rope_then_append(dec, cuda, kind):
    for t, hq, hk, d in ((1, 8, 1, 64), (29, 6, 3, 128), (7, 4, 2, 256), (130, 64, 8, 64)):
        q, k, v, (wq, wk), pos = heads(t, hq, hk, d, t, cuda)
        table = dec.rope_table(500, d // 2 if t == 29 else d, device=cuda)
        cache = dec.PagedKVCache(20, 16, hk, d, kind, device=cuda)
        slots = torch.randperm(320, generator=torch.Generator().manual_seed(t))[:t].to(cuda)
        slots[0] = -1  # skipped
        got = cache.append_qkv(q, k, v, pos, slots, table, wq, wk)
        qs, _ = dec.qk_norm_rope(q, k, pos, table, wq, wk)
        assert torch.equal(got, qs)
        kv, vv = cache.read(slots)
        assert not kv[0].any() and not vv[0].any()
        want = R.norm_rope(k, wk, pos, table, 1e-6, False)
        err = (kv[1:].double() - want[1:]).abs()
        top = want[1:].abs().amax(-1, keepdim=True)
        # one rounding: BF16 half an ulp; E4M3 2^-4 and the subnormals' step; E2M1 at most 1/4 of a value or half a step of
        # its block (scale <= 17/16 amax / 6), then BF16
        bound = {"bf16": 2.0 ** -8 * want[1:].abs(), "fp8": 0.07 * want[1:].abs() + 2.0 ** -10 * top / 448.0,
                 "nvfp4": 0.27 * want[1:].abs() + 0.3 * top / 6.0}[kind]
        assert (err <= bound + 1e-6).all()
        ref = dec.PagedKVCache(20, 16, hk, d, kind, device=cuda)
        ref.append(k, v, slots)
        assert torch.equal(raw(ref.v_pages), raw(cache.v_pages))  # values go in as they are
        none = cache.append_qkv(q, k, v, None, slots, None)
        assert torch.equal(none, q) and torch.equal(raw(ref.k_pages), raw(cache.k_pages))


def test_slots_out_of_range(dec, cuda, fp4):
    fp4.device_error()
    cache = dec.PagedKVCache(3, 4, 2, 64, "bf16", device=cuda)
    k = torch.randn(4, 2, 64, device=cuda).to(torch.bfloat16)
    slots = torch.tensor([2, 12, -5, 11], device=cuda)
    cache.append(k, k, slots)
    assert fp4.device_error() == 11
    got, _ = cache.read(slots)
    assert fp4.device_error() == 11
    assert torch.equal(got[[0, 3]], k[[0, 3]]) and not got[[1, 2]].any()
    assert int((cache.k_pages != 0).any(-1).sum()) == 4
    cache.append(k, k, torch.tensor([2 ** 40, -2 ** 40, 0, 1], device=cuda))
    assert fp4.device_error() == 11


def test_cache_refusals(dec, cuda):
    with pytest.raises(ValueError, match="dtype"):
        dec.PagedKVCache(4, 16, 2, 64, "int8", device=cuda)
    for bad in ((0, 16, 2, 64), (4, 24, 2, 64), (4, 2048, 2, 64), (4, 16, 2, 96)):
        with pytest.raises(ValueError):
            dec.PagedKVCache(*bad, device=cuda)
    with pytest.raises(ValueError, match="CUDA"):
        dec.PagedKVCache(4, 16, 2, 64, device="cpu")
    c = dec.PagedKVCache(4, 16, 2, 64, "fp8", device=cuda)
    with pytest.raises(ValueError, match="needs scales"):
        dec.PagedKVCache.wrap(c.k_pages, c.v_pages)
    with pytest.raises(ValueError, match="alike"):
        dec.PagedKVCache.wrap(c.k_pages, c.v_pages[:2], c.k_scales, c.v_scales)
    with pytest.raises(ValueError, match="scales must be"):
        dec.PagedKVCache.wrap(c.k_pages, c.v_pages, c.k_scales, c.v_scales.double())
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=cuda)
    for args in ((k, k[:2], torch.zeros(3, dtype=torch.int64, device=cuda)), (k[:, :1], k[:, :1], torch.zeros(3, dtype=torch.int64, device=cuda)),
                 (k, k, torch.zeros(2, dtype=torch.int64, device=cuda)), (k, k, torch.zeros(3, device=cuda)),
                 (k, k, torch.zeros(3, dtype=torch.int64)), (k.cpu(), k, torch.zeros(3, dtype=torch.int64, device=cuda))):
        with pytest.raises(ValueError):
            c.append(*args)
    c.append(k[:0], k[:0], torch.zeros(0, dtype=torch.int64, device=cuda))
    assert c.read(torch.zeros(0, dtype=torch.int64, device=cuda))[0].shape == (0, 2, 64)


# ------------------------------------------------------------------------------------------------------ attention

def attention_case(dec, cuda, kind, d, hq, hk, page, lens, seed=0, spread=1.5, width=None):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = max(1, sum(need)) + 2
    cache = dec.PagedKVCache(pages, page, hk, d, kind, device=cuda)
    k, v = ((torch.randn(pages * page, hk, d, generator=g) * s).to(torch.bfloat16).to(cuda) for s in (spread, 1.0))
    cache.append(k, v, torch.arange(pages * page, device=cuda))
    order = torch.randperm(pages, generator=g).to(torch.int32)
    width = max([1] + need) if width is None else width
    table = torch.full((len(lens), width), -7, dtype=torch.int32)  # entries past a sequence's pages are never read
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at: at + n]
        at += n
    q = (torch.randn(len(lens), hq, d, generator=g) * spread).to(torch.bfloat16).to(cuda)
    return q, cache, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)


def attention_check(dec, q, cache, table, lens, window=0, sinks=None, scale=None, rows=None):
    out, lse = dec.decode_attention(q, cache, table, lens, scale=scale, window=window, sinks=sinks, return_lse=True)
    k, v = rows or (R.cache_values(cache.k_pages, cache.k_scales, cache.dtype), R.cache_values(cache.v_pages, cache.v_scales, cache.dtype))
    want, wlse, mag = R.attention(q, k, v, table, lens, cache.page_size, q.shape[-1] ** -0.5 if scale is None else scale, window, sinks)
    vmax = torch.nan_to_num(v.abs(), nan=0.0, posinf=0.0).max()
    n = float(lens.max()) if lens.numel() else 0.0
    err = (out.double() - want).abs()
    bad = err > 2.0 ** -8 * want.abs() + 2.0 ** -10 * mag + n * 2.0 ** -25 * vmax
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {err.max().item()}"
    # a score is a sum of D products in fp32, log and exp another few 2^-22 of a number of its size
    smax = (q.double().norm(dim=-1).max() * torch.nan_to_num(k, nan=0.0).norm(dim=-1).max() * abs(q.shape[-1] ** -0.5 if scale is None else scale)).item()
    both = torch.isfinite(wlse)
    assert torch.equal(torch.isfinite(lse), both)
    assert (lse.double() - wlse)[both].abs().max().item() <= 2.0 ** -18 * (1 + smax) if both.any() else True
    assert torch.equal(out, dec.decode_attention(q, cache, table, lens, scale=scale, window=window, sinks=sinks)), "not the same twice"
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_lengths(dec, cuda, fp4, kind, d):
    lens = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 255, 300, 1025]
    case = attention_case(dec, cuda, kind, d, 8, 2, 16, lens, seed=d)
    attention_check(dec, *case)
    for n in (1, 5, 64, 700):
        attention_check(dec, *attention_case(dec, cuda, kind, d, 4, 1, 32, [n], seed=n))
    assert fp4.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hk", [(1, 1), (2, 2), (3, 1), (8, 1), (9, 1), (16, 2), (10, 2), (17, 1), (40, 1), (48, 3), (16, 16)])
def test_attention_head_layouts(dec, cuda, kind, hq, hk):
    attention_check(dec, *attention_case(dec, cuda, kind, 64, hq, hk, 8, [0, 77, 200, 1], seed=hq))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 32, 128, 1024])
def test_attention_pages(dec, cuda, kind, page):
    attention_check(dec, *attention_case(dec, cuda, kind, 128, 4, 2, page, [3, 333, 0, 1050, 129], seed=page))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("page", [1, 8, 16, 32, 64])
def test_attention_pages_of_other_heads(dec, cuda, kind, d, page):
    attention_check(dec, *attention_case(dec, cuda, kind, d, 4, 2, page, [3, 333, 0, 1050, 129], seed=page + d))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [500, 900, 1500, 1793, 2600, 3329])
def test_attention_of_middle_lengths(dec, cuda, kind, d, n):
    attention_check(dec, *attention_case(dec, cuda, kind, d, 4, 2, 32, [n, n - 257], seed=n))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 8, 16, 32, 64])
def test_attention_without_the_pages_before_a_window(dec, cuda, fp4, kind, page):
    # what lies before a sequence's window may have been given back: its table entries are not read
    for d in (64, 128):
        q, cache, table, seq = attention_case(dec, cuda, kind, d, 4, 2, page, [64, 333, 20, 1050, 129], seed=page)
        for window in (1, 33, 70, 200):
            want = dec.decode_attention(q, cache, table, seq, window=window)
            short = table.clone()
            for i, n in enumerate(seq.tolist()):
                short[i, : max(0, n - window) // page] = -1
            assert torch.equal(dec.decode_attention(q, cache, short, seq, window=window), want)
    assert fp4.device_error() == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 128, 5000])
def test_attention_window_and_sinks(dec, cuda, kind, window):
    case = attention_case(dec, cuda, kind, 64, 8, 2, 16, [0, 1, 16, 17, 99, 100, 101, 500, 1027], seed=window)
    attention_check(dec, *case, window=window)
    sinks = torch.randn(8, generator=torch.Generator().manual_seed(1)).to(cuda) * 4
    sinks[3], sinks[4] = float("-inf"), 60.0
    attention_check(dec, *case, window=window, sinks=sinks)
    attention_check(dec, *case, sinks=sinks)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_many_and_long(dec, cuda, kind):
    g = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.randint(0, 90, (301,), generator=g)]
    lens[100] = 9000
    attention_check(dec, *attention_case(dec, cuda, kind, 64, 4, 2, 16, lens, seed=9))
    attention_check(dec, *attention_case(dec, cuda, kind, 128, 8, 1, 64, [40001, 3, 20000], seed=10))


@pytest.mark.parametrize("kind", KINDS)
def test_attention_sharp_and_flat_softmax(dec, cuda, kind):
    for spread, scale in ((6.0, 1.0), (0.01, 1.0), (1.0, -0.3), (1.0, 0.0)):
        case = attention_case(dec, cuda, kind, 64, 6, 2, 16, [900, 33, 4], seed=4, spread=spread)
        attention_check(dec, *case, scale=scale)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_large_and_small_queries(dec, cuda, kind):
    q, cache, table, lens = attention_case(dec, cuda, kind, 64, 6, 2, 16, [300, 33, 4], seed=4)
    for f in (2.0 ** 40, 2.0 ** -40, 2.0 ** 100):
        attention_check(dec, (q.float() * f).to(torch.bfloat16), cache, table, lens, scale=0.125 / f)


def test_attention_values_of_uneven_scale(dec, cuda):
    # fp8 rows whose scales differ by many powers of two: small values with large weights and the reverse
    g = torch.Generator().manual_seed(3)
    n = 500
    cache = dec.PagedKVCache(32, 16, 1, 64, "fp8", device=cuda)
    k = torch.randn(n, 1, 64, generator=g).to(torch.bfloat16)
    v = torch.randn(n, 1, 64, generator=g) * 2.0 ** torch.randint(-30, 30, (n, 1, 1), generator=g).float()
    cache.append(k.to(cuda), v.to(torch.bfloat16).to(cuda), torch.arange(n, device=cuda))
    q = torch.randn(1, 4, 64, generator=g).to(torch.bfloat16).to(cuda)
    table, lens = torch.arange(32, dtype=torch.int32, device=cuda).reshape(1, 32), torch.tensor([n], dtype=torch.int32, device=cuda)
    attention_check(dec, q, cache, table, lens)
    small = dec.PagedKVCache(32, 16, 1, 64, "fp8", device=cuda)
    small.append(k.to(cuda), (v * 2.0 ** -60).to(torch.bfloat16).to(cuda), torch.arange(n, device=cuda))
    attention_check(dec, q, small, table, lens)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_never_looks_at_what_is_masked(dec, cuda, kind):
    # NaN everywhere that no sequence sees: behind its length, before its window, in other pages
    lens = [0, 1, 37, 64, 130]
    q, cache, table, seq = attention_case(dec, cuda, kind, 64, 4, 2, 16, lens, seed=6)
    for window in (0, 20):
        want = dec.decode_attention(q, cache, table, seq, window=window)
        seen = torch.zeros(cache.num_pages * 16, dtype=torch.bool)
        for i, n in enumerate(lens):
            for j in range(max(0, n - window) if window else 0, n):
                seen[int(table[i, j // 16]) * 16 + j % 16] = True
        dirty = dec.PagedKVCache.wrap(*(None if x is None else x.clone() for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)))
        hidden = (~seen).reshape(cache.num_pages, 16).to(cuda)
        for t in (dirty.k_pages, dirty.v_pages, dirty.k_scales, dirty.v_scales):
            if t is not None:
                t.transpose(1, 2)[hidden] = 0x7F if t.dtype == torch.uint8 else torch.tensor(float("nan"), device=cuda).to(t.dtype)
        assert torch.equal(dec.decode_attention(q, dirty, table, seq, window=window), want)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_attention_non_finite_keys_and_values_show(dec, cuda, kind):
    q, cache, table, seq = attention_case(dec, cuda, kind, 64, 4, 2, 16, [50, 60], seed=6)
    want = dec.decode_attention(q, cache, table, seq)
    bad = torch.randn(1, 2, 64, device=cuda).to(torch.bfloat16)
    good, _ = cache.read(table[1, 2:3].long() * 16 + 3)
    bad[0, 1, 5] = float("nan")
    bad[0, 0] = good[0, 0]
    cache.append(bad, good, table[1, 2:3].long() * 16 + 3)
    out = dec.decode_attention(q, cache, table, seq)
    assert torch.equal(out[0], want[0]) and torch.isnan(out[1, 2:]).all() and not torch.isnan(out[1, :2]).any()


def test_attention_strides_streams_and_graph(dec, cuda):
    q, cache, table, seq = attention_case(dec, cuda, "nvfp4", 64, 8, 2, 16, [50, 600, 0, 7], seed=6)
    want = dec.decode_attention(q, cache, table, seq)
    wide = torch.zeros(4, 8, 100, dtype=torch.bfloat16, device=cuda)
    for at in (0, 4, 1):
        wide[..., at: at + 64] = q
        assert torch.equal(dec.decode_attention(wide[..., at: at + 64], cache, table, seq), want)
    more = torch.full((4, 90), -1, dtype=torch.int32, device=cuda)
    more[:, : table.shape[1]] = table
    assert torch.equal(dec.decode_attention(q, cache, more, seq), want)
    assert torch.equal(dec.decode_attention(q, cache, more[:, : table.shape[1]], seq), want)
    assert torch.equal(dec.decode_attention(q, cache, table.t().contiguous().t(), seq), want)
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        outs = [dec.decode_attention(q, cache, table, seq) for _ in range(20)]
    outs += [dec.decode_attention(q, cache, table, seq) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = dec.decode_attention(q, cache, table, seq)
        graphs.append((g, out))
    for stream in (side, torch.cuda.Stream(cuda)):
        for g, out in graphs:
            out.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                g.replay()
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out in graphs)


def test_attention_out_of_range_pages_and_lengths(dec, cuda, fp4):
    q, cache, table, seq = attention_case(dec, cuda, "bf16", 64, 4, 2, 16, [50, 60, 20], seed=6)
    want = dec.decode_attention(q, cache, table, seq)
    fp4.device_error()
    for bad in (cache.num_pages, -1, 2 ** 30):
        broken = table.clone()
        broken[1, 1] = bad
        out = dec.decode_attention(q, cache, broken, seq)
        assert fp4.device_error() == 13
        assert torch.equal(out[[0, 2]], want[[0, 2]]) and torch.isfinite(out).all()
    for bad in (65, 2 ** 31 - 1, -1):  # longer than the table has pages for (64 keys here)
        long = seq.clone()
        long[1] = bad
        full = table.clone()
        full[:, 3] = 0
        out = dec.decode_attention(q, cache, full, long)
        assert fp4.device_error() == 13
        assert torch.equal(out[[2]], want[[2]]) and torch.isfinite(out).all()
    assert torch.equal(dec.decode_attention(q, cache, table, seq), want) and fp4.device_error() == 0


def test_attention_refusals(dec, cuda):
    q, cache, table, seq = attention_case(dec, cuda, "bf16", 64, 4, 2, 16, [50, 60, 20], seed=6)
    for args in ((q[:, :3], cache, table, seq), (q[..., :32], cache, table, seq), (q[:2], cache, table, seq), (q, cache, table.long(), seq),
                 (q, cache, table, seq.long()), (q, cache, table, seq[:2]), (q, cache, table.cpu(), seq), (q.cpu(), cache, table, seq),
                 (q, cache, table[0], seq)):
        with pytest.raises(ValueError):
            dec.decode_attention(*args)
    with pytest.raises(ValueError, match="window"):
        dec.decode_attention(q, cache, table, seq, window=-1)
    with pytest.raises(ValueError, match="sinks"):
        dec.decode_attention(q, cache, table, seq, sinks=torch.zeros(3, device=cuda))
    with pytest.raises(RuntimeError, match="scale finite"):
        dec.decode_attention(q, cache, table, seq, scale=float("inf"))
    assert dec.decode_attention(q[:0], cache, table[:0], seq[:0]).shape == (0, 4, 64)


def test_attention_parts_join_by_their_lse(dec, cuda):
    q, cache, table, seq = attention_case(dec, cuda, "fp8", 64, 8, 2, 16, [600], seed=6)
    whole, lse = dec.decode_attention(q, cache, table, seq, return_lse=True)
    a, la = dec.decode_attention(q, cache, table, torch.full_like(seq, 320), return_lse=True)
    b, lb = dec.decode_attention(q, cache, table[:, 20:], seq - 320, return_lse=True)
    both = torch.logaddexp(la, lb)
    joined = a.double() * (la - both).exp().unsqueeze(-1) + b.double() * (lb - both).exp().unsqueeze(-1)
    assert (both - lse).abs().max() < 1e-5
    close(whole, joined, a.double().abs() + b.double().abs(), 2 ** 13, "joined")
