"""fp4_decode.sample where its bins end: zeros of both signs under temperatures next to nothing."""
import pytest
import torch

from tests.test_gpu_sample import TYPES, check

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec(cuda):
    import fp4_decode
    return fp4_decode


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1e-33, 1.6e-34, 1e-36, 1e-38, 1e-40])
@pytest.mark.parametrize("v", [8, 256, 20000])
def test_zeros_of_both_signs_are_equal(dec, cuda, dtype, temperature, v):
    # all weights are 1, whatever the sign: token j for u in [j / V, (j + 1) / V)
    b = min(v, 64)
    at = torch.arange(b, device=cuda) * (v // b) + torch.arange(b, device=cuda) % (v // b)
    u = ((at.double() + 0.5) / v).float()
    logits = torch.zeros(b, v, device=cuda)
    logits[:, ::2] = -0.0
    logits[1::2, ::3] = 0.0
    logits = logits.to(dtype)
    assert check(dec, logits, u, temperature).tolist() == at.tolist()
    check(dec, logits, u, temperature, 5, 1.0, 0.0)
    check(dec, logits, u, temperature, 0, 0.3, 0.0)
    check(dec, logits, u, temperature, v // 2 + 1, 0.7, 0.5)
    assert check(dec, logits, u, temperature, 1).tolist() == [0] * b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size,temperature", [(1e-36, 1e-36), (2.0 ** -112, 2.0 ** -114), (2.0 ** -126, 2.0 ** -128), (2.0 ** -133, 2.0 ** -133), (2.0 ** -120, 1e-40)])
def test_logits_next_to_zero(dec, cuda, dtype, size, temperature):
    # the bins' least magnitudes: small multiples of a small number (some of them subnormal) among zeros of both signs
    g = torch.Generator(cuda).manual_seed(7)
    b, v = 24, 3000
    steps = torch.randint(-6, 4, (b, v), generator=g, device=cuda)
    logits = (steps * size).to(dtype)
    logits[steps == 0] *= torch.where(torch.rand(int((steps == 0).sum()), generator=g, device=cuda) < 0.5, -1.0, 1.0).to(dtype)
    u = torch.rand(b, generator=g, device=cuda)
    check(dec, logits, u, temperature)
    check(dec, logits, u, temperature, 900, 0.8, 0.01)


def test_wide_counts_are_not_cut(dec, cuda):
    # k as int64, beyond 32 bits either way: more than the vocabulary is all of it, less than 0 too
    g = torch.Generator(cuda).manual_seed(8)
    k = torch.tensor([1, 5, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 1, 2 ** 32 + 1, 2 ** 32 + 5, 2 ** 62 + 3, -1, -2 ** 31 - 1, -2 ** 32 + 5, -2 ** 62 + 1], device=cuda)
    b, v = len(k), 500
    logits, u = torch.randn(1, v, generator=g, device=cuda).expand(b, v), torch.full((b,), 0.93, device=cuda)
    whole = [1, 5] + [0] * (b - 2)
    assert torch.equal(dec.sample(logits, u, 1.0, k), dec.sample(logits, u, 1.0, torch.tensor(whole, dtype=torch.int32, device=cuda)))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_logits_in_one_bin_take_no_time_of_their_own(dec, cuda, dtype):
    # zeros (a padded vocabulary, a mask by multiplication) and equal or nearly equal logits meet at one sum in shared memory:
    # the tokens are right, and a row takes a few times an ordinary one's time, not a hundred times
    g = torch.Generator(cuda).manual_seed(9)
    b, v = 256, 65536
    ordinary = (2.0 * torch.randn(b, v, generator=g, device=cuda) - 2.0).to(dtype)
    zeros = ordinary.masked_fill(torch.rand(b, v, generator=g, device=cuda) < 0.5, 0.0)
    close = (20.0 + 1e-3 * torch.randn(b, v, generator=g, device=cuda)).to(dtype)
    equal = torch.full((b, v), 3.0, device=cuda).to(dtype)
    u = torch.rand(b, generator=g, device=cuda)

    def time(logits):
        times = []
        for _ in range(4):
            began, ended = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda._sleep(1_000_000)
            began.record()
            for _ in range(3):
                dec.sample(logits, u, 0.8, 0, 0.95)
            ended.record()
            torch.cuda.synchronize()
            times.append(began.elapsed_time(ended))
        return min(times)

    usual = time(ordinary)
    for what, logits in (("zeros", zeros), ("close", close), ("equal", equal)):
        check(dec, logits[:8], u[:8], 0.8, what=what)
        check(dec, logits[:8], u[:8], 0.8, 1000, 0.95, 0.01, what=what)
        took = time(logits)
        assert took < 15 * usual, (what, took, usual)
