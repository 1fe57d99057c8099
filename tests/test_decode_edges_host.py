"""Host side of the decode operators where shapes only just fit (no GPU)."""
import pytest

import fp4_gemm

lib = fp4_gemm._lib
STEP = 128        # elements of K of a step
HELD = 65536      # bytes of x in FP16 that a CTA can hold: its threads' registers and its shared memory are made for that many


def slices_of(m, n, k):
    """Into how many slices a call cuts K, by the sums that it wants room for (m rows of at most one tile)."""
    tile = 8 if m <= 8 else 16
    need = lib.fp4b_gemv_workspace(m, k, n)
    slices, rest = divmod(need, tile * (-(-n // 128) * 128) * 4)
    assert need >= 0 and rest == 0
    return max(slices, 1)


@pytest.mark.parametrize("m", range(1, 17))
def test_longest_slice_of_x_fits_a_cta(m):
    # slices are whole steps, the longest of them one longer than the shortest
    ns = sorted({1, 100, 512, 1000, 2880, 4096, 5120, 9000, 14336, 16384, 160000} | {128 * i for i in range(3, 460, 11)})
    ks = sorted({1, 129, 65536, 100000} | {128 * i for i in range(1, 513)} | {128 * i - 127 for i in range(1, 512, 17)})
    bad = []
    for n in ns:
        for k in ks:
            steps = -(-(-(-k // STEP)) // slices_of(m, n, k))
            if steps * m * STEP * 2 > HELD:
                bad.append((m, n, k, steps))
    assert not bad, f"{len(bad)} shapes, such as {bad[:5]}"


@pytest.mark.parametrize("m,n,k", [(6, 19072, 16384), (9, 15360, 14464), (12, 12288, 16384), (14, 10240, 16384), (13, 12416, 12288),
                                   (7, 28672, 9344), (9, 16384, 14400), (10, 14336, 16384), (14, 53248, 16384), (11, 16384, 53248)])
def test_slices_of_shapes_that_did_not_fit(m, n, k):
    assert -(-(-(-k // STEP)) // slices_of(m, n, k)) * m * STEP * 2 <= HELD


def test_slices_of_a_very_long_row():
    # K * rows passes 32 bits in bytes
    for k in (1 << 26, (1 << 26) + 128, 100_000_000):
        assert -(-(-(-k // STEP)) // slices_of(16, 128, k)) * 16 * STEP * 2 <= HELD
