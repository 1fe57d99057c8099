"""Host side of the decode operators where shapes only just fit (no GPU)."""
import pytest
import torch

import fp4_decode
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


def test_page_tables_of_any_strides():
    # entry i of row b is read at b * distance + i from the table's address
    base = torch.arange(60, dtype=torch.int32)
    forms = {"plain": base.view(6, 10), "wide": base.view(6, 10)[:, :7], "part": base.view(6, 10)[1:4, 2:9], "one row": base[:9].view(1, 9),
             "one row for all": base[:9].view(1, 9).expand(5, 9), "one entry for all": base[:1].view(1, 1).expand(5, 7),
             "one column": base.view(6, 10)[:, 3:4], "one column for all": base[:1].view(1, 1).expand(5, 1), "turned": base.view(10, 6).t(),
             "overlapping": base.as_strided((4, 9), (3, 1)), "every other": base.view(6, 10)[:, ::2], "every other row": base.view(6, 10)[::2],
             "one row of a turned table": base.view(10, 6).t()[2:3], "one row, every third": base[::3].view(1, 20), "far rows": base.as_strided((1, 5), (0, 1)),
             "no columns": base.view(6, 10)[:, :0], "no rows": base.view(6, 10)[:0]}
    for name, table in forms.items():
        got, distance = fp4_decode._table(table)
        b, width = table.shape
        assert distance >= width, name
        flat = got.as_strided((max(0, (b - 1) * distance + width) if b and width else 0,), (1,))
        for r in range(b):
            assert flat[r * distance: r * distance + width].tolist() == table[r].tolist(), name
        if name in ("plain", "wide", "part", "one row", "one column", "every other row"):
            assert got.data_ptr() == table.data_ptr(), name  # nothing to copy


def test_workspace_of_many_rows_is_bounded():
    for n, k in ((128, 128), (128, 4096), (2880, 2880), (16384, 16384), (160000, 65536)):
        one = lib.fp4b_gemv_workspace(16, k, n)
        for m in (17, 40, 1000, 8192, 65535, 65536, 1 << 20, (1 << 31) - 1):
            need = lib.fp4b_gemv_workspace(m, k, n)
            assert one <= need <= max(one, 256 << 20), (m, n, k, need)
            assert one == 0 or need % one == 0  # whole tiles of 16 rows


def test_cleanup_without_a_gpu():
    if not torch.cuda.is_initialized():
        fp4_gemm.cleanup()
        assert not torch.cuda.is_initialized()
