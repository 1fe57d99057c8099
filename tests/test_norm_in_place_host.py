"""fp4b_block_norm with residual_out the residual itself: refused where a row's result would lie over another row (no GPU)."""
import pytest

from tests.test_decode_step_host import last, norm_call

SAME = dict(residual=0x20000, residual_out=0x20000)


@pytest.mark.parametrize("fp32", [0, 1])
@pytest.mark.parametrize("stride", [0, 1, 63, 65, 72, 128])
def test_rows_apart_are_refused(fp32, stride):
    assert norm_call(**SAME, rows=2, residual_stride=stride, residual_fp32=fp32) == -1
    assert "in place" in last()


def test_nothing_to_do_is_not():
    assert norm_call(**SAME, rows=0, residual_stride=65) == 0
