"""fp4b_shared_attention without a device that it can size its workspace for: refused before anything is laid out or launched."""
import pytest
import torch

from tests.test_decode_step_host import last, shared_call


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where there is no GPU to read them")
@pytest.mark.parametrize("cache", [{}, dict(kind=1, k_scale=0x30000, v_scale=0x40000), dict(kind=2, k_scale=0x30000, v_scale=0x40000)])
def test_no_device(cache):
    assert shared_call(cache) == -1
    assert "no device" in last()
