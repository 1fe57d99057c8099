"""What a kernel does that gives up while copies into its shared memory are under way: it waits for them, and for nobody else."""
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_copies_land_without_the_partner_that_stopped(cuda, fp4):
    assert fp4.device_error(clear=True) == 0
    stream = torch.cuda.current_stream(cuda).cuda_stream
    began = time.monotonic()
    for _ in range(3):
        assert fp4._lib.fp4b_selftest_flights(stream) == 0, fp4._last_error()
    assert fp4.device_error(clear=True) == 0  # synchronises
    assert time.monotonic() - began < 1.5  # one wait that gives up takes 2 s
