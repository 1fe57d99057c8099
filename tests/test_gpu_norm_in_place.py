"""fp4b_block_norm of a residual that is updated in place, as the C entry point allows: the same bytes as into a new one."""
import pytest
import torch

from tests.test_gpu_block_norm import inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec(cuda):
    import fp4_decode
    return fp4_decode


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
# a warp's width, a CTA's, a cluster's (few rows; too wide for one CTA), in pieces of 8, 2 and 1; rows of one wave and of more
@pytest.mark.parametrize("t,h", [(1, 264), (3, 8192), (1, 16384), (2, 32767), (7, 32768), (5, 20002), (300, 2880), (3001, 1000), (40000, 24), (2500, 4097), (700, 20001)])
def test_in_place(dec, cuda, kind, t, h):
    x, residual, (w, post), gates = inputs(t, h, cuda, kind)
    want = dec.block_norm(x, residual, w, post, gates[2], 0.5)
    normed = torch.empty_like(want[0])
    for stride in {h, h if t > 1 else 7 * h}:  # (one row has no other to lie over)
        r = residual.clone()
        dec._call(r.device, dec._block_norm, "block_norm", dec._NORM.pack(
            x.data_ptr(), h, r.data_ptr(), stride, gates[2].data_ptr(), h, w.data_ptr(), post.data_ptr(), normed.data_ptr(), r.data_ptr(), t, h,
            kind == torch.float32, 0.5, 1e-6))
        assert torch.equal(normed, want[0]) and torch.equal(r, want[1])
