"""The prefix kernel's scores go over the weights of an earlier tile in tensor memory, and tensor instructions of other shapes
are not bound to their order: the product that reads those weights has ended first.  No run shows a missing wait, so the order
is checked in the source (no GPU)."""
import os
import re

from tests.conftest import ROOT


def test_scores_wait_for_the_product_that_reads_their_columns():
    with open(os.path.join(ROOT, "fp4-gemm-blackwell_b200", "csrc", "shared_attention.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    role = text[text.index("s_desc = ptx::idesc_f16"):]
    loop = role[role.index("ok && j < n; ++j, ++it"):]
    before = loop[: loop.index("scores(it + kAhead)")]
    # tile it - 1's, whose buffer is the one of tile it + BUFFERS - 1
    assert re.search(r"kAhead = C::BUFFERS - 1", role)
    assert re.search(r"if \(j > 0\) ok = wait\(o_done \+ .*\(it - 1\) & 1.*\(\(it - 1\) / SLOTS\) & 1\)", before)
