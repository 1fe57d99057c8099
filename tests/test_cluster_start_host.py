"""Kernels that touch another CTA's shared memory meet their cluster first: a CTA that has not started has none.  An idle GPU
hides a missing meeting, so the order is checked in the sources (no GPU)."""
import os
import re

import pytest

from tests.conftest import ROOT

CSRC = os.path.join(ROOT, "fp4-gemm-blackwell_b200", "csrc")
REMOTE = r"map_shared_rank\s*\(|mapa_shared\s*\(|mapa\."
MEETING = r"cluster_start_wait\s*\(\)|cluster\.sync\s*\(\)|cluster_sync\s*\(\)"


def body(text, at):
    """The braces' content that opens behind `at`."""
    begin = text.index("{", at)
    depth = 0
    for i in range(begin, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[begin: i + 1]
    raise ValueError("unbalanced braces")


def parts(name):
    """(kernels {name: body}, pattern of what reaches another CTA's memory) of a source file."""
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    helpers = []
    for m in re.finditer(r"__device__ __forceinline__ [\w:<> ,*&]*?\b(\w+)\(", text):
        if re.search(REMOTE, body(text, m.end())):
            helpers.append(r"\b%s\s*(?:<[^<>;]*>)?\s*\(" % m.group(1))
    kernels = {}
    for m in re.finditer(r"__global__ void __launch_bounds__\(", text):
        depth, i = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[i], 0)
            i += 1
        kernels[re.match(r"\s*(\w+)", text[i:]).group(1)] = body(text, i)
    return kernels, "|".join([REMOTE, *helpers])


def check(name):
    kernels, remote = parts(name)
    assert kernels
    for kernel, text in kernels.items():
        first, met = re.search(remote, text), re.search(MEETING, text)
        assert first, f"{kernel}: no access to another CTA"
        assert met and met.start() < first.start(), f"{kernel}: another CTA's shared memory before the first meeting of the cluster"


def test_block_norm():
    check("block_norm.cu")


def test_sample():
    check("sample.cu")
