"""Host side of the operators that close a decoding step (no GPU): the argument structs and the C entry points' refusals before
any device work."""
import ctypes
import os
import struct
import subprocess

import pytest
import torch

import fp4_decode
import fp4_gemm
from tests.conftest import ROOT

lib = fp4_gemm._lib


def last():
    return fp4_gemm._last_error()


STRUCTS = {"fp4b_norm": (fp4_decode._NORM, "PlPlPlPPPPiiiff", ["x", "x_stride", "residual", "residual_stride", "gate", "gate_stride", "weight",
                                                               "post_weight", "normed", "residual_out", "rows", "width", "residual_fp32", "scale", "eps"]),
           "fp4b_sampling": (fp4_decode._SAMPLING, "PlPPPPPPPiiififf", ["logits", "stride", "u", "temperature", "top_k", "top_p", "min_p", "tokens",
                                                                        "probs", "rows", "vocab", "type", "temperature1", "top_k1", "top_p1", "min_p1"])}


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_structs_match_the_header(tmp_path, name):
    form, codes, members = STRUCTS[name]
    src = f'#include <stddef.h>\n#include <stdio.h>\n#include "fp4gemm.h"\nint main(void) {{\nprintf("%zu", sizeof({name}));\n'
    src += "".join(f'printf(" %zu", offsetof({name}, {m}));\n' for m in members) + "return 0;\n}\n"
    (tmp_path / "s.c").write_text(src)
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    got = list(map(int, subprocess.check_output([str(tmp_path / "s")], text=True).split()))
    assert got == [form.size] + [struct.calcsize("@" + codes[:i] + "0" + codes[i]) for i in range(len(codes))]


def test_shared_struct_matches_the_header(tmp_path):
    own = ["q", "q_sb", "q_sh", "cache", "page_table", "table_stride", "seq_lens", "sinks", "out", "lse", "workspace", "workspace_bytes", "batch",
           "q_heads", "table_width", "window", "scale"]
    members = [f"own.{m}" for m in own] + ["prefix_table", "prefix_stride", "prefix_lens", "prefixes", "prefix_width"]
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "fp4gemm.h"\nint main(void) {\nprintf("%zu", sizeof(fp4b_shared));\n'
    src += "".join(f'printf(" %zu", offsetof(fp4b_shared, {m}));\n' for m in members) + "return 0;\n}\n"
    (tmp_path / "s.c").write_text(src)
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    got = list(map(int, subprocess.check_output([str(tmp_path / "s")], text=True).split()))
    codes = "PllPPlPPPPPliiiifPlPii"
    assert len(codes) == len(members)
    assert got == [fp4_decode._SHARED.size] + [struct.calcsize("@" + codes[:i] + "0" + codes[i]) for i in range(len(codes))]


def shared_call(cache_fields=(), **other):
    fields = dict(k=0x10000, v=0x20000, k_scale=None, v_scale=None, num_pages=4, kv_heads=2, page_size=16, head_dim=64, kind=0)
    cache = fp4_decode._CacheView(**{**fields, **dict(cache_fields)})
    v = dict(q=0x10000, q_sb=512, q_sh=64, cache=ctypes.addressof(cache), page_table=0x20000, table_stride=4, seq_lens=0x30000, sinks=0, out=0x40000,
             lse=0, workspace=0x50000, workspace_bytes=1 << 40, batch=4, q_heads=8, table_width=4, window=0, scale=0.125, prefix_table=0x60000,
             prefix_stride=8, prefix_lens=0x70000, prefixes=2, prefix_width=8)
    v.update(other)
    return lib.fp4b_shared_attention(fp4_decode._SHARED.pack(*v.values()), None)


def test_bad_shared_attention_calls_are_refused():
    for other in (dict(batch=-1), dict(q_heads=0), dict(q_heads=7), dict(q=0), dict(out=0), dict(seq_lens=0), dict(page_table=0), dict(table_width=-1),
                  dict(table_stride=3), dict(window=1), dict(window=-1), dict(scale=float("nan")), dict(q=0x10004), dict(q_sb=511), dict(out=0x40008),
                  dict(workspace=0), dict(workspace=0x50004), dict(prefixes=0), dict(prefixes=-2), dict(prefixes=3), dict(prefix_lens=0),
                  dict(prefix_table=0), dict(prefix_width=-1), dict(prefix_stride=7), dict(prefix_width=1 << 28, prefix_stride=1 << 28),
                  dict(batch=1 << 20, prefixes=1 << 20, prefix_width=1 << 12, prefix_stride=1 << 12), dict(cache=0)):
        assert shared_call(**other) == -1, other
        assert "fp4b_shared_attention" in last()
    for bad in (dict(k=None), dict(page_size=24), dict(head_dim=96), dict(kind=1)):
        assert shared_call(bad) == -1, bad
    assert lib.fp4b_shared_attention(None, None) == -1
    assert shared_call(batch=0) == 0
    assert lib.fp4b_shared_attention_workspace(1, 4, 7, 2, 64) == -1


def norm_call(**other):
    v = dict(x=0x10000, x_stride=64, residual=0x20000, residual_stride=64, gate=0, gate_stride=0, weight=0x30000, post_weight=0, normed=0x40000,
             residual_out=0x50000, rows=1, width=64, residual_fp32=0, scale=1.0, eps=1e-6)
    v.update(other)
    return lib.fp4b_block_norm(fp4_decode._NORM.pack(*v.values()), None)


def test_bad_norm_calls_are_refused():
    for other in (dict(rows=-1), dict(width=0), dict(width=-8), dict(width=32769), dict(residual=0), dict(weight=0), dict(normed=0), dict(residual_out=0),
                  dict(x=0, gate=0x60000), dict(x=0, post_weight=0x60000), dict(scale=float("nan")), dict(scale=float("inf")), dict(eps=-1e-9),
                  dict(eps=float("nan")), dict(x=0x10001), dict(residual=0x20001), dict(residual=0x20002, residual_fp32=1), dict(gate=0x60001),
                  dict(weight=0x30001), dict(post_weight=0x60001), dict(normed=0x40001), dict(residual_out=0x50002, residual_fp32=1)):
        assert norm_call(**other) == -1, other
        assert "fp4b_block_norm" in last()
    assert lib.fp4b_block_norm(None, None) == -1
    assert norm_call(rows=0) == 0


def sample_call(**other):
    v = dict(logits=0x10000, stride=100, u=0x20000, temperature=0, top_k=0, top_p=0, min_p=0, tokens=0x30000, probs=0, rows=1, vocab=100, type=0,
             temperature1=1.0, top_k1=0, top_p1=1.0, min_p1=0.0)
    v.update(other)
    return lib.fp4b_sample(fp4_decode._SAMPLING.pack(*v.values()), None)


def test_bad_sampling_calls_are_refused():
    for other in (dict(rows=-1), dict(rows=(1 << 27) + 1), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(type=3), dict(type=-1), dict(logits=0), dict(u=0),
                  dict(tokens=0), dict(logits=0x10001), dict(logits=0x10002, type=2), dict(temperature1=-0.5), dict(temperature1=float("nan"))):
        assert sample_call(**other) == -1, other
        assert "fp4b_sample" in last()
    assert lib.fp4b_sample(None, None) == -1
    assert sample_call(rows=0) == 0


def test_tensors_on_the_host_are_refused():
    x, w, u = torch.zeros(2, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16), torch.zeros(2)
    with pytest.raises(ValueError):
        fp4_decode.block_norm(x, x, w)
    with pytest.raises(ValueError):
        fp4_decode.sample(x, u)
