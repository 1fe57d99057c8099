"""Host side of the decode operators (no GPU): the argument structs, the C entry points' refusals before any device work,
and the Python layer's checks."""
import ctypes
import os
import subprocess

import pytest
import torch

import fp4_decode
import fp4_gemm
from tests.conftest import ROOT

lib = fp4_gemm._lib


def last():
    return fp4_gemm._last_error()


def test_structs_match_the_header(tmp_path):
    fields = {"fp4b_rows": ["q", "q_st", "q_sh", "k", "k_st", "k_sh", "v", "v_st", "v_sh", "positions", "slots", "rope", "q_weight", "k_weight",
                            "q_out", "k_out", "cache", "tokens", "q_heads", "kv_heads", "head_dim", "rope_rows", "rot", "interleaved", "pos64",
                            "slot64", "eps"],
              "fp4b_decode": ["q", "q_sb", "q_sh", "cache", "page_table", "table_stride", "seq_lens", "sinks", "out", "lse", "workspace",
                              "workspace_bytes", "batch", "q_heads", "table_width", "window", "scale"],
              "fp4b_kv_cache": [n for n, _ in fp4_decode._CacheView._fields_]}
    src = '#include <stddef.h>\n#include <stdio.h>\n#include "fp4gemm.h"\nint main(void) {\n'
    for name, members in fields.items():
        src += f'printf("%zu", sizeof({name}));\n' + "".join(f'printf(" %zu", offsetof({name}, {m}));\n' for m in members) + 'printf("\\n");\n'
    src += 'printf("%d %d %d %d\\n", FP4B_KV_BF16, FP4B_KV_FP8, FP4B_KV_NVFP4, FP4B_DECODE_COUNTER_BYTES);\nreturn 0;\n}\n'
    (tmp_path / "s.c").write_text(src)
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")])
    rows, decode, cache, enums = (list(map(int, l.split())) for l in subprocess.check_output([str(tmp_path / "s")], text=True).splitlines())

    def offsets(form):
        import struct
        codes = [c for c in form[1:] if c.isalpha()]
        return [struct.calcsize("@" + "".join(codes[:i]) + "0" + codes[i]) for i in range(len(codes))]

    assert rows == [fp4_decode._ROWS.size] + offsets("@PllPllPllPPPPPPPPiiiiiiiiif")
    assert decode == [fp4_decode._DECODE.size] + offsets("@PllPPlPPPPPliiiif")
    assert cache == [ctypes.sizeof(fp4_decode._CacheView)] + [getattr(fp4_decode._CacheView, n).offset for n in fields["fp4b_kv_cache"]]
    assert enums == [fp4_decode.KV_KINDS["bf16"], fp4_decode.KV_KINDS["fp8"], fp4_decode.KV_KINDS["nvfp4"], fp4_decode._COUNTER_BYTES]


def view(**other):
    """A cache description of fake addresses: nothing is dereferenced."""
    v = dict(k=0x10000, v=0x20000, k_scale=0x30000, v_scale=0x40000, num_pages=4, kv_heads=2, page_size=16, head_dim=64, kind=1)
    v.update(other)
    return fp4_decode._CacheView(**v)


BAD_CACHES = [dict(k=None), dict(num_pages=0), dict(kv_heads=0), dict(page_size=0), dict(page_size=24), dict(page_size=2048), dict(head_dim=96),
              dict(kind=3), dict(kind=-1), dict(k=0x10008), dict(v_scale=None), dict(k_scale=0x30004),
              dict(num_pages=1 << 30, kv_heads=8)]


@pytest.mark.parametrize("other", BAD_CACHES)
def test_bad_caches_are_refused(other):
    v = view(**other)
    ref = ctypes.addressof(v)
    assert lib.fp4b_kv_read(ref, 0x50000, 1, 4, 0x60000, 0x70000, None) == -1 and "fp4b_kv_read" in last()
    rows = fp4_decode._ROWS.pack(0, 0, 0, 0x50000, 128, 64, 0x60000, 128, 64, 0, 0x70000, 0, 0, 0, 0, 0, ref, 1, 0, 2, 64, 0, 0, 0, 0, 1, 0.0)
    assert lib.fp4b_kv_rows(rows, None) == -1 and "fp4b_kv_rows" in last()
    call = fp4_decode._DECODE.pack(0x50000, 512, 64, ref, 0x60000, 4, 0x70000, 0, 0x80000, 0, 0x90000, 1 << 40, 1, 8, 4, 0, 0.125)
    assert lib.fp4b_decode_attention(call, None) == -1 and "fp4b_decode_attention" in last()


def rows_call(**other):
    v = dict(q=0x10000, q_st=512, q_sh=64, k=0x20000, k_st=128, k_sh=64, v=0, v_st=0, v_sh=0, positions=0x30000, slots=0, rope=0x40000, q_weight=0,
             k_weight=0, q_out=0x50000, k_out=0x60000, cache=0, tokens=1, q_heads=8, kv_heads=2, head_dim=64, rope_rows=10, rot=64, interleaved=0,
             pos64=1, slot64=0, eps=1e-6)
    v.update(other)
    return lib.fp4b_kv_rows(fp4_decode._ROWS.pack(*v.values()), None)


def test_bad_rows_are_refused():
    good_cache = view()
    ref = ctypes.addressof(good_cache)
    for other in (dict(tokens=-1), dict(q_heads=-1), dict(kv_heads=0), dict(head_dim=40), dict(head_dim=288), dict(head_dim=0), dict(q=0x10004),
                  dict(q_st=511), dict(k_sh=66), dict(rot=0), dict(rot=72), dict(rot=12), dict(rope_rows=0), dict(positions=0), dict(q_weight=0x7),
                  dict(q_out=0), dict(k_out=0), dict(q_out=0x50004), dict(q=0, k=0), dict(v=0x90000, v_st=128, v_sh=64),
                  dict(tokens=1 << 30, kv_heads=8), dict(cache=ref), dict(cache=ref, v=0x90000, v_st=128, v_sh=64),
                  dict(cache=ref, v=0x90000, v_st=128, v_sh=64, slots=0xA0000, kv_heads=4),
                  dict(cache=ref, v=0x90000, v_st=128, v_sh=64, slots=0xA0000, head_dim=128, rot=64)):
        assert rows_call(**other) == -1, other
        assert "fp4b_kv_rows" in last()
    assert lib.fp4b_kv_rows(None, None) == -1
    assert rows_call(tokens=0) == 0  # nothing to do


def decode_call(**other):
    cache = view(kind=0, k_scale=None, v_scale=None)
    v = dict(q=0x10000, q_sb=512, q_sh=64, cache=ctypes.addressof(cache), page_table=0x20000, table_stride=4, seq_lens=0x30000, sinks=0, out=0x40000,
             lse=0, workspace=0x50000, workspace_bytes=1 << 40, batch=1, q_heads=8, table_width=4, window=0, scale=0.125)
    v.update(other)
    return lib.fp4b_decode_attention(fp4_decode._DECODE.pack(*v.values()), None)


def test_bad_attention_calls_are_refused():
    for other in (dict(batch=-1), dict(q_heads=0), dict(q_heads=7), dict(q=0), dict(out=0), dict(seq_lens=0), dict(page_table=0),
                  dict(table_width=-1), dict(table_stride=3), dict(table_width=1 << 28, table_stride=1 << 28), dict(window=-1),
                  dict(scale=float("inf")), dict(scale=float("nan")), dict(q=0x10004), dict(q_sb=511), dict(out=0x40008), dict(workspace=0),
                  dict(workspace=0x50004), dict(batch=1 << 30, q_heads=1 << 20),
                  dict(batch=1 << 20, table_width=1 << 22, table_stride=1 << 22)):
        assert decode_call(**other) == -1, other
        assert "fp4b_decode_attention" in last()
    assert lib.fp4b_decode_attention(None, None) == -1
    assert decode_call(batch=0) == 0
    assert lib.fp4b_decode_attention_workspace(7, 2, 64) == -1


def test_bad_gemv_calls_are_refused():
    assert lib.fp4b_gemv_cached(0x10000, 1, 128, 128, None, 128, 0x20000, 128, None, None, 0, None) == -1
    assert "cache handle" in last()
    for bad in ((0, 128, 128), (1, 0, 128), (1, 128, 0)):
        assert lib.fp4b_gemv_workspace(*bad) == -1
    # x of one to a few rows fits a CTA; a large one is cut into slices, whose sums take 4 bytes each
    assert lib.fp4b_gemv_workspace(1, 2880, 2880) == 0 and lib.fp4b_gemv_workspace(8, 2880, 15360) == 0
    slices, rest = divmod(lib.fp4b_gemv_workspace(16, 16384, 16384), 16 * 16384 * 4)
    assert rest == 0 and 8 <= slices <= 148  # 64 KB of x at most in a CTA, one CTA an SM
    for m in (1, 3, 8, 9, 16, 40):
        for k in (100, 3000, 9000, 20000):
            for n in (1, 500, 4000, 20000):
                need, tile = lib.fp4b_gemv_workspace(m, k, n), 8 if m <= 8 else 16
                assert need % (-(-m // tile) * tile * (-(-n // 128) * 128) * 4) == 0


def test_python_checks_without_a_gpu():
    x = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        fp4_decode.qk_norm_rope(x, x, None, None)
    with pytest.raises(ValueError, match="dtype must be one of"):
        fp4_decode.PagedKVCache(1, 16, 2, 64, "int4", device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        fp4_decode.PagedKVCache(1, 16, 2, 64, "bf16", device="cpu")
    for bad in ((0, 64), (8, 0), (8, 12)):
        with pytest.raises(ValueError):
            fp4_decode.rope_table(*bad, device="cpu")


def test_rope_table_on_the_cpu():
    import math
    table = fp4_decode.rope_table(70, 24, base=1000.0, device="cpu")
    assert table.shape == (70, 24) and table.dtype == torch.float32
    for p in (0, 1, 69):
        for i in range(12):
            a = p * 1000.0 ** (-2 * i / 24)
            assert abs(table[p, i].item() - math.cos(a)) < 2.0 ** -24 and abs(table[p, 12 + i].item() - math.sin(a)) < 2.0 ** -24
