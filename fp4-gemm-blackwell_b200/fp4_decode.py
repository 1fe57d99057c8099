"""
The decode side of a decoder layer on B200 (sm_100a), beside the NVFP4 linears of ``fp4_gemm``: what lies between the QKV
linear and the output linear when a model answers token by token.

    rope_table(rows, rot, base)                         cosines and sines of the positions, fp32 [rows, rot]
    qk_norm_rope(q, k, positions, rope, ...)            norms of queries and keys for each head + the rotation, one pass
    PagedKVCache(num_pages, page_size, kv_heads, ...)   keys and values in pages: BF16, fp8 (E4M3) or NVFP4
        .append(k, v, slots)                            quantizes as it writes
        .append_qkv(q, k, v, positions, slots, rope)    norm + rotation + write, one pass; returns the queries
        .read(slots)                                    keys and values back in BF16
    decode_attention(q, cache, page_table, seq_lens)    one new token a sequence, split over the cache's length

(The linears' own form for few rows is ``fp4_gemm.fp4_cached_gemv``.)  Tensors are BF16 on one CUDA device; work is queued
on PyTorch's current stream and nothing synchronises, so a decode step can be captured in a CUDA graph.  Inference only,
like the rest of the library: no gradients.  Slots, positions, page tables and lengths live on the GPU; one out of
range is never followed and shows in ``fp4_gemm.device_error()``: 11 a slot (nothing written, zeros read), 12 a position (no
rotation), 13 a page (its keys count as rows of zeros: score 0, value 0) or a length (clamped to the table's pages).
"""

import ctypes
import struct

import torch

from fp4_gemm import _bind, _f, _i, _last_error, _lib, _on_cleanup, _vp

_l = ctypes.c_long

KV_KINDS = {"bf16": 0, "fp8": 1, "nvfp4": 2}


class _CacheView(ctypes.Structure):
    """fp4b_kv_cache of fp4gemm.h."""

    _fields_ = [("k", _vp), ("v", _vp), ("k_scale", _vp), ("v_scale", _vp), ("num_pages", _i), ("kv_heads", _i),
                ("page_size", _i), ("head_dim", _i), ("kind", _i)]


# fp4b_rows and fp4b_decode, as one call packs them (0: NULL).
_ROWS, _DECODE = struct.Struct("@PllPllPllPPPPPPPPiiiiiiiiif"), struct.Struct("@PllPPlPPPPPliiiif0l")

_bind("fp4b_kv_rows", _i, [ctypes.c_char_p, _vp])
_bind("fp4b_kv_read", _i, [_vp, _vp, _i, _l, _vp, _vp, _vp])
_bind("fp4b_decode_attention_workspace", _l, [_i, _i, _i])
_bind("fp4b_decode_attention", _i, [ctypes.c_char_p, _vp])

_kv_rows, _kv_read, _attention = _lib.fp4b_kv_rows, _lib.fp4b_kv_read, _lib.fp4b_decode_attention


# A call's host time is what a small decode step costs, so the current device and stream are asked for without the
# objects that torch.cuda makes of them.
_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_capturing = torch._C._cuda_isCurrentStreamCapturing


def _call(device, fn, what: str, *args):
    """fn(*args, stream) with `device` current; raises on a failure code."""
    index = device.index
    if index == _current_device():
        rc = fn(*args, _current_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _current_stream(index))
    if rc != 0:
        raise RuntimeError(f"{what} failed with error code {rc} ({_last_error()})")


def _rows(t: torch.Tensor, what: str, device=None) -> torch.Tensor:
    """t [tokens, heads, D] as BF16 rows that a kernel can read in 8-byte pieces (copied only if they are not)."""
    if t.dim() != 3:
        raise ValueError(f"{what} must be [tokens, heads, head_dim], got shape {tuple(t.shape)}")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{what} must be on the CUDA device of the call")
    if t.dtype != torch.bfloat16:
        t = t.to(torch.bfloat16)
    st, sh, se = t.stride()
    if se != 1 or (st | sh) & 3 or t.data_ptr() & 7:
        # a new tensor always: contiguous() keeps one that starts anywhere, and the strides of dimensions of size one
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _indices(t: torch.Tensor, count: int, what: str, device) -> torch.Tensor:
    if t.dtype not in (torch.int64, torch.int32) or t.device != device or t.numel() != count:
        raise ValueError(f"{what} must be {count} int32 or int64 numbers on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def _table(t: torch.Tensor):
    """(t, distance of its rows) of a page table [B, W] as the kernel goes over it, entry i of row b at b * distance + i: copied
    where its rows are not of unit stride, are one row for all (expand) or overlap.  A single row's distance is its length."""
    b, width = t.shape
    if (width > 1 and t.stride(1) != 1) or (b > 1 and t.stride(0) < width):
        t = t.contiguous()
    return t, t.stride(0) if b > 1 else width


def _weight(w, d: int, what: str, device):
    if w is None:
        return None
    if w.numel() != d or w.device != device:
        raise ValueError(f"{what} must have {d} elements on {device}")
    if w.dtype != torch.bfloat16:
        w = w.to(torch.bfloat16)
    w = w if w.is_contiguous() else w.contiguous()
    return w if w.data_ptr() & 7 == 0 else w.clone()


def _address(t) -> int:
    return 0 if t is None else t.data_ptr()


def _rope(rope, d: int, device):
    """(address, rows, rotated size) of a table; zeros for none."""
    if rope is None:
        return 0, 0, 0
    if rope.dim() != 2 or rope.dtype != torch.float32 or rope.device != device or not rope.is_contiguous():
        raise ValueError("rope must be a contiguous fp32 [rows, rot] table on the queries' device (see rope_table)")
    rows, rot = rope.shape
    if rows == 0 or rot == 0 or rot > d or rot % 8:
        raise ValueError(f"the rotated size must be a multiple of 8 up to head_dim {d}, got {rot}")
    return rope.data_ptr(), rows, rot


def rope_table(rows: int, rot: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """fp32 [rows, rot]: of each position p < rows the cosines, then the sines, of p * base^(-2i / rot), i < rot / 2
    (angles in 64 bits, rounded once).  A model with another rule for its frequencies fills a table of its own."""
    if rows <= 0 or rot <= 0 or rot % 8:
        raise ValueError("rows must be positive and rot a positive multiple of 8")
    inv = float(base) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(rows, dtype=torch.float64, device=device).unsqueeze(1) * inv
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rope: torch.Tensor, q_weight: torch.Tensor = None,
                 k_weight: torch.Tensor = None, eps: float = 1e-6, interleaved: bool = False):
    """
    Queries and keys, normed for each head and rotated to their positions.

    q is [T, Hq, D], k [T, Hk, D] (any token and head strides: slices of the QKV linear's output are read in place), D a
    multiple of 32 up to 256; positions [T] int32 or int64; rope a table as of ``rope_table`` with rot <= D (the elements
    from rot up stay) or None.  With a weight [D], each head's x becomes x / sqrt(mean(x^2) + eps) * weight first.  The
    rotation turns the pairs (i, i + rot / 2), or (2i, 2i + 1) with interleaved=True.  All in fp32, rounded once.

    Returns new BF16 tensors ([T, Hq, D], [T, Hk, D]).
    """
    q = _rows(q, "q")
    dev = q.device
    k = _rows(k, "k", dev)
    t, hq, d = q.shape
    hk = k.shape[1]
    if k.shape[0] != t or k.shape[2] != d:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} have other tokens or head sizes")
    table, rows, rot = _rope(rope, d, dev)
    if table:
        positions = _indices(positions, t, "positions", dev)
    q_out, k_out = _like(q), _like(k)
    if t == 0:
        return q_out, k_out
    q_weight, k_weight = _weight(q_weight, d, "q_weight", dev), _weight(k_weight, d, "k_weight", dev)
    qs, ks = q.stride(), k.stride()
    _call(dev, _kv_rows, "qk_norm_rope", _ROWS.pack(
        q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], 0, 0, 0, positions.data_ptr() if table else 0, 0, table,
        _address(q_weight), _address(k_weight), q_out.data_ptr(), k_out.data_ptr(), 0, t, hq, hk, d, rows, rot, interleaved,
        table != 0 and positions.dtype == torch.int64, 0, eps))
    return q_out, k_out


class PagedKVCache:
    """
    Keys and values of many sequences in pages of `page_size` tokens.

    ``k_pages`` / ``v_pages`` are [num_pages, kv_heads, page_size, ...]: BF16 [..., head_dim]; for "fp8"
    torch.float8_e4m3fn [..., head_dim] with one fp32 scale a (token, head) in ``k_scales`` / ``v_scales``
    [num_pages, kv_heads, page_size] (scale = absmax / 448); for "nvfp4" uint8 [..., head_dim / 2], the weight
    quantizer's codes, with UE4M3 bytes [..., head_dim / 16] as scales.  Which page belongs to whom is the caller's
    business: a token's slot number is page * page_size + its place in the page.
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: str = "nvfp4", device="cuda"):
        if dtype not in KV_KINDS:
            raise ValueError(f"dtype must be one of {sorted(KV_KINDS)}, got {dtype!r}")
        if min(num_pages, page_size, kv_heads, head_dim) <= 0:
            raise ValueError("num_pages, page_size, kv_heads and head_dim must be positive")
        shape = (num_pages, kv_heads, page_size)

        def pages():
            if dtype == "nvfp4":
                return (torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device=device),
                        torch.zeros(*shape, head_dim // 16, dtype=torch.uint8, device=device))
            if dtype == "fp8":
                return (torch.zeros(*shape, head_dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
                        torch.zeros(shape, dtype=torch.float32, device=device))
            return torch.zeros(*shape, head_dim, dtype=torch.bfloat16, device=device), None

        k, v = pages(), pages()
        self._adopt(k[0], v[0], k[1], v[1])

    @classmethod
    def wrap(cls, k_pages, v_pages, k_scales=None, v_scales=None) -> "PagedKVCache":
        """A cache on page tensors that the caller owns (laid out as above; nothing is copied)."""
        self = cls.__new__(cls)
        self._adopt(k_pages, v_pages, k_scales, v_scales)
        return self

    def _adopt(self, k_pages, v_pages, k_scales, v_scales):
        kinds = {torch.bfloat16: "bf16", torch.float8_e4m3fn: "fp8", torch.uint8: "nvfp4"}
        if k_pages.dtype not in kinds or k_pages.dim() != 4:
            raise ValueError("pages must be 4-D BF16, float8_e4m3fn or uint8 tensors")
        self.dtype = kinds[k_pages.dtype]
        n, h, s, w = k_pages.shape
        d = w * 2 if self.dtype == "nvfp4" else w
        if d not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {d}")
        if s <= 0 or s & (s - 1) or s > 1024:
            raise ValueError(f"page_size must be a power of two up to 1024, got {s}")
        scales = {"bf16": None, "fp8": ((n, h, s), torch.float32), "nvfp4": ((n, h, s, d // 16), torch.uint8)}[self.dtype]
        if not k_pages.is_cuda:
            raise ValueError("pages must be on a CUDA device")
        for p, sc in ((k_pages, k_scales), (v_pages, v_scales)):
            if p.shape != k_pages.shape or p.dtype != k_pages.dtype or p.device != k_pages.device or not p.is_contiguous():
                raise ValueError("key and value pages must be alike and contiguous")
            if (sc is None) != (scales is None):
                raise ValueError(f"a {self.dtype} cache {'has no' if scales is None else 'needs'} scales")
            if scales and (tuple(sc.shape) != scales[0] or sc.dtype != scales[1] or sc.device != p.device or not sc.is_contiguous()):
                raise ValueError(f"scales must be contiguous {scales[1]} {scales[0]} on {p.device}")
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = n, h, s, d
        self.device = k_pages.device
        self.k_pages, self.v_pages, self.k_scales, self.v_scales = k_pages, v_pages, k_scales, v_scales
        self._view = _CacheView(k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr() if scales else None,
                                v_scales.data_ptr() if scales else None, n, h, s, d, KV_KINDS[self.dtype])
        self._ref = ctypes.addressof(self._view)
        self._bf16 = torch.empty(0, dtype=torch.bfloat16, device=self.device)  # what results are made like
        self._attention_bytes = {}  # query heads -> bytes of decode_attention's workspace

    @property
    def nbytes(self) -> int:
        return sum(t.nbytes for t in (self.k_pages, self.v_pages, self.k_scales, self.v_scales) if t is not None)

    def _kv(self, k, v):
        k, v = _rows(k, "k", self.device), _rows(v, "v", self.device)
        if k.shape != v.shape or k.shape[1] != self.kv_heads or k.shape[2] != self.head_dim:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [tokens, {self.kv_heads}, {self.head_dim}]")
        return k, v

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Write k, v [T, kv_heads, head_dim] to slots [T] (int32 or int64; a negative one skips its token; no slot twice
        in a call), quantized to the cache's format."""
        k, v = self._kv(k, v)
        t = k.shape[0]
        slots = _indices(slots, t, "slots", self.device)
        if t:
            ks, vs = k.stride(), v.stride()
            _call(self.device, _kv_rows, "append", _ROWS.pack(
                0, 0, 0, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], 0, slots.data_ptr(), 0, 0, 0, 0, 0, self._ref, t, 0,
                self.kv_heads, self.head_dim, 0, 0, 0, 0, slots.dtype == torch.int64, 0.0))

    def append_qkv(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                   rope: torch.Tensor, q_weight: torch.Tensor = None, k_weight: torch.Tensor = None, eps: float = 1e-6,
                   interleaved: bool = False) -> torch.Tensor:
        """``qk_norm_rope`` and ``append`` in one pass: returns the queries [T, Hq, head_dim]; the keys go from fp32 straight
        to the cache's format (one rounding), the values as they are."""
        q = _rows(q, "q", self.device)
        k, v = self._kv(k, v)
        t, hq, d = q.shape
        dev = self.device
        if k.shape[0] != t or d != self.head_dim:
            raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} have other tokens or head sizes")
        slots = _indices(slots, t, "slots", dev)
        table, rows, rot = _rope(rope, d, dev)
        if table:
            positions = _indices(positions, t, "positions", dev)
        q_out = _like(q)
        if t == 0:
            return q_out
        q_weight, k_weight = _weight(q_weight, d, "q_weight", dev), _weight(k_weight, d, "k_weight", dev)
        qs, ks, vs = q.stride(), k.stride(), v.stride()
        _call(dev, _kv_rows, "append_qkv", _ROWS.pack(
            q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], positions.data_ptr() if table else 0,
            slots.data_ptr(), table, _address(q_weight), _address(k_weight), q_out.data_ptr(), 0, self._ref, t, hq, self.kv_heads, d,
            rows, rot, interleaved, table != 0 and positions.dtype == torch.int64, slots.dtype == torch.int64, eps))
        return q_out

    def read(self, slots: torch.Tensor):
        """Keys and values of slots [n] as new BF16 tensors [n, kv_heads, head_dim] each; zeros for a negative slot."""
        n = slots.numel()
        slots = _indices(slots, n, "slots", self.device)
        k = self._bf16.new_empty(n, self.kv_heads, self.head_dim)
        v = torch.empty_like(k)
        if n:
            _call(self.device, _kv_read, "read", self._ref, slots.data_ptr(), slots.dtype == torch.int64, n, k.data_ptr(), v.data_ptr())
        return k, v

    def __repr__(self):
        return "PagedKVCache(%d pages x %d tokens, %d heads of %d, %s, %.1f MB)" % (
            self.num_pages, self.page_size, self.kv_heads, self.head_dim, self.dtype, self.nbytes / 2 ** 20)


_WORKSPACES = {}  # (device, stream) -> uint8 tensor whose counters decode_attention leaves zeroed
_COUNTER_BYTES = 16384  # FP4B_DECODE_COUNTER_BYTES


def _workspace(device, need: int) -> torch.Tensor:
    """Workspace of the calls on the current stream, which run in order.  A captured graph gets one of its own, its counters
    zeroed in the graph: it may be replayed on any stream, beside anything."""
    if _capturing():
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        ws[:_COUNTER_BYTES].zero_()
        return ws
    key = (device.index, _current_stream(device.index))
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < need:
        ws = _WORKSPACES[key] = torch.zeros(need, dtype=torch.uint8, device=device)
    return ws


def _drop_workspaces(index: int) -> None:
    for key in [key for key in _WORKSPACES if key[0] == index]:
        del _WORKSPACES[key]  # back to the allocator, which hands it out in the order of its stream


_on_cleanup.append(_drop_workspaces)


def decode_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, seq_lens: torch.Tensor, scale: float = None,
                     window: int = 0, sinks: torch.Tensor = None, return_lse: bool = False):
    """
    Attention of one new token of each sequence over its keys and values in the cache.

    q is [B, Hq, head_dim] BF16, Hq a multiple of the cache's heads (query head h reads key head h // (Hq // kv_heads));
    page_table [B, W] int32, its first ceil(len / page_size) entries the sequence's pages in order (the others, and
    those wholly before the window, are not read); seq_lens [B] int32, the new token's own key included if it is to be
    seen.  scale defaults to head_dim ** -0.5; window > 0 lets a token see its last `window` keys only; sinks [Hq] is one
    more logit of each head's softmax that no value belongs to.  A sequence of length 0 gives zeros.  Sums and statistics
    are fp32; the softmax's weights enter their products with 22 bits over an fp8 or nvfp4 cache, 16 over a BF16 one.

    Returns BF16 [B, Hq, head_dim]; with return_lse=True also fp32 [B, Hq], the natural logarithm of the softmax's
    denominator (-inf where there was nothing), by which results over parts of a context can be joined.
    """
    q = _rows(q, "q", cache.device)
    b, hq, d = q.shape
    dev = cache.device
    if d != cache.head_dim or hq == 0 or hq % cache.kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {cache.kv_heads} heads of {cache.head_dim}")
    if page_table.dim() != 2 or page_table.shape[0] != b or page_table.dtype != torch.int32 or page_table.device != dev:
        raise ValueError(f"page_table must be int32 [{b}, W] on {dev}")
    if seq_lens.dim() != 1 or seq_lens.shape[0] != b or seq_lens.dtype != torch.int32 or seq_lens.device != dev:
        raise ValueError(f"seq_lens must be int32 [{b}] on {dev}")
    if window < 0:
        raise ValueError("window must not be negative")
    page_table, table_stride = _table(page_table)
    if seq_lens.stride(0) != 1:
        seq_lens = seq_lens.contiguous()
    if sinks is not None:
        if sinks.numel() != hq or sinks.device != dev:
            raise ValueError(f"sinks must have {hq} elements on {dev}")
        sinks = sinks.to(torch.float32).contiguous()
    out = _like(q)
    lse = torch.empty((b, hq), dtype=torch.float32, device=dev) if return_lse else None
    if b:
        need = cache._attention_bytes.get(hq)
        if need is None:
            with torch.cuda.device(dev):
                need = cache._attention_bytes[hq] = _lib.fp4b_decode_attention_workspace(hq, cache.kv_heads, d)
        ws = _workspace(dev, need)
        qs = q.stride()
        _call(dev, _attention, "decode_attention", _DECODE.pack(
            q.data_ptr(), qs[0], qs[1], cache._ref, page_table.data_ptr(), table_stride, seq_lens.data_ptr(),
            _address(sinks), out.data_ptr(), _address(lse), ws.data_ptr(), ws.numel(), b, hq, page_table.shape[1], window,
            d ** -0.5 if scale is None else scale))
    return (out, lse) if return_lse else out
