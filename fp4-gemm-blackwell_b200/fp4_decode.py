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
    shared_prefix_attention(q, cache, prefix_table, prefix_lens, page_table, seq_lens)
                                                        the same where sequences share a prefix, read together
    block_norm(x, residual, weight, ...)                norm after a block, gate, residual, norm before the next, one pass
    sample(logits, u, temperature, top_k, top_p, min_p) the next tokens, from given uniform numbers

(The linears' own form for few rows is ``fp4_gemm.fp4_cached_gemv``.)  Tensors are BF16 on one CUDA device; work is queued
on PyTorch's current stream and nothing synchronises, so a decode step can be captured in a CUDA graph.  Inference only,
like the rest of the library: no gradients.  Slots, positions, page tables and lengths live on the GPU; one out of
range is never followed and shows in ``fp4_gemm.device_error()``: 11 a slot (nothing written, zeros read), 12 a position (no
rotation), 13 a page (its keys count as rows of zeros: score 0, value 0) or a length (clamped to the table's pages).  14 there
means that shared_prefix_attention's kernel gave up a wait: its results are not valid.
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


# The arguments of the C entry points, as one call packs them (0: NULL): fp4b_rows and fp4b_decode,
_ROWS, _DECODE = struct.Struct("@PllPllPllPPPPPPPPiiiiiiiiif"), struct.Struct("@PllPPlPPPPPliiiif0l")
_SHARED = struct.Struct(_DECODE.format.replace("0l", "") + "PlPii0l")  # fp4b_shared: an fp4b_decode, then the prefixes
_NORM, _SAMPLING = struct.Struct("@PlPlPlPPPPiiiff0l"), struct.Struct("@PlPPPPPPPiiififf0l")  # fp4b_norm, fp4b_sampling

_bind("fp4b_kv_rows", _i, [ctypes.c_char_p, _vp])
_bind("fp4b_kv_read", _i, [_vp, _vp, _i, _l, _vp, _vp, _vp])
_bind("fp4b_decode_attention_workspace", _l, [_i, _i, _i])
_bind("fp4b_decode_attention", _i, [ctypes.c_char_p, _vp])
_bind("fp4b_shared_attention_workspace", _l, [_i, _i, _i, _i, _i])
_bind("fp4b_shared_attention", _i, [ctypes.c_char_p, _vp])
_bind("fp4b_block_norm", _i, [ctypes.c_char_p, _vp])
_bind("fp4b_sample", _i, [ctypes.c_char_p, _vp])

_kv_rows, _kv_read, _attention = _lib.fp4b_kv_rows, _lib.fp4b_kv_read, _lib.fp4b_decode_attention
_shared_attention, _block_norm, _sample = _lib.fp4b_shared_attention, _lib.fp4b_block_norm, _lib.fp4b_sample


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


def _pages(table, lens, b: int, table_name: str, lens_name: str, device):
    """(page table, distance of its rows, lengths) of b sequences, as the kernels read them."""
    if table.dim() != 2 or table.shape[0] != b or table.dtype != torch.int32 or table.device != device:
        raise ValueError(f"{table_name} must be int32 [{b}, W] on {device}")
    if lens.dim() != 1 or lens.shape[0] != b or lens.dtype != torch.int32 or lens.device != device:
        raise ValueError(f"{lens_name} must be int32 [{b}] on {device}")
    table, stride = _table(table)
    return table, stride, lens if lens.stride(0) == 1 else lens.contiguous()


def _sinks(sinks, hq: int, device):
    if sinks is None:
        return None
    if sinks.numel() != hq or sinks.device != device:
        raise ValueError(f"sinks must have {hq} elements on {device}")
    return sinks.to(torch.float32).contiguous()


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
    page_table, table_stride, seq_lens = _pages(page_table, seq_lens, b, "page_table", "seq_lens", dev)
    if window < 0:
        raise ValueError("window must not be negative")
    sinks = _sinks(sinks, hq, dev)
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


def shared_prefix_attention(q: torch.Tensor, cache: PagedKVCache, prefix_table: torch.Tensor, prefix_lens: torch.Tensor, page_table: torch.Tensor,
                            seq_lens: torch.Tensor, scale: float = None, sinks: torch.Tensor = None, return_lse: bool = False):
    """
    ``decode_attention`` of sequences that share prefixes: one system prompt before all, or several answers to each prompt.

    Each of the G prefixes is read once for every 128 of its rows (its sequences times a key head's query heads) instead of
    once a sequence: prefix_table [G, W0] int32 and prefix_lens [G] int32 hold its pages and length, and sequence b of q's B
    (a multiple of G) belongs to prefix b // (B // G).  page_table [B, W] and seq_lens [B] are the sequence's own keys behind
    the prefix, on pages of their own from their first on; either length may be 0.  One softmax goes over both.  q, scale,
    sinks, the result and its precision as in ``decode_attention`` (no window).

    It pays from a few sequences a prefix on; decode_attention over tables that repeat the prefix's pages gives the same.
    """
    q = _rows(q, "q", cache.device)
    b, hq, d = q.shape
    dev = cache.device
    if d != cache.head_dim or hq == 0 or hq % cache.kv_heads:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {cache.kv_heads} heads of {cache.head_dim}")
    groups = prefix_lens.shape[0] if prefix_lens.dim() == 1 else 0
    if groups == 0 or b % groups:
        raise ValueError(f"prefix_lens must be int32 [G] with {b} sequences a multiple of G, got {tuple(prefix_lens.shape)}")
    prefix_table, prefix_stride, prefix_lens = _pages(prefix_table, prefix_lens, groups, "prefix_table", "prefix_lens", dev)
    page_table, table_stride, seq_lens = _pages(page_table, seq_lens, b, "page_table", "seq_lens", dev)
    sinks = _sinks(sinks, hq, dev)
    out = _like(q)
    lse = torch.empty((b, hq), dtype=torch.float32, device=dev) if return_lse else None
    if b:
        need = cache._attention_bytes.get((groups, b, hq))
        if need is None:
            with torch.cuda.device(dev):
                need = cache._attention_bytes[groups, b, hq] = _lib.fp4b_shared_attention_workspace(groups, b, hq, cache.kv_heads, d)
        ws = _workspace(dev, need)
        qs = q.stride()
        _call(dev, _shared_attention, "shared_prefix_attention", _SHARED.pack(
            q.data_ptr(), qs[0], qs[1], cache._ref, page_table.data_ptr(), table_stride, seq_lens.data_ptr(),
            _address(sinks), out.data_ptr(), _address(lse), ws.data_ptr(), ws.numel(), b, hq, page_table.shape[1], 0,
            d ** -0.5 if scale is None else scale, prefix_table.data_ptr(), prefix_stride, prefix_lens.data_ptr(), groups, prefix_table.shape[1]))
    return (out, lse) if return_lse else out


def _wide(t: torch.Tensor, what: str, index: int):
    """(t, row stride) of BF16 rows [..., H] as [rows, H] with elements in one run (cast or copied only if they are not)."""
    if t.get_device() != index:
        raise ValueError(f"{what} must be on cuda:{index}, got {t.device}")
    if t.dtype is not torch.bfloat16:
        t = t.to(torch.bfloat16)
    return (t, t.shape[-1]) if t.is_contiguous() else _strided(t)


def _strided(t: torch.Tensor):
    t = t.reshape(-1, t.shape[-1])
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _vector(t, h: int, what: str, index: int):
    """A weight [H] in BF16, its elements in one run."""
    if t.numel() != h or t.get_device() != index:
        raise ValueError(f"{what} must have {h} elements on cuda:{index}")
    if t.dtype is not torch.bfloat16:
        t = t.to(torch.bfloat16)
    return t if t.is_contiguous() else t.contiguous()


def block_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, post_weight: torch.Tensor = None, gate: torch.Tensor = None,
               scale: float = 1.0, eps: float = 1e-6):
    """
    What lies between two blocks: the norm after a block, its gate, its residual and the norm before the next block, in one pass.

    With x [..., H] the block's output and residual [..., H] what it is added to:

        y = x / sqrt(mean(x^2) + eps) * post_weight     (without post_weight: y = x)
        r = residual + scale * gate * y                 (without gate: 1)
        normed = r / sqrt(mean(r^2) + eps) * weight

    x is BF16, residual BF16 or fp32 (a residual stream in 32 bits), gate [H] (each channel's) or of x's shape, the weights
    [H], all BF16 (other types are cast).  Rows may have any stride.  In fp32 throughout: normed is made from r as it is before
    its rounding.  x None: normed of the residual alone (before the first block).  H up to 32768.

    Returns new tensors (normed, r): normed BF16, r of residual's type (residual itself where x is None).
    """
    index, shape = residual.get_device(), residual.shape
    if index < 0:
        raise ValueError("residual must be on a CUDA device")
    h = shape[-1] if len(shape) else 0
    if not 0 < h <= 32768:
        raise ValueError(f"rows must have 1 to 32768 elements, got shape {tuple(shape)}")
    fp32 = residual.dtype is torch.float32
    if not fp32 and residual.dtype is not torch.bfloat16:
        residual = residual.to(torch.bfloat16)
    r_rows, r_stride = (residual, h) if residual.is_contiguous() else _strided(residual)
    weight = _vector(weight, h, "weight", index)
    normed = weight.new_empty(shape)
    out = residual
    x_at = x_stride = gate_at = gate_stride = post_at = 0
    if x is not None:
        if x.shape != shape:
            raise ValueError(f"x {tuple(x.shape)} and residual {tuple(shape)} have other shapes")
        x, x_stride = _wide(x, "x", index)
        x_at = x.data_ptr()
        if post_weight is not None:
            post_weight = _vector(post_weight, h, "post_weight", index)
            post_at = post_weight.data_ptr()
        if gate is not None:
            if gate.dim() == 1 and gate.shape[0] == h:
                gate = _vector(gate, h, "gate", index)
            elif gate.shape == shape:
                gate, gate_stride = _wide(gate, "gate", index)
            else:
                raise ValueError(f"gate must be [{h}] or {tuple(shape)}, got {tuple(gate.shape)}")
            gate_at = gate.data_ptr()
        out = residual.new_empty(shape)
    elif post_weight is not None or gate is not None:
        raise ValueError("post_weight and gate belong to a block's output: x is None")
    rows = normed.numel() // h
    if rows:
        _call(normed.device, _block_norm, "block_norm", _NORM.pack(
            x_at, x_stride, r_rows.data_ptr(), r_stride, gate_at, gate_stride, weight.data_ptr(), post_at, normed.data_ptr(),
            out.data_ptr() if x_at else 0, rows, h, fp32, scale, eps))
    return normed, out


_LOGITS = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}  # FP4B_LOGITS_*


def _setting(v, rows: int, dtype, what: str, index: int):
    """(address, number, tensor to keep) of a setting: one number for all rows, or a tensor [rows]."""
    if not isinstance(v, torch.Tensor):
        return 0, v, None
    if v.get_device() != index or v.numel() != rows:
        raise ValueError(f"{what} must be a number or {rows} numbers on cuda:{index}, got {tuple(v.shape)} on {v.device}")
    if v.dtype is not dtype:
        if v.dtype is torch.int64 and dtype is torch.int32:
            v = v.clamp(-1 << 31, (1 << 31) - 1)  # (a cast alone keeps the low 32 bits)
        v = v.to(dtype)
    if not v.is_contiguous():
        v = v.contiguous()
    return v.data_ptr(), 0, v


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_prob: bool = False):
    """
    The next token of each row of logits, by temperature, top-k, top-p and min-p, from given uniform numbers.

    logits is [B, V] BF16, FP16 or fp32, rows of any stride; u [B] fp32 in [0, 1) (numbers outside count as the nearest of
    these).  Each setting is a number or a tensor [B] (top_k int32, the others fp32).  The tokens of a row are taken by logit,
    largest first, equal ones by index, with w = exp((logit - max) / temperature); -inf (a masked token) and NaN are no
    candidates.  Kept are

        the first top_k                                        (0 or less: all),
        of those the ones before which less than top_p of their weights' sum lies   (1 or more: all; the first always),
        of those the ones with w >= min_p                      (0 or less: all; the first always),

    and the token is the first with which more than u of the kept ones' sum is reached.  A temperature of 0 gives the largest
    logit's first index.  Weights are whole multiples of 2^-44 of the largest (vocabularies up to 2^18; one bit less for each
    doubling) and their sums exact, so the same call gives the same tokens.

    Returns int64 [B], -1 for a row without candidates; with return_prob=True also fp32 [B], the share of the kept ones' sum
    that the token has (1 at temperature 0, 0 where there is none).
    """
    kind = _LOGITS.get(logits.dtype)
    if kind is None or logits.dim() != 2:
        raise ValueError(f"logits must be [B, V] BF16, FP16 or fp32, got {logits.dtype} {tuple(logits.shape)}")
    index = logits.get_device()
    if index < 0:
        raise ValueError("logits must be on a CUDA device")
    b, v = logits.shape
    if v == 0 or v > 1 << 30:
        raise ValueError(f"the vocabulary must be 1 to 2^30 tokens, got {v}")
    if u.dtype is not torch.float32 or u.get_device() != index or u.numel() != b:
        raise ValueError(f"u must be {b} fp32 numbers on cuda:{index}, got {u.dtype} {tuple(u.shape)} on {u.device}")
    if not u.is_contiguous():
        u = u.contiguous()
    stride, step = logits.stride()
    if step != 1 and v > 1:
        logits, stride = logits.contiguous(), v
    t_at, t_one, t_keep = _setting(temperature, b, torch.float32, "temperature", index)
    k_at, k_one, k_keep = _setting(top_k, b, torch.int32, "top_k", index)
    p_at, p_one, p_keep = _setting(top_p, b, torch.float32, "top_p", index)
    m_at, m_one, m_keep = _setting(min_p, b, torch.float32, "min_p", index)
    if t_at == 0 and not t_one >= 0.0:
        raise ValueError(f"temperature must not be negative, got {t_one}")
    tokens = u.new_empty(b, dtype=torch.int64)
    probs = u.new_empty(b) if return_prob else None
    if b:
        _call(tokens.device, _sample, "sample", _SAMPLING.pack(
            logits.data_ptr(), stride, u.data_ptr(), t_at, k_at, p_at, m_at, tokens.data_ptr(), probs.data_ptr() if return_prob else 0, b, v,
            kind, t_one, min(max(int(k_one), 0), v), p_one, m_one))
    return (tokens, probs) if return_prob else tokens
