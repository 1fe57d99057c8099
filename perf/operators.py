"""The decode-side operators' workloads: the matrix-vector product on a cached NVFP4 weight, the norm and rotation of queries and
keys, the paged key-value cache as it is written and read back, and the attention of one new token over it.

`run` computes them in plain torch operations in 32 bits (`own` False) or by the framework's calls (`own` True)."""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6
FP8_FLOOR = 2.0 ** -100  # smallest absmax of an fp8 row's scale


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp4-gemm-blackwell_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import fp4_decode
    import fp4_gemm
    return fp4_gemm, fp4_decode


# ---------------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # One sequence's next token through a square projection (the 2880-wide linears): all latency.
        {"name": "gemv 1 x 2880 x 2880", "op": "gemv", "m": 1, "n": 2880, "k": 2880, "bias": False},
        # Five sequences through the widest linear of the decoder stack (gate_up 2880 -> 15360), with its bias.
        {"name": "gemv 5 x 15360 x 2880", "op": "gemv", "m": 5, "n": 15360, "k": 2880, "bias": True},
        # A full small batch on the largest square weight of the benchmarks.
        {"name": "gemv 16 x 16384 x 16384", "op": "gemv", "m": 16, "n": 16384, "k": 16384, "bias": False},
        # One token's heads out of a 5120-wide QKV row (64 + 8 + 8 heads of 64).
        {"name": "norm rope 1 x (64+8) x 64", "op": "norm_rope", "t": 1, "hq": 64, "hk": 8, "d": 64, "rot": 64, "norm": True, "pairs": False},
        # The decoder stack's 8192-token prompt.
        {"name": "norm rope 8192 x (64+8) x 64", "op": "norm_rope", "t": 8192, "hq": 64, "hk": 8, "d": 64, "rot": 64, "norm": True, "pairs": False},
        # A batch's new tokens normed, rotated and written in one pass, and the written rows read back.
        {"name": "append qkv fp8 33 x 8 x 64", "op": "append_qkv", "t": 33, "hq": 64, "hk": 8, "d": 64, "kind": "fp8", "page": 16},
        # A ragged prompt chunk written to the cache in 4 bits and read back for the prompt's own attention.
        {"name": "append nvfp4 4099 x 8 x 128", "op": "append", "t": 4099, "hk": 8, "d": 128, "kind": "nvfp4", "page": 32},
        # A long cached prefix read back in BF16.
        {"name": "read nvfp4 131072 x 8 x 64", "op": "read", "t": 131072, "hk": 8, "d": 64, "kind": "nvfp4", "page": 64},
        # One short sequence: latency.
        {"name": "attention nvfp4 1 x 77", "op": "attention", "b": 1, "len": 77, "ragged": False, "hq": 64, "hk": 8, "d": 64, "kind": "nvfp4",
         "page": 16, "window": 0, "sinks": False, "lse": False},
        # A serving batch of uneven lengths (some of zero), heads of 128 in groups of four.
        {"name": "attention fp8 33 x 8000", "op": "attention", "b": 33, "len": 8000, "ragged": True, "hq": 32, "hk": 8, "d": 128, "kind": "fp8",
         "page": 32, "window": 0, "sinks": False, "lse": True},
        # A few long contexts in 4 bits, with learned sinks.
        {"name": "attention nvfp4 3 x 131072", "op": "attention", "b": 3, "len": 131072, "ragged": False, "hq": 64, "hk": 8, "d": 64, "kind": "nvfp4",
         "page": 64, "window": 0, "sinks": True, "lse": False},
        # Unquantized cache, a key head for every query head, wide heads.
        {"name": "attention bf16 8 x 4095", "op": "attention", "b": 8, "len": 4095, "ragged": True, "hq": 16, "hk": 16, "d": 256, "kind": "bf16",
         "page": 16, "window": 0, "sinks": False, "lse": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    op = rng.choice(["gemv", "gemv", "norm_rope", "append_qkv", "append", "read", "attention", "attention", "attention", "attention"])
    kind, page = rng.choice(["nvfp4", "fp8", "bf16"]), rng.choice([1, 16, 32, 64, 128])
    hk, d = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 256])
    hq = hk * rng.choice([1, 2, 4, 5, 8, 12, 16])
    if op == "gemv":
        return {"op": op, "m": _log(rng, 1, 16), "n": _log(rng, 64, 16384), "k": _log(rng, 64, 16384), "bias": rng.random() < 0.5}
    if op == "norm_rope":
        return {"op": op, "t": _log(rng, 1, 8192), "hq": hq, "hk": hk, "d": d, "rot": rng.choice([d, d, d // 2]), "norm": rng.random() < 0.8,
                "pairs": rng.random() < 0.3}
    if op == "append_qkv":
        return {"op": op, "t": _log(rng, 1, 8192), "hq": hq, "hk": hk, "d": d, "kind": rng.choice(["fp8", "bf16"]), "page": page}
    if op in ("append", "read"):
        return {"op": op, "t": _log(rng, 1, 131072), "hk": hk, "d": d, "kind": kind, "page": page}
    return {"op": op, "b": _log(rng, 1, 64), "len": _log(rng, 1, 131072), "ragged": rng.random() < 0.6, "hq": hq, "hk": hk, "d": d, "kind": kind,
            "page": page, "window": rng.choice([0, 0, 128, 4095]), "sinks": rng.random() < 0.3, "lse": rng.random() < 0.3}


def _cost(case):
    """What the plain form moves, roughly: drawn cases stay within the listed ones' largest."""
    if case["op"] == "attention":
        return 14.0 * case["b"] * case["len"] * case["hk"] * case["d"]
    if case["op"] == "gemv":
        return 8.0 * case["n"] * case["k"]
    return 24.0 * case["t"] * (case["hk"] + case.get("hq", 0)) * case["d"]


def draw(rng):
    most = max(_cost(c) for c in listed())
    top = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        case = _drawn(rng)
        w = work(case)
        if _cost(case) <= most and w["bytes"] <= top["bytes"] and w["flops"] <= top["flops"]:
            return case


# ---------------------------------------------------------------------------------------------------------------- their work

def _cell(kind, d):
    """Bytes of one (token, head) row of the cache."""
    return {"bf16": 2 * d, "fp8": d + 4, "nvfp4": d // 2 + d // 16}[kind]


def _lengths(case):
    """The sequences' lengths, known from the case alone: even ones, or spread over (0, len] with every eighth empty."""
    if not case["ragged"]:
        return [case["len"]] * case["b"]
    return [0 if i % 8 == 7 else max(1, case["len"] * ((i * 7919 + 4001) % 9973) // 9973) if i else case["len"] for i in range(case["b"])]


def work(case):
    op = case["op"]
    if op == "gemv":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k * 9 / 16 + 2 * m * k + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2.0 * m * n * k}
    if op == "attention":
        keys = sum(min(x, case["window"] or x) for x in _lengths(case))
        return {"bytes": keys * case["hk"] * 2.0 * _cell(case["kind"], case["d"]) + 4 * case["b"] * case["hq"] * case["d"],
                "flops": 4.0 * keys * case["hq"] * case["d"]}
    t, hk, d = case["t"], case["hk"], case["d"]
    if op == "norm_rope":
        n = t * (case["hq"] + hk) * d
        return {"bytes": 4.0 * n + 4 * t * case["rot"] + 8 * t, "flops": 8.0 * n}
    cells = t * hk * 2.0 * _cell(case["kind"], d)
    if op == "read":
        return {"bytes": cells + 4.0 * t * hk * d + 8 * t, "flops": 2.0 * t * hk * d}
    if op == "append":  # written, and read back
        return {"bytes": 8.0 * t * hk * d + 2 * cells + 8 * t, "flops": 10.0 * t * hk * d}
    return {"bytes": 4.0 * t * case["hq"] * d + 8.0 * t * hk * d + 2 * cells + 4 * t * d + 16 * t, "flops": 8.0 * t * (case["hq"] + 2 * hk) * d}


# ---------------------------------------------------------------------------------------------------------------- the codecs

def _ue4m3_value(code):
    c = code.to(torch.int32)
    e, m = (c >> 3) & 15, (c & 7).float()
    return torch.where(e == 0, m * 2.0 ** -9, torch.ldexp(m + 8.0, e - 10))


def _e2m1_value(code):
    """Values of 4-bit codes (sign in bit 3)."""
    c = code.to(torch.int32)
    h = c & 7
    mag = torch.where(h < 2, h * 0.5, torch.ldexp(1.0 + 0.5 * (h & 1), (h >> 1) - 1))
    return torch.where(c > 7, -mag, mag)


def _nvfp4_encode(x):
    """x [..., D] -> codes [..., D / 2] (even element in the low nibble) and scale bytes [..., D / 16]."""
    x = x.float()
    b = x.reshape(*x.shape[:-1], -1, 16)
    amax = b.abs().amax(-1)
    s = (amax / torch.full_like(amax, 6.0)).clamp(2.0 ** -9, 480.0)
    u = s.view(torch.int32)
    e, m = (u >> 23) - 127 + 7, u & 0x7FFFFF
    low = ((m | 0x800000) >> (21 - e.clamp(-2, 0))).clamp(max=7)
    byte = torch.where(e <= 0, low, torch.where(e >= 15, torch.full_like(e, 127), e * 8 + ((m + (1 << 19)) >> 20)))
    v = b * (1.0 / _ue4m3_value(byte)).unsqueeze(-1)
    a = v.abs()
    one = torch.ones((), dtype=torch.uint8, device=x.device)
    # the levels below |v|, by the midpoints between them: a tie keeps the lower magnitude
    code = (a > 0.25) * one + (a > 0.75) + (a > 1.25) + (a > 1.75) + (a > 2.5) + (a > 3.5) + (a > 5.0)
    code = (code + 8 * one * (v < 0)).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte.to(torch.uint8)


def _nvfp4_decode(codes, scales):
    v = torch.stack((_e2m1_value(codes & 15), _e2m1_value(codes >> 4)), -1)
    v = v.reshape(*codes.shape[:-1], -1, 16) * _ue4m3_value(scales).unsqueeze(-1)
    return v.reshape(*codes.shape[:-1], -1)


def _fp8_encode(x):
    x = x.float()
    amax = x.abs().amax(-1).clamp(min=FP8_FLOOR)
    top = torch.full_like(amax, 448.0)
    return (x * (top / amax).unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), amax / top


def _encode(x, kind):
    if kind == "bf16":
        return x.to(torch.bfloat16), None
    return _fp8_encode(x) if kind == "fp8" else _nvfp4_encode(x)


def _decode(codes, scales, kind):
    if kind == "bf16":
        return codes.float()
    if kind == "fp8":
        return codes.float() * scales.unsqueeze(-1)
    return _nvfp4_decode(codes, scales)


def _sf_index(rows, blocks, device):
    """Byte offset of each (row, block)'s scale in a weight cache: atoms of 128 rows x 4 blocks."""
    r = torch.arange(rows, device=device).unsqueeze(1)
    kb = torch.arange(blocks, device=device).unsqueeze(0)
    return (r % 32) * 16 + (r // 32 % 4) * 4 + kb % 4 + (kb // 4) * 512 + (r // 128) * 128 * blocks


# ---------------------------------------------------------------------------------------------------------------- the inputs

def _rope_table(rows, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    a = torch.arange(rows, device=DEV, dtype=torch.float64).unsqueeze(1) * inv
    return torch.cat((a.cos(), a.sin()), -1).float()


def _pages(case, pages, g):
    """Page arrays of a used cache: keys and values of every slot, as written by earlier steps."""
    hk, d, page, kind = case["hk"], case["d"], case["page"], case["kind"]
    made = {}
    for name, spread in (("k", 1.5), ("v", 1.0)):
        x = torch.randn(pages, hk, page, d, generator=g, device=DEV, dtype=torch.bfloat16) * spread
        made[name + "_pages"], made[name + "_scales"] = _encode(x, kind)
    return made


def _cache_handle(s, case):
    if own:
        _, fd = _framework()
        s["cache"] = fd.PagedKVCache.wrap(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    op, s = case["op"], {"case": case}

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    if op == "gemv":
        m, n, k = case["m"], case["n"], case["k"]
        np_, kp = -(-n // 128) * 128, -(-k // 128) * 128
        w = torch.zeros(np_, kp, device=DEV)
        # N(0, 0.02) weights, times the power of two that puts the largest block scale below 480 (two-level NVFP4)
        w[:n, :k] = randn(n, k).float() * 0.02
        two = math.floor(math.log2(6.0 * 480.0 / (0.02 * 6.0)))
        codes, scales = _nvfp4_encode(w * 2.0 ** two)
        sf = torch.empty(np_ * kp // 16, dtype=torch.uint8, device=DEV)
        sf[_sf_index(np_, kp // 16, DEV)] = scales
        s.update(x=randn(m, k), codes=codes, sf=sf, alpha=2.0 ** -two, bias=randn(n) * 0.01 if case["bias"] else None)
        if own:
            fg, _ = _framework()
            s["cache"] = fg.FP4WeightCache.from_state_dict({"fp4": codes, "sf": sf, "N_orig": n, "K_orig": k, "bias": s["bias"], "global_scale": 2.0 ** two})
        return s
    if op == "attention":
        b, page, lens = case["b"], case["page"], _lengths(case)
        wide = max(1, -(-case["len"] // page))
        need = [-(-x // page) for x in lens]
        pages = max(1, sum(need))
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        needed = (seq_lens + page - 1) // page
        at = torch.arange(wide, device=DEV).unsqueeze(0)
        first = (needed.cumsum(0) - needed).unsqueeze(1)
        table = torch.where(at < needed.unsqueeze(1), order[(first + at).clamp(max=pages - 1)], torch.full((), -1, dtype=torch.int32, device=DEV))
        s.update(_pages(case, pages, g), table=table.contiguous(), lens=seq_lens, q=randn(b, case["hq"], case["d"]) * 1.5,
                 sinks=randn(case["hq"], dtype=torch.float32) if case["sinks"] else None)
        _cache_handle(s, case)
        return s
    t, hk, d = case["t"], case["hk"], case["d"]
    if op in ("norm_rope", "append_qkv"):
        hq, rot = case["hq"], case.get("rot", d)
        s["qkv"] = randn(t, (hq + 2 * hk) * d) * 2.0
        s["rope"] = _rope_table(32768, rot)
        s["positions"] = torch.randint(0, 32768 - t, (1,), generator=g, device=DEV) + torch.arange(t, device=DEV)
        norm = case.get("norm", True)
        s["q_weight"], s["k_weight"] = ((1.0 + 0.1 * randn(d, dtype=torch.float32)).to(torch.bfloat16) if norm else None for _ in range(2))
    if op == "append":
        s["k"], s["v"] = randn(t, hk, d) * 1.5, randn(t, hk, d)
    if op != "norm_rope":
        page = case["page"]
        pages = -(-t // page) + 3
        order = torch.randperm(pages, generator=g, device=DEV)
        at = torch.arange(t, device=DEV) + int(seed) % page  # the sequence's first free slot lies inside a page
        s["slots"] = order[at // page] * page + at % page
        s.update(_pages(case, pages, g))
        _cache_handle(s, case)
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass

def _heads(qkv, hq, hk, d):
    q, k, v = qkv[:, : hq * d], qkv[:, hq * d: (hq + hk) * d], qkv[:, (hq + hk) * d: (hq + 2 * hk) * d]
    return q.unflatten(1, (hq, d)), k.unflatten(1, (hk, d)), v.unflatten(1, (hk, d))


def _norm_rope(x, weight, rows, pairs):
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()
    h = rows.shape[1] // 2
    c, s = rows[:, None, :h], rows[:, None, h:]
    if pairs:
        a, b = x[..., 0: 2 * h: 2], x[..., 1: 2 * h: 2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h: 2 * h]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((turned, x[..., 2 * h:]), -1)


def _write(s, name, x, page, slot):
    codes, scales = _encode(x, s["case"]["kind"])
    s[name + "_pages"][page, :, slot] = codes
    if scales is not None:
        s[name + "_scales"][page, :, slot] = scales


def _rows(s, name, page, slot):
    scales = s[name + "_scales"]
    return _decode(s[name + "_pages"][page, :, slot], None if scales is None else scales[page, :, slot], s["case"]["kind"])


def _plain_cache(s, op):
    case, out = s["case"], {}
    page, slot = s["slots"] // case["page"], s["slots"] % case["page"]
    if op == "append_qkv":
        q, k, v = _heads(s["qkv"], case["hq"], case["hk"], case["d"])
        rows = s["rope"][s["positions"]]
        out["q"] = _norm_rope(q, s["q_weight"], rows, False).to(torch.bfloat16)
        k, v = _norm_rope(k, s["k_weight"], rows, False), v
    elif op == "append":
        k, v = s["k"], s["v"]
    if op != "read":
        _write(s, "k", k, page, slot)
        _write(s, "v", v, page, slot)
    out["k"], out["v"] = (_rows(s, n, page, slot).to(torch.bfloat16) for n in ("k", "v"))
    return out


def _plain_attention(s):
    case = s["case"]
    b, hk, d, page = case["b"], case["hk"], case["d"], case["page"]
    n = case["len"]
    at = torch.arange(n, device=DEV)
    pages = s["table"].long()[:, at // page].clamp(min=0)  # [b, n]
    slot = (at % page).expand(b, n)
    k, v = (_rows(s, name, pages, slot) for name in ("k", "v"))  # [b, n, hk, d]
    lens = s["lens"].unsqueeze(1)
    seen = at < lens
    if case["window"]:
        seen = seen & (at >= lens - case["window"])
    q = s["q"].float().reshape(b, hk, -1, d)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * d ** -0.5  # [b, hk, group, n]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if case["sinks"]:
        sink = s["sinks"].float().reshape(1, hk, -1, 1).expand(b, -1, -1, -1)
        top = torch.maximum(top, sink)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    if case["sinks"]:
        total = total + torch.exp(sink - top)
    v = v.masked_fill(~seen[:, :, None, None], 0.0)
    acc = torch.matmul(p, v.permute(0, 2, 1, 3))
    out = torch.where(total > 0, acc / total, torch.zeros_like(acc)).reshape(b, -1, d).to(torch.bfloat16)
    return (out, (top + torch.log(total)).reshape(b, -1)) if case["lse"] else out


def _plain_gemv(s):
    case = s["case"]
    n, k = case["n"], case["k"]
    np_, half = s["codes"].shape
    w = _nvfp4_decode(s["codes"], s["sf"][_sf_index(np_, half // 8, DEV)])[:n, :k]
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    y = torch.matmul(s["x"].float(), w.t()) * s["alpha"]
    torch.backends.cuda.matmul.allow_tf32 = tf32
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(torch.bfloat16)


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        if op == "gemv":
            return _plain_gemv(s)
        if op == "attention":
            return _plain_attention(s)
        if op == "norm_rope":
            q, k, _ = _heads(s["qkv"], case["hq"], case["hk"], case["d"])
            rows = s["rope"][s["positions"]]
            return tuple(_norm_rope(x, w, rows, case["pairs"]).to(torch.bfloat16) for x, w in ((q, s["q_weight"]), (k, s["k_weight"])))
        return _plain_cache(s, op)
    fg, fd = _framework()
    if op == "gemv":
        return fg.fp4_cached_gemv(s["x"], s["cache"])
    if op == "attention":
        return fd.decode_attention(s["q"], s["cache"], s["table"], s["lens"], window=case["window"], sinks=s["sinks"], return_lse=case["lse"])
    if op == "norm_rope":
        q, k, _ = _heads(s["qkv"], case["hq"], case["hk"], case["d"])
        return fd.qk_norm_rope(q, k, s["positions"], s["rope"], s["q_weight"], s["k_weight"], eps=EPS, interleaved=case["pairs"])
    out = {}
    if op == "append":
        s["cache"].append(s["k"], s["v"], s["slots"])
    elif op == "append_qkv":
        q, k, v = _heads(s["qkv"], case["hq"], case["hk"], case["d"])
        out["q"] = s["cache"].append_qkv(q, k, v, s["positions"], s["slots"], s["rope"], s["q_weight"], s["k_weight"], eps=EPS)
    out["k"], out["v"] = s["cache"].read(s["slots"])
    return out


# ---------------------------------------------------------------------------------------------------------------- in 64 bits

def _exact_scale(amax):
    """UE4M3 value nearest to amax / 6 by the quantizer's rule: half up, subnormals truncated, from 256 up the largest."""
    s = (amax.double() / 6.0).clamp(2.0 ** -9, 480.0)
    step = torch.exp2(torch.floor(torch.log2(s))) / 8.0
    normal = torch.floor(s / step + 0.5) * step
    small = torch.floor(s * 512.0).clamp(max=7.0) / 512.0
    return torch.where(s < 2.0 ** -6, small, torch.where(s >= 256.0, torch.full_like(s, 480.0), normal))


def _exact_stored(x, kind):
    """The values that the cache holds after x (64 bits) was written to it."""
    if kind == "bf16":
        return x
    if kind == "fp8":
        amax = x.abs().amax(-1, keepdim=True).clamp(min=FP8_FLOOR)
        scale, v = amax / 448.0, x * (448.0 / amax).float().double()  # the factor is a 32-bit number by definition
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))) / 8.0
        return (torch.round(v / step) * step).clamp(-448.0, 448.0) * scale
    b = x.unflatten(-1, (-1, 16))
    scale = _exact_scale(b.abs().amax(-1, keepdim=True))
    v = b * (1.0 / scale).float().double()  # as in the weight quantizer, the factor is a 32-bit number
    levels = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    edges = (levels[1:] + levels[:-1]) / 2.0
    return (torch.copysign(levels[torch.bucketize(v.abs(), edges)], v) * scale).flatten(-2)  # an edge itself counts to the lower level


def _exact_values(codes, scales, kind):
    """What pages of codes stand for, in 64 bits, by tables of all codes."""
    if kind == "bf16":
        return codes.double()
    if kind == "fp8":
        return codes.double() * scales.double().unsqueeze(-1)
    four = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=codes.device)
    eight = torch.tensor([(c & 7) / 512.0 if c % 128 < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10) for c in range(256)], dtype=torch.float64, device=codes.device)
    v = four[torch.stack((codes % 16, codes // 16), -1).int()].flatten(-2)
    return v * eight[scales.int()].repeat_interleave(16, -1)


def _exact_turned(x, weight, positions, rot, table, pairs):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.double()
    row = table[positions].double().unsqueeze(1)
    z = torch.complex(row[..., : rot // 2], row[..., rot // 2:])
    out = x.clone()
    if pairs:
        turned = torch.view_as_complex(x[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * z
        out[..., 0:rot:2], out[..., 1:rot:2] = turned.real, turned.imag
    else:
        turned = torch.complex(x[..., : rot // 2], x[..., rot // 2: rot]) * z
        out[..., : rot // 2], out[..., rot // 2: rot] = turned.real, turned.imag
    return out


def _exact_attention(s):
    """Sequence by sequence, over its own keys only."""
    case = s["case"]
    hk, d, page, kind = case["hk"], case["d"], case["page"], case["kind"]
    outs, lses = [], []
    for i, n in enumerate(_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        at = torch.arange(first, n, device=DEV)
        pages, slot = s["table"][i].long()[at // page], at % page
        k, v = (_exact_values(s[x + "_pages"][pages, :, slot], None if s[x + "_scales"] is None else s[x + "_scales"][pages, :, slot], kind) for x in ("k", "v"))
        q = s["q"][i].double().reshape(hk, -1, d)
        scores = torch.einsum("hgd,nhd->hgn", q, k) / math.sqrt(d)
        if case["sinks"]:
            sink = s["sinks"].double().reshape(hk, -1, 1)
            scores = torch.cat((scores, sink), -1)
            v = torch.cat((v, torch.zeros(1, hk, d, dtype=torch.float64, device=DEV)), 0)
        if scores.shape[-1]:
            outs.append(torch.einsum("hgn,nhd->hgd", torch.softmax(scores, -1), v).reshape(-1, d))
            lses.append(torch.logsumexp(scores, -1).reshape(-1))
        else:
            outs.append(torch.zeros(case["hq"], d, dtype=torch.float64, device=DEV))
            lses.append(torch.full((case["hq"],), -math.inf, dtype=torch.float64, device=DEV))
    return (torch.stack(outs), torch.stack(lses)) if case["lse"] else torch.stack(outs)


def exact(case, seed):
    global own
    kept, own = own, False
    s = prepare(case, seed)
    own = kept
    op = case["op"]
    if op == "gemv":
        np_, half = s["codes"].shape
        at = torch.arange(np_, device=DEV)[:, None], torch.arange(half // 8, device=DEV)[None]
        atoms = s["sf"].reshape(np_ // 128, half // 32, 32, 4, 4)  # row tile, block / 4, row % 32, row / 32 % 4, block % 4
        scales = atoms[at[0] // 128, at[1] // 4, at[0] % 32, at[0] % 128 // 32, at[1] % 4]
        y = torch.empty(case["m"], case["n"], dtype=torch.float64, device=DEV)
        for r in range(0, case["n"], 2048):
            w = _exact_values(s["codes"][r: r + 2048], scales[r: r + 2048], "nvfp4")
            y[:, r: r + 2048] = (s["x"].double() @ w[: case["n"] - r, : case["k"]].T) * s["alpha"]
        return y if s["bias"] is None else y + s["bias"].double()
    if op == "attention":
        return _exact_attention(s)
    if op == "norm_rope":
        q, k, _ = _heads(s["qkv"], case["hq"], case["hk"], case["d"])
        return tuple(_exact_turned(x, w, s["positions"], case["rot"], s["rope"], case["pairs"]) for x, w in ((q, s["q_weight"]), (k, s["k_weight"])))
    kind, out = case["kind"], {}
    if op == "read":
        page, slot = s["slots"] // case["page"], s["slots"] % case["page"]
        return {x: _exact_values(s[x + "_pages"][page, :, slot], None if s[x + "_scales"] is None else s[x + "_scales"][page, :, slot], kind) for x in ("k", "v")}
    if op == "append":
        k, v = s["k"].double(), s["v"].double()
    else:
        q, k, v = _heads(s["qkv"], case["hq"], case["hk"], case["d"])
        out["q"], k = (_exact_turned(x, w, s["positions"], case["d"], s["rope"], False) for x, w in ((q, s["q_weight"]), (k, s["k_weight"])))
        v = v.double()
    out["k"], out["v"] = _exact_stored(k, kind), _exact_stored(v, kind)
    return out
