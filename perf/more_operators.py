"""Workloads of the operators that close a decoding step: the attention of a batch over a prefix that its sequences share, the norms
around a block with its gate and residual, and the choice of the next tokens.

`run` computes them in plain torch operations (`own` False) or by the framework's calls (`own` True)."""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6
FP8_FLOOR = 2.0 ** -100  # smallest absmax of an fp8 row's scale
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LOGITS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _framework():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp4-gemm-blackwell_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import fp4_decode
    return fp4_decode


# ---------------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # Two answers to one short prompt, a few tokens in: all latency.
        {"name": "shared bf16 2 x 500 + 30", "op": "shared", "prefixes": 1, "each": 2, "prefix": 500, "length": 30, "hq": 64, "hk": 8, "d": 64,
         "kind": "bf16", "page": 16, "sinks": False, "lse": False},
        # A serving batch behind one long system prompt in 4 bits, each sequence with a turn or two of its own.
        {"name": "shared nvfp4 32 x 32768 + 512", "op": "shared", "prefixes": 1, "each": 32, "prefix": 32768, "length": 512, "hq": 64, "hk": 8, "d": 64,
         "kind": "nvfp4", "page": 64, "sinks": True, "lse": False},
        # Sixteen answers to each of four prompts of uneven lengths, heads of 128.
        {"name": "shared fp8 4 x 16 x 8000 + 1000", "op": "shared", "prefixes": 4, "each": 16, "prefix": 8000, "length": 1000, "hq": 32, "hk": 8, "d": 128,
         "kind": "fp8", "page": 32, "sinks": False, "lse": True},
        # A large batch over a whole document, unquantized.
        {"name": "shared bf16 128 x 65536 + 2048", "op": "shared", "prefixes": 1, "each": 128, "prefix": 65536, "length": 2048, "hq": 64, "hk": 8, "d": 64,
         "kind": "bf16", "page": 64, "sinks": False, "lse": False},
        # One token between two blocks of the decoder stack: all latency.
        {"name": "norm 1 x 2880", "op": "norm", "t": 1, "h": 2880, "post": False, "gate": "", "scale": 1.0, "residual": "bf16"},
        # An odd batch over an odd width, every part of the operator, residual stream in 32 bits.
        {"name": "norm 1021 x 5003 all", "op": "norm", "t": 1021, "h": 5003, "post": True, "gate": "token", "scale": 0.5, "residual": "fp32"},
        # A batch's tokens in the widest model of the benchmarks, norms before and after and a gate for each channel.
        {"name": "norm 33 x 16384 post gate", "op": "norm", "t": 33, "h": 16384, "post": True, "gate": "channel", "scale": 1.0, "residual": "bf16"},
        # The decoder stack's 8192-token prompt.
        {"name": "norm 8192 x 2880 post", "op": "norm", "t": 8192, "h": 2880, "post": True, "gate": "", "scale": 0.22, "residual": "bf16"},
        # One sequence's next token from a nucleus: all latency.
        {"name": "sample 1 x 32768 top-p", "op": "sample", "b": 1, "v": 32768, "type": "bf16", "how": "top_p", "masked": False},
        # A serving batch whose requests each have settings of their own, a few greedy.
        {"name": "sample 64 x 131072 mixed", "op": "sample", "b": 64, "v": 131072, "type": "bf16", "how": "mixed", "masked": False},
        # An odd vocabulary in 32 bits (after penalties), under a grammar's mask.
        {"name": "sample 7 x 100003 fp32 masked", "op": "sample", "b": 7, "v": 100003, "type": "fp32", "how": "top_k_p", "masked": True},
        # Many answers from the whole distribution, as for training on what a model says.
        {"name": "sample 256 x 131072 all", "op": "sample", "b": 256, "v": 131072, "type": "bf16", "how": "all", "masked": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    op = rng.choice(["shared", "norm", "sample"])
    if op == "norm":
        h = rng.choice([_log(rng, 64, 16384), 8 * _log(rng, 8, 2048)])
        return {"op": op, "t": _log(rng, 1, 8192), "h": h, "post": rng.random() < 0.6, "gate": rng.choice(["", "", "channel", "token"]),
                "scale": rng.choice([1.0, 0.5, 0.22]), "residual": rng.choice(["bf16", "bf16", "fp32"])}
    if op == "sample":
        return {"op": op, "b": _log(rng, 1, 256), "v": _log(rng, 500, 262144), "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "how": rng.choice(["top_p", "top_k_p", "min_p", "mixed", "all"]), "masked": rng.random() < 0.3}
    hk = rng.choice([1, 2, 4, 8])
    return {"op": op, "prefixes": rng.choice([1, 1, 1, 2, 3, 5]), "each": _log(rng, 1, 128), "prefix": _log(rng, 1, 65536), "length": _log(rng, 1, 4096),
            "hq": hk * rng.choice([1, 2, 4, 5, 8, 16]), "hk": hk, "d": rng.choice([64, 64, 128, 256]), "kind": rng.choice(["nvfp4", "fp8", "bf16"]),
            "page": rng.choice([1, 16, 32, 64, 128]), "sinks": rng.random() < 0.3, "lse": rng.random() < 0.3}


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        top[c["op"]] = {k: max(w[k], top.get(c["op"], w)[k]) for k in w}
    while True:
        case = _drawn(rng)
        w = work(case)
        if all(w[k] <= top[case["op"]][k] for k in w):
            return case


# ---------------------------------------------------------------------------------------------------------------- their work

def _cell(kind, d):
    """Bytes of one (token, head) row of the cache."""
    return {"bf16": 2 * d, "fp8": d + 4, "nvfp4": d // 2 + d // 16}[kind]


def _spread(longest, count):
    """Lengths known from the case alone: the first the longest, the others anywhere in [1, longest], every eighth none."""
    return [longest if i == 0 else 0 if i % 8 == 7 else max(1, longest * ((i * 7919 + 4001) % 9973) // 9973) for i in range(count)]


def work(case):
    op = case["op"]
    if op == "sample":
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": float(case["b"]) * (case["v"] * size + 4 + 8), "flops": 3.0 * case["b"] * case["v"]}
    if op == "norm":
        n, r = case["t"] * case["h"], 4 if case["residual"] == "fp32" else 2
        gates = {"": 0, "channel": case["h"], "token": n}[case["gate"]]
        return {"bytes": n * (2.0 + 2 * r + 2) + 2 * gates + 2 * case["h"] * (1 + case["post"]), "flops": n * (8.0 if case["post"] else 5.0)}
    b = case["prefixes"] * case["each"]
    shared, mine = _spread(case["prefix"], case["prefixes"]), _spread(case["length"], b)
    pairs = sum(shared) * case["each"] + sum(mine)
    return {"bytes": (sum(shared) + sum(mine)) * case["hk"] * 2.0 * _cell(case["kind"], case["d"]) + 4.0 * b * case["hq"] * case["d"],
            "flops": 4.0 * pairs * case["hq"] * case["d"]}


# ---------------------------------------------------------------------------------------------------------------- the cache's formats

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


def _encode(x, kind):
    """Codes and scales of a used cache's rows [..., D]."""
    if kind == "bf16":
        return x.to(torch.bfloat16), None
    x = x.float()
    if kind == "fp8":
        amax = x.abs().amax(-1).clamp(min=FP8_FLOOR)
        return (x * (448.0 / amax).unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), amax / 448.0
    b = x.reshape(*x.shape[:-1], -1, 16)
    scale = (b.abs().amax(-1) / 6.0).clamp(2.0 ** -6, 448.0).to(torch.float8_e4m3fn)
    a = (b / scale.float().unsqueeze(-1)).abs()
    one = torch.ones((), dtype=torch.uint8, device=x.device)
    code = (a > 0.25) * one + (a > 0.75) + (a > 1.25) + (a > 1.75) + (a > 2.5) + (a > 3.5) + (a > 5.0)
    code = (code + 8 * one * (b < 0)).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.view(torch.uint8)


def _decode(codes, scales, kind):
    if kind == "bf16":
        return codes.float()
    if kind == "fp8":
        return codes.float() * scales.unsqueeze(-1)
    v = torch.stack((_e2m1_value(codes & 15), _e2m1_value(codes >> 4)), -1)
    v = v.reshape(*codes.shape[:-1], -1, 16) * _ue4m3_value(scales).unsqueeze(-1)
    return v.reshape(*codes.shape[:-1], -1)


# ---------------------------------------------------------------------------------------------------------------- the inputs

def _tables(lens, page, order, taken):
    """Page table [len(lens), W] of sequences that take their pages from `order` in turn, from entry `taken` on; -1 where there is none."""
    wide = max(1, -(-max(lens) // page))
    need = torch.tensor([-(-x // page) for x in lens], device=DEV)
    first = (need.cumsum(0) - need + taken).unsqueeze(1)
    at = torch.arange(wide, device=DEV).unsqueeze(0)
    table = torch.where(at < need.unsqueeze(1), order[(first + at).clamp(max=len(order) - 1)], torch.full((), -1, dtype=torch.int32, device=DEV))
    return table.contiguous(), taken + sum(-(-x // page) for x in lens)


def _settings(case, g):
    """Each request's temperature, k, p and min-p."""
    b, how = case["b"], case["how"]

    def between(lo, hi):
        return lo + (hi - lo) * torch.rand(b, generator=g, device=DEV)

    temperature = between(0.5, 1.2)
    top_k, top_p, min_p = torch.zeros(b, dtype=torch.int32, device=DEV), torch.ones(b, device=DEV), torch.zeros(b, device=DEV)
    if how in ("top_k_p", "mixed"):
        top_k = torch.randint(10, 2000, (b,), generator=g, device=DEV, dtype=torch.int32)
    if how in ("top_p", "top_k_p", "mixed"):
        top_p = between(0.8, 0.99)
    if how in ("min_p", "mixed"):
        min_p = between(0.01, 0.1)
    if how == "mixed":  # what a request does not ask for is off; every fifth is greedy
        i = torch.arange(b, device=DEV)
        temperature = torch.where(i % 5 == 4, torch.zeros_like(temperature), temperature)
        top_k = torch.where(i % 2 == 0, top_k, torch.zeros_like(top_k))
        top_p = torch.where(i % 3 != 1, top_p, torch.ones_like(top_p))
        min_p = torch.where(i % 4 == 3, min_p, torch.zeros_like(min_p))
    return temperature, top_k, top_p, min_p


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    op, s = case["op"], {"case": case}

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)

    def near_one(n):
        return (1.0 + 0.1 * randn(n, dtype=torch.float32)).to(torch.bfloat16)

    if op == "sample":
        b, v = case["b"], case["v"]
        # a bulk of unlikely tokens and some dozens that the context speaks for
        logits = 2.0 * randn(b, v, dtype=torch.float32) - 2.0
        apart = v // 48  # one in each 48th of the vocabulary
        likely = torch.arange(48, device=DEV) * apart + torch.randint(0, apart, (b, 48), generator=g, device=DEV)
        logits.scatter_(1, likely, 8.0 + 3.0 * randn(b, 48, dtype=torch.float32))
        if case["masked"]:  # a grammar allows about a fifth of the tokens
            logits.masked_fill_(torch.rand(b, v, generator=g, device=DEV) < 0.8, -math.inf)
        s["logits"] = logits.to(LOGITS[case["type"]])
        s["u"] = torch.rand(b, generator=g, device=DEV)
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = _settings(case, g)
        return s
    if op == "norm":
        t, h = case["t"], case["h"]
        s["x"] = randn(t, h) * 0.7
        s["residual"] = (randn(t, h, dtype=torch.float32) * 3.0).to(torch.float32 if case["residual"] == "fp32" else torch.bfloat16)
        s["weight"], s["post"] = near_one(h), near_one(h) if case["post"] else None
        s["gate"] = {"": lambda: None, "channel": lambda: near_one(h), "token": lambda: torch.sigmoid(randn(t, h, dtype=torch.float32)).to(torch.bfloat16)}[case["gate"]]()
        return s
    each, page, hk, d = case["each"], case["page"], case["hk"], case["d"]
    b = case["prefixes"] * each
    shared, mine = _spread(case["prefix"], case["prefixes"]), _spread(case["length"], b)
    pages = sum(-(-x // page) for x in shared + mine)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)  # strewn over the cache
    s["prefix_table"], taken = _tables(shared, page, order, 0)
    s["table"], _ = _tables(mine, page, order, taken)
    s["prefix_lens"], s["lens"] = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (shared, mine))
    for name, spread in (("k", 1.5), ("v", 1.0)):
        s[name + "_pages"], s[name + "_scales"] = _encode(randn(pages, hk, page, d) * spread, case["kind"])
    s["q"] = randn(b, case["hq"], d) * 1.5
    s["sinks"] = randn(case["hq"], dtype=torch.float32) if case["sinks"] else None
    if own:
        s["cache"] = _framework().PagedKVCache.wrap(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass

def _rows(s, name, table, count):
    """Rows [sequences, count, kv_heads, D] of a page table's first `count` tokens."""
    case = s["case"]
    at = torch.arange(count, device=DEV)
    pages, slot = table.long()[:, at // case["page"]].clamp(min=0), at % case["page"]
    scales = s[name + "_scales"]
    return _decode(s[name + "_pages"][pages, :, slot], None if scales is None else scales[pages, :, slot], case["kind"])


def _plain_shared(s):
    case = s["case"]
    groups, each, hk, d = case["prefixes"], case["each"], case["hk"], case["d"]
    b, scale = groups * each, d ** -0.5

    def scores(q, name_table, count, lens):
        k = _rows(s, "k", name_table, count).permute(0, 2, 3, 1)  # [sequences, hk, D, keys]
        seen = torch.arange(count, device=DEV) < lens.unsqueeze(1)
        return torch.matmul(q, k).mul_(scale).masked_fill_(~seen[:, None, None], -math.inf)

    q = s["q"].float().reshape(b, hk, -1, d)
    group = q.shape[2]
    # all queries of a prefix together, as one matrix for each key head
    together = q.reshape(groups, each, hk, group, d).transpose(1, 2).reshape(groups, hk, each * group, d)
    first = scores(together, s["prefix_table"], case["prefix"], s["prefix_lens"])
    second = scores(q, s["table"], case["length"], s["lens"])

    def apart(x):  # [groups, hk, each * group, n] -> [b, hk, group, n]
        return x.reshape(groups, hk, each, group, -1).transpose(1, 2).reshape(b, hk, group, -1)

    def joined(x):  # and back
        return x.reshape(groups, each, hk, group, -1).transpose(1, 2).reshape(groups, hk, each * group, -1)

    top = torch.maximum(apart(first.amax(-1, keepdim=True)), second.amax(-1, keepdim=True))
    if case["sinks"]:
        sink = s["sinks"].reshape(1, hk, group, 1).expand(b, -1, -1, -1)
        top = torch.maximum(top, sink)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p, mine = first.sub_(joined(top)).exp_(), second.sub_(top).exp_()
    total = apart(p.sum(-1, keepdim=True)) + mine.sum(-1, keepdim=True)
    if case["sinks"]:
        total = total + torch.exp(sink - top)
    acc = apart(torch.matmul(p, _rows(s, "v", s["prefix_table"], case["prefix"]).transpose(1, 2)))
    acc = acc + torch.matmul(mine, _rows(s, "v", s["table"], case["length"]).transpose(1, 2))
    out = torch.where(total > 0, acc / total, torch.zeros_like(acc)).reshape(b, -1, d).to(torch.bfloat16)
    return (out, (top + torch.log(total)).reshape(b, -1)) if case["lse"] else out


def _rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _plain_norm(s):
    y, residual = s["x"].float(), s["residual"]
    if s["post"] is not None:
        y = _rms(y) * s["post"].float()
    if s["gate"] is not None:
        y = y * s["gate"].float()
    r = residual.float() + s["case"]["scale"] * y
    return {"normed": (_rms(r) * s["weight"].float()).to(torch.bfloat16), "residual": r.to(residual.dtype)}


def _plain_sample(s):
    # In 64 bits: which token it is turns on sums over the whole vocabulary that lie next to a border.
    t, k = s["temperature"].double().unsqueeze(1), s["top_k"].long().unsqueeze(1)
    v = s["logits"].shape[1]
    ranked, token = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)  # equal ones by index
    ranked = ranked.double()
    w = torch.where(t > 0, torch.exp((ranked - ranked[:, :1]) / t), torch.zeros_like(ranked))
    w[:, 0] = 1.0
    rank = torch.arange(v, device=DEV)
    kept = torch.where((k > 0) & (rank >= k), torch.zeros_like(w), w)
    before = kept.cumsum(1) - kept
    p = s["top_p"].double().unsqueeze(1)
    kept = torch.where((p < 1) & (before >= p * kept.sum(1, keepdim=True)), torch.zeros_like(kept), kept)
    kept = torch.where(w < s["min_p"].double().unsqueeze(1), torch.zeros_like(kept), kept)
    mass = kept.cumsum(1)
    total = mass[:, -1:]
    at = (mass <= s["u"].double().unsqueeze(1) * total).sum(1, keepdim=True).clamp(max=v - 1)
    return {"token": token.gather(1, at).squeeze(1), "prob": (kept.gather(1, at) / total).squeeze(1).float()}


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"shared": _plain_shared, "norm": _plain_norm, "sample": _plain_sample}[op](s)
    fd = _framework()
    if op == "shared":
        return fd.shared_prefix_attention(s["q"], s["cache"], s["prefix_table"], s["prefix_lens"], s["table"], s["lens"], sinks=s["sinks"], return_lse=case["lse"])
    if op == "norm":
        normed, residual = fd.block_norm(s["x"], s["residual"], s["weight"], post_weight=s["post"], gate=s["gate"], scale=case["scale"], eps=EPS)
        return {"normed": normed, "residual": residual}
    token, prob = fd.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], return_prob=True)
    return {"token": token, "prob": prob}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits

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


def _exact_shared(s):
    """Prefix by prefix and key head by key head, each sequence's own keys behind the prefix's in one softmax."""
    case = s["case"]
    each, hk, d, page, kind = case["each"], case["hk"], case["d"], case["page"], case["kind"]
    b, group = case["prefixes"] * each, case["hq"] // hk
    out = torch.zeros(b, hk, group, d, dtype=torch.float64, device=DEV)
    lse = torch.full((b, hk, group), -math.inf, dtype=torch.float64, device=DEV)

    def of(name, table, n, h):
        at = torch.arange(n, device=DEV)
        pages, slot = table.long()[at // page], at % page
        scales = s[name + "_scales"]
        return _exact_values(s[name + "_pages"][pages, h, slot], None if scales is None else scales[pages, h, slot], kind)

    shared, mine = _spread(case["prefix"], case["prefixes"]), _spread(case["length"], b)
    for i in range(case["prefixes"]):
        for h in range(hk):
            k, v = (of(x, s["prefix_table"][i], shared[i], h) for x in ("k", "v"))
            q = s["q"][i * each: (i + 1) * each].double().reshape(each, hk, group, d)[:, h]
            first = torch.einsum("egd,nd->egn", q, k) / math.sqrt(d)
            for j in range(each):
                row = i * each + j
                ko, vo = (of(x, s["table"][row], mine[row], h) for x in ("k", "v"))
                x = torch.cat((first[j], q[j] @ ko.T / math.sqrt(d)), 1)
                if case["sinks"]:
                    x = torch.cat((x, s["sinks"].double().reshape(hk, group, 1)[h]), 1)
                if x.shape[1]:
                    w = torch.softmax(x, 1)
                    out[row, h] = w[:, : shared[i]] @ v + w[:, shared[i]: shared[i] + mine[row]] @ vo
                    lse[row, h] = torch.logsumexp(x, 1)
    out, lse = out.reshape(b, -1, d), lse.reshape(b, -1)
    return (out, lse) if case["lse"] else out


def _exact_norm(s):
    y, r = s["x"].double(), s["residual"].double()
    if s["post"] is not None:
        y = y / (y.pow(2).sum(1, keepdim=True) / y.shape[1] + EPS).sqrt() * s["post"].double()
    if s["gate"] is not None:
        y = y * s["gate"].double()
    r = r + y * s["case"]["scale"]
    return {"normed": r / (r.pow(2).sum(1, keepdim=True) / r.shape[1] + EPS).sqrt() * s["weight"].double(), "residual": r}


def _exact_sample(s):
    """Row by row, on the host."""
    logits = s["logits"].double().cpu().numpy()
    u, t, k, p, least = (s[x].double().cpu().numpy() for x in ("u", "temperature", "top_k", "top_p", "min_p"))
    tokens, probs = [], []
    for i, l in enumerate(logits):
        order = np.argsort(-l, kind="stable")
        if t[i] == 0:
            order = order[:1]
        elif k[i] > 0:
            order = order[: int(k[i])]
        w = np.exp((l[order] - l[order[0]]) / t[i]) if t[i] else np.ones(1)
        if p[i] < 1:
            sums = np.cumsum(w)
            w = w[: max(1, int(np.searchsorted(sums[:-1], p[i] * sums[-1], side="left")) + 1)]  # those with less than p before them
        w = w[w >= least[i]]
        sums = np.cumsum(w)
        at = min(int(np.searchsorted(sums, u[i] * sums[-1], side="right")), len(w) - 1)
        tokens.append(order[at])
        probs.append(w[at] / sums[-1])
    return {"token": torch.tensor(np.array(tokens), dtype=torch.int64), "prob": torch.tensor(np.array(probs), dtype=torch.float64)}


def exact(case, seed):
    global own
    kept, own = own, False
    s = prepare(case, seed)
    own = kept
    return {"shared": _exact_shared, "norm": _exact_norm, "sample": _exact_sample}[case["op"]](s)
