"""Plain 64-bit restatements of the decode-side operators, for their tests: the cache's formats decoded by table, the
norm + rotation, attention key by key of each sequence.  Nothing here calls the library."""
import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
UE4M3 = [(c & 7) / 512.0 if (c >> 3) & 15 == 0 else (8 + (c & 7)) * 2.0 ** (((c >> 3) & 15) - 10) for c in range(256)]


def e2m1_values(packed: torch.Tensor) -> torch.Tensor:
    """[..., n] bytes -> [..., 2n] values, the low nibble first."""
    lut = torch.tensor(E2M1, dtype=torch.float64, device=packed.device)
    b = packed.to(torch.int64)
    return torch.stack([lut[b & 15], lut[b >> 4]], dim=-1).flatten(-2)


def ue4m3_values(codes: torch.Tensor) -> torch.Tensor:
    return torch.tensor(UE4M3, dtype=torch.float64, device=codes.device)[codes.to(torch.int64)]


def cache_values(pages, scales, kind) -> torch.Tensor:
    """All rows of a cache's pages [P, H, S, D] in 64 bits."""
    if kind == "bf16":
        return pages.double()
    if kind == "fp8":
        return pages.float().double() * scales.double().unsqueeze(-1)
    return e2m1_values(pages) * ue4m3_values(scales).repeat_interleave(16, dim=-1)


def norm_rope(x, weight, positions, table, eps, interleaved):
    """x [T, H, D] -> 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if table is None:
        return x
    rot = table.shape[1]
    half = rot // 2
    row = table.double()[positions.long()]
    out = x.clone()
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = row[:, None, i], row[:, None, half + i]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def attention(q, k_rows, v_rows, page_table, lens, page_size, scale, window, sinks):
    """(out, lse, sum of p |v|) in 64 bits; k_rows, v_rows: all pages' values [P, H, S, D]."""
    b, hq, d = q.shape
    hk = k_rows.shape[1]
    g = hq // hk
    outs, lses, mags = [], [], []
    for i in range(b):
        n = int(lens[i])
        first = max(0, n - window) if window else 0
        at = torch.arange(first, n, device=q.device)
        pages = page_table[i].long()[at // page_size]
        k, v = k_rows[pages, :, at % page_size], v_rows[pages, :, at % page_size]  # [n, hk, d]
        for h in range(hq):
            s = (k[:, h // g] @ q[i, h].double()) * scale
            if sinks is not None:
                s = torch.cat([s, sinks[h].double().reshape(1)])
            if s.numel() == 0:
                outs.append(torch.zeros(d, dtype=torch.float64, device=q.device))
                mags.append(outs[-1])
                lses.append(torch.tensor(-math.inf, dtype=torch.float64, device=q.device))
                continue
            top = s.max()
            p = torch.exp(s - top)
            total = p.sum()
            p = p[: len(at)] / total
            outs.append(p @ v[:, h // g])
            mags.append(p @ v[:, h // g].abs())
            lses.append(top + torch.log(total))
    return torch.stack(outs).reshape(b, hq, d), torch.stack(lses).reshape(b, hq), torch.stack(mags).reshape(b, hq, d)
