"""Plain 64-bit restatement of fp4_decode.shared_prefix_attention.  Nothing here calls the library."""
import math

import torch


def keys_of(rows, table, n, page_size):
    """[n, kv_heads, D] of a page table's first n tokens; a page out of range counts as zeros."""
    at = torch.arange(n, device=rows.device)
    pages = table.long()[at // page_size]
    there = (pages >= 0) & (pages < rows.shape[0])
    return rows[pages.clamp(0, rows.shape[0] - 1), :, at % page_size] * there.reshape(-1, 1, 1)


def attention(q, k_rows, v_rows, prefix_table, prefix_lens, page_table, lens, page_size, scale, sinks):
    """(out, lse, sum of p |v|) in 64 bits; k_rows, v_rows: all pages' values [P, H, S, D]."""
    b, hq, d = q.shape
    hk = k_rows.shape[1]
    groups, each = prefix_lens.shape[0], b // prefix_lens.shape[0]
    out, mag = (torch.zeros(b, hk, hq // hk, d, dtype=torch.float64, device=q.device) for _ in range(2))
    lse = torch.full((b, hk, hq // hk), -math.inf, dtype=torch.float64, device=q.device)
    for g in range(groups):
        shared = [keys_of(r, prefix_table[g], max(0, min(int(prefix_lens[g]), prefix_table.shape[1] * page_size)), page_size) for r in (k_rows, v_rows)]
        for i in range(g * each, (g + 1) * each):
            own = [keys_of(r, page_table[i], max(0, min(int(lens[i]), page_table.shape[1] * page_size)), page_size) for r in (k_rows, v_rows)]
            k, v = (torch.cat(x) for x in zip(shared, own))
            s = torch.einsum("hgd,nhd->hgn", q[i].double().reshape(hk, -1, d), k) * scale
            if sinks is not None:
                s = torch.cat((s, sinks.double().reshape(hk, -1, 1)), -1)
            if s.shape[-1] == 0:
                continue
            p = torch.softmax(s, -1)[..., : len(k)]
            out[i], mag[i], lse[i] = torch.einsum("hgn,nhd->hgd", p, v), torch.einsum("hgn,nhd->hgd", p, v.abs()), torch.logsumexp(s, -1)
    return out.reshape(b, hq, d), lse.reshape(b, hq), mag.reshape(b, hq, d)
