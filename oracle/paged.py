"""Paged-cache operators in float64 (torch, any device): attention of new tokens over pages,
the norm/rotary/store of a chunk, with the sums of magnitudes the tests' error bounds need."""

from __future__ import annotations

import torch

EPS = 1e-6


def gather_rows(cache, table, rows):
    """Rows `rows` (a list of positions) of one sequence: float64 [len(rows), heads, dim]."""
    page_rows = cache.shape[1]
    at = torch.tensor(rows, dtype=torch.long, device=cache.device)
    pages = torch.tensor([table[r // page_rows] for r in rows], dtype=torch.long, device=cache.device)
    return cache[pages, at % page_rows].double()


def attention(q, k_cache, v_cache, tables, lens, scale=1.0, window=0):
    """q [T, Hq, D]; lens [(new tokens, cache rows)] per sequence; tables: lists of pages.
    Returns (out, weight): out[t, h] and weight[t, h] = sum_j p_j |v_j|, float64."""
    tokens, hq, d = q.shape
    hkv = k_cache.shape[2]
    g = hq // hkv
    out = torch.zeros(tokens, hq, d, dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(out)
    t0 = 0
    for s, (n, kv) in enumerate(lens):
        pos = [kv - n + i for i in range(n)]
        lo = max(0, pos[0] - window + 1) if window and n else 0
        rows = list(range(lo, kv))
        if n and rows:
            k, v = gather_rows(k_cache, tables[s], rows), gather_rows(v_cache, tables[s], rows)
            at = torch.tensor(pos, device=q.device)[:, None]
            j = torch.tensor(rows, device=q.device)[None, :]
            see = (j <= at) & ((j > at - window) if window else torch.ones_like(j, dtype=torch.bool))
            some = see.any(1)
            for h in range(hq):
                x = (q[t0:t0 + n, h].double() @ k[:, h // g].T) * scale
                p = torch.zeros_like(x)
                p[some] = torch.softmax(x[some].masked_fill(~see[some], float("-inf")), 1)
                out[t0:t0 + n, h] = p @ v[:, h // g]
                weight[t0:t0 + n, h] = p @ v[:, h // g].abs()
        t0 += n
    return out, weight


def norm(x, w=None):
    x = x.double()
    y = x / ((x * x).mean(-1, keepdim=True) + EPS).sqrt()
    return y if w is None else y * w.double()


def rotate(x, cos, sin):
    """(x cos + swapped halves * sin, sum of the two products' magnitudes); sin's low half is
    negated already; cos, sin [T, D]."""
    half = x.shape[-1] // 2
    other = torch.cat([x[..., half:], x[..., :half]], -1)
    a, b = x * cos.double()[:, None], other * sin.double()[:, None]
    return a + b, a.abs() + b.abs()
