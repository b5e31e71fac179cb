"""Differential attention from its definition, in 64 bits, one sequence and pair at a time.

out_h = (1 - init) * norm(A_0 - lambda A_1), A_m = softmax(scale q_{2h+m} K_{2p+m}^T) [V_2p | V_2p+1]
with p = h // (Hq / Hk), causal and aligned to the bottom right.
"""
from __future__ import annotations

import math

import torch


def diff_attention_ref(q, k, v, scale, lambdas, lambda_init, weight=None, eps=1e-5, n_hidden=0):
    """One sequence: q [Lq, Hq, D], k and v [Lk, Hk, D] -> [Lq, Hq/2, 2 D] float64. Query j sees keys
    0 .. Lk - Lq + j; ``n_hidden`` more keys at the front of k are seen by nobody."""
    q, k, v, l = q.double(), k.double(), v.double(), lambdas.double()
    Lq, Hq, D = q.shape
    Lk, Hk, _ = k.shape
    lam = math.exp(float(l[0] @ l[1])) - math.exp(float(l[2] @ l[3])) + lambda_init
    out = torch.zeros(Lq, Hq // 2, 2 * D, dtype=torch.float64)
    seen = torch.arange(Lk)[None] <= (Lk - Lq + torch.arange(Lq))[:, None]
    seen &= torch.arange(Lk)[None] >= n_hidden
    for h in range(Hq // 2):
        p = h // (Hq // Hk)
        value = torch.cat([v[:, 2 * p], v[:, 2 * p + 1]], dim=1)
        maps = []
        for m in (0, 1):
            s = (q[:, 2 * h + m] @ k[:, 2 * p + m].T * scale).masked_fill(~seen, -math.inf)
            a = torch.zeros(Lq, 2 * D, dtype=torch.float64)
            rows = seen.any(1)
            if rows.any():
                a[rows] = torch.softmax(s[rows], dim=1) @ value
            maps.append(a)
        o = maps[0] - lam * maps[1]
        o = (1 - lambda_init) * o / (o.square().mean(1, keepdim=True) + eps).sqrt()
        out[:, h] = o if weight is None else o * weight.double()
    return out


def gather_rows(cache, table, n, block_size, zeros=False, scale=1.0):
    """The first n rows of a paged cache [NB, B, Hk, D] by a block table: float64 [rows, Hk, D]. Rows
    past the table or in an invalid block are left out, or (``zeros``) zeros."""
    NB = cache.size(0)
    rows = []
    for t in range(n):
        b = int(table[t // block_size]) if t // block_size < len(table) else -1
        if 0 <= b < NB:
            rows.append(cache[b, t % block_size].double() * scale)
        elif zeros:
            rows.append(torch.zeros(cache.shape[2:], dtype=torch.float64))
    return torch.stack(rows) if rows else torch.zeros(0, *cache.shape[2:], dtype=torch.float64)
