"""ORACLE (test infrastructure): the block-scaled K/V cache in 64 bits, one tile and row at a time.

A tile is 32 rows of one head under one scale 2^e: code = E4M3(x * 2^-e), read as code * 2^e. The cache
is uint8 [blocks, block_size, Hk * D + 16]; its rows stand in tiles of 32, the heads' codes (32 * D bytes
each, in the orders of ``places``), then Hk bytes e + 127 (0: nothing written). It stands beside
store_kvcache and the attention calls of nanokvllm/layers/attention.py:33-40, 96-107.
"""
from __future__ import annotations

import math

import torch

from .fp8_ref import e4m3fn_table, nearest_e4m3fn

TILE, PAD, E_MIN, E_MAX = 32, 16, -100, 119


def places(D: int):
    """Byte of (token, dim) among a head's codes: for K, for V (each [32, D])."""
    k, v = torch.empty(TILE, D, dtype=torch.int64), torch.empty(TILE, D, dtype=torch.int64)
    for t in range(2):
        for i in range(D // 64):
            for g in range(4):
                for r in range(16):
                    at = ((t * (D // 64) + i) * 64 + r + 16 * g) * 16
                    dim = 64 * i + 16 * g
                    k[8 * (r // 4) + 4 * t + r % 4, dim:dim + 16] = torch.arange(at, at + 16)
    for j in range(D // 32):
        for g in range(4):
            for c in range(16):
                for u in range(2):
                    at = (j * 64 + c + 16 * g) * 16 + 8 * u
                    v[8 * g:8 * g + 8, 32 * j + 16 * u + c] = torch.arange(at, at + 8)
    return k, v


def exponent(a: float) -> int:
    """The smallest e in range with a <= 448 * 2^e."""
    e = E_MIN
    while e < E_MAX and a > math.ldexp(448.0, e):
        e += 1
    return e


def codes_of(x: torch.Tensor, e: int) -> torch.Tensor:
    """E4M3 codes (uint8) of x * 2^-e, x float64: nearest even, +-448 at most, NaN kept."""
    y = (x * math.ldexp(1.0, -e)).clamp(-448, 448)
    return torch.where(y.isnan(), 0x7f, nearest_e4m3fn(y.nan_to_num()).int()).to(torch.uint8)


def _tile(cache, i):
    return cache.view(-1, TILE * cache.size(2))[i]


def scaled_store_ref(key, value, k_cache, v_cache, slots) -> None:
    """Into the caches in place. A tile's tokens count together wherever they stand in ``slots``."""
    N, Hk, D = key.shape
    n_slots = k_cache.size(0) * k_cache.size(1)
    table = e4m3fn_table()
    groups: dict = {}
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < n_slots:
            groups.setdefault(s // TILE, {})[s % TILE] = i  # of two for a slot the later one
    for x, cache, place in zip((key, value), (k_cache, v_cache), places(D)):
        for tile, rows in groups.items():
            mem = _tile(cache, tile)
            at, src = torch.tensor(list(rows)), torch.tensor(list(rows.values()))
            for h in range(Hk):
                new = x[src, h].double()
                a = torch.where(new.isfinite(), new.abs(), 0).max().item()
                codes = mem[h * TILE * D:(h + 1) * TILE * D]
                old = min(max(int(mem[TILE * Hk * D + h]) - 127, E_MIN), E_MAX)
                e = exponent(a)
                if 0 not in rows:
                    e = max(e, old)
                    if e > old:
                        held = table[codes.long()]
                        codes.copy_(torch.where(held.isnan(), codes, codes_of(held, e - old)))
                codes[place[at].flatten()] = codes_of(new, e).flatten()
                mem[TILE * Hk * D + h] = e + 127


def scaled_rows_ref(cache, is_v: bool, table, n: int, Hk: int, D: int, start: int = 0,
                    zeros: bool = True) -> torch.Tensor:
    """Rows [start, start + n) of a sequence in 64 bits [n, Hk, D]; where its table has no valid block
    zeros, or (``zeros`` false) no row."""
    NB, B = cache.size(0), cache.size(1)
    place, values, out = places(D)[int(is_v)], e4m3fn_table(), []
    for p in range(start, start + n):
        b = int(table[p // B]) if p // B < len(table) else -1
        if not 0 <= b < NB:
            if zeros:
                out.append(torch.zeros(Hk, D, dtype=torch.float64))
            continue
        mem = _tile(cache, (b * B + p % B) // TILE)
        heads = mem[:TILE * Hk * D].view(Hk, TILE * D)[:, place[p % TILE]]
        e = mem[TILE * Hk * D:TILE * Hk * D + Hk].double() - 127
        out.append(values[heads.long()] * torch.exp2(e.clamp(E_MIN, E_MAX))[:, None])
    return torch.stack(out) if out else torch.zeros(0, Hk, D, dtype=torch.float64)


def attention_rows_ref(q, k, v, scale: float) -> torch.Tensor:
    """Causal attention (bottom right) of q [Lq, Hq, D] over k, v [Lk, Hk, D] in 64 bits: a row's keys
    are sliced, so that none that it does not see takes part; a row without any is zero."""
    Lq, Hq, D = q.shape
    Lk, Hk = k.size(0), k.size(1)
    out = torch.zeros(Lq, Hq, D, dtype=torch.float64)
    for j in range(Lq):
        n = Lk - Lq + j + 1
        if n <= 0:
            continue
        for h in range(Hq):
            p = torch.softmax(k[:n, h * Hk // Hq] @ q[j, h].double() * scale, 0)
            out[j, h] = p @ v[:n, h * Hk // Hq]
    return out
