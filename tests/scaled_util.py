"""Block-scaled caches for the tests: filled through the oracle's definition."""
import torch

from oracle.scaled_ref import PAD, TILE, codes_of, exponent, places

BF, I32, U8 = torch.bfloat16, torch.int32, torch.uint8


def cache_of(x, is_v):
    """A cache that holds x [blocks, B, Hk, D] (every row of every tile written at once)."""
    NB, B, Hk, D = x.shape
    cache = torch.zeros(NB, B, Hk * D + PAD, dtype=U8)
    mem, place = cache.view(-1, TILE * (Hk * D + PAD)), places(D)[int(is_v)].flatten()
    rows = x.double().view(-1, TILE, Hk, D)
    for i in range(rows.size(0)):
        for h in range(Hk):
            e = exponent(rows[i, :, h].abs().max().item())
            mem[i, h * TILE * D:(h + 1) * TILE * D][place] = codes_of(rows[i, :, h], e).flatten()
            mem[i, TILE * Hk * D + h] = e + 127
    return cache


def tables_of(lens, B, seed=0, width=None, spare=2):
    """Block tables (shuffled, -1 past each sequence's blocks) and the number of blocks."""
    counts = [-(-n // B) for n in lens]
    NB = sum(counts) + spare
    ids = torch.randperm(NB, generator=torch.Generator().manual_seed(seed)).int()
    bt, at = torch.full((len(lens), width or max(counts + [0]) + 1), -1, dtype=I32), 0
    for i, c in enumerate(counts):
        bt[i, :c] = ids[at:at + c]
        at += c
    return bt, NB


def values(n, Hk, D, g, outliers=True):
    """bf16 rows whose heads, dims and tokens differ in size."""
    x = torch.randn(n, Hk, D, generator=g)
    if outliers:
        x *= torch.exp(1.5 * torch.randn(Hk, 1, generator=g)) * torch.exp(torch.randn(D, generator=g))
        x *= torch.exp(0.5 * torch.randn(n, 1, 1, generator=g))
    return x.to(BF)


def slots_of(bt, B, i, lo, hi):
    return [int(bt[i, p // B]) * B + p % B for p in range(lo, hi)]
