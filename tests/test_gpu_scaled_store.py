"""Block-scaled caches: rows stored and read back. Both are exact by their definition (powers of two,
one rounding to E4M3), so every byte is compared; a NaN may have either sign."""
import importlib
import random

import pytest
import torch

from oracle.scaled_ref import PAD, TILE, scaled_rows_ref, scaled_store_ref
from scaled_util import BF, I32, U8, slots_of, tables_of, values

pytestmark = pytest.mark.gpu

nkv = importlib.import_module("nanokv-llm_amd")
L = importlib.import_module("nanokv-llm_amd._lib")


def plain_nan(c):
    return torch.where((c & 0x7f) == 0x7f, torch.full_like(c, 0x7f), c)


def same_cache(got, want, Hk, D):
    """Codes and scale bytes; the rest of a tile is unused."""
    n = TILE * Hk * D
    got, want = (x.cpu().view(-1, TILE * (Hk * D + PAD)) for x in (got, want))
    assert torch.equal(got[:, n:], want[:, n:])
    bad = (plain_nan(got[:, :n]) != plain_nan(want[:, :n])).nonzero()
    assert not len(bad), (len(bad), bad[:4].tolist())


class Caches:
    """Caches on the GPU and the oracle's, given the same calls."""

    def __init__(self, dev, NB, B, Hk, D, fill=None):
        g = torch.Generator().manual_seed(99)
        shape = (NB, B, Hk * D + PAD)
        self.ref = [torch.zeros(shape, dtype=U8) if fill is None else
                    torch.randint(0, 256, shape, generator=g, dtype=U8) for _ in range(2)]
        self.gpu = [c.to(dev) for c in self.ref]
        self.dev, self.Hk, self.D = dev, Hk, D

    def store(self, key, value, slots):
        slots = torch.as_tensor(slots, dtype=I32)
        nkv.scaled_store_kvcache(key.to(self.dev), value.to(self.dev), *self.gpu,
                                 slots.to(self.dev))
        scaled_store_ref(key, value, *self.ref, slots)

    def check(self):
        for got, want in zip(self.gpu, self.ref):
            same_cache(got, want, self.Hk, self.D)


@pytest.mark.parametrize("Hk,D,B", [(1, 64, 32), (2, 64, 64), (3, 64, 96), (1, 128, 32), (2, 128, 64),
                                    (5, 128, 32), (8, 64, 32)])
@pytest.mark.parametrize("seed", [0, 1])
def test_prompts_chunks_and_steps(dev, Hk, D, B, seed):
    """Sequences that grow call by call: chunks that begin and end inside tiles, single tokens, and
    magnitudes that make scales grow."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    lens = [rng.randint(1, 140) for _ in range(4)]
    bt, NB = tables_of(lens, B, seed)
    c, at = Caches(dev, NB, B, Hk, D), [0] * 4
    for step in range(12):
        slots, rows = [], []
        for i in rng.sample(range(4), 4):
            n = min(lens[i] - at[i], rng.choice([0, 1, 1, 2, rng.randint(1, 70)]))
            slots += slots_of(bt, B, i, at[i], at[i] + n)
            at[i] += n
        n = len(slots)
        if n:
            x, y = (values(n, Hk, D, g) * 2.0 ** rng.randint(-3, 3) for _ in range(2))
            c.store(x.to(BF), y.to(BF), slots)
    c.check()


@pytest.mark.parametrize("D", [64, 128])
def test_a_long_list_and_a_short_one_write_the_same(dev, D):
    """The list's length chooses how many tokens a wave looks at: runs across their borders."""
    Hk, B = 8, 256
    g = torch.Generator().manual_seed(4)
    lens = [1, 31, 700, 33, 5] + [1] * 90 + [64, 300, 7]
    bt, NB = tables_of(lens, B)
    first = [i % 29 for i in range(len(lens))]  # begin inside tiles
    bt2, NB2 = tables_of([a + b for a, b in zip(first, lens)], B)
    slots = [s for i, n in enumerate(lens) for s in slots_of(bt2, B, i, first[i], first[i] + n)]
    x, y = values(len(slots), Hk, D, g), values(len(slots), Hk, D, g)
    whole, parts = (torch.zeros(2, NB2, B, Hk * D + PAD, dtype=U8, device=dev) for _ in range(2))
    s = torch.tensor(slots, dtype=I32, device=dev)
    xg, yg = x.to(dev), y.to(dev)
    nkv.scaled_store_kvcache(xg, yg, whole[0], whole[1], s)
    at = 0
    for n in lens:
        nkv.scaled_store_kvcache(xg[at:at + n], yg[at:at + n], parts[0], parts[1], s[at:at + n])
        at += n
    assert torch.equal(whole, parts)
    ref = [torch.zeros(NB2, B, Hk * D + PAD, dtype=U8) for _ in range(2)]
    scaled_store_ref(x, y, *ref, torch.tensor(slots))
    same_cache(whole[0], ref[0], Hk, D)
    same_cache(whole[1], ref[1], Hk, D)


@pytest.mark.parametrize("D", [64, 128])
def test_any_order_within_a_tile_and_two_for_a_slot(dev, D):
    g = torch.Generator().manual_seed(5)
    c = Caches(dev, 3, 32, 2, D)
    order = torch.randperm(32, generator=g)
    c.store(values(32, 2, D, g), values(32, 2, D, g), 32 + order)
    c.store(values(4, 2, D, g), values(4, 2, D, g), [64, 64, 66, 64])     # the last one stays
    c.store(values(100, 2, D, g), values(100, 2, D, g), [7] * 100)        # more than a wave's lanes
    c.check()


@pytest.mark.parametrize("D", [64, 128])
def test_slots_that_are_skipped(dev, D):
    """Padding and slots outside the cache write nothing; a call of nothing else leaves all as it was."""
    g = torch.Generator().manual_seed(6)
    c = Caches(dev, 2, 32, 2, D, fill="random")
    x, y = values(6, 2, D, g), values(6, 2, D, g)
    c.store(x, y, [-1, -1, 64, 2 ** 31 - 1, -7, -2 ** 31])
    c.check()
    c.store(x, y, [-1, 0, 1, -1, 64, 40])
    c.store(x[:0], y[:0], [])
    c.check()


@pytest.mark.parametrize("Hk,D,n", [(2, 64, 6), (2, 128, 6), (8, 64, 200), (8, 128, 200)])
def test_slots_that_are_skipped_inside_a_tile(dev, Hk, D, n):
    """Skipped slots between a tile's tokens, up to 31 at once and over the borders of what a wave
    looks at: one scale all the same, also where it grows and the rows held are rounded again."""
    rng, g = random.Random(n), torch.Generator().manual_seed(n)
    c = Caches(dev, n, 32, Hk, D)
    c.store(values(n, Hk, D, g) * 2.0 ** -6, values(n, Hk, D, g) * 2.0 ** -6,
            [32 * i + 3 for i in range(n)])
    slots = []
    for i in range(n):
        for r in sorted(rng.sample(range(1, 32), rng.choice([1, 2, 5, 31]))):
            slots += [32 * i + r] + [-1] * rng.choice([0, 0, 0, 1, 2, 7, 31])
        slots += [-1] * rng.choice([0, 40])
    c.store(values(len(slots), Hk, D, g), values(len(slots), Hk, D, g), slots)
    c.check()


@pytest.mark.parametrize("D", [64, 128])
def test_special_values(dev, D):
    """NaN, infinities, zeros of both signs, subnormals and the largest values."""
    g = torch.Generator().manual_seed(7)
    big = float(torch.finfo(BF).max)
    for pick in ([float("nan")], [float("inf"), -float("inf")], [big, -big], [0.0, -0.0],
                 [2.0 ** -133, 2.0 ** -126, 2.0 ** -109, 2.0 ** -110], [float("nan"), big, 1e-30]):
        c = Caches(dev, 2, 32, 2, D)
        for n, first in ((20, 0), (3, 20), (32, 32)):
            x, y = values(n, 2, D, g), values(n, 2, D, g)
            for t in (x, y):
                at = torch.randint(0, t.numel(), (9,), generator=g)
                t.view(-1)[at] = torch.tensor(pick, dtype=BF)[torch.arange(9) % len(pick)]
            c.store(x, y, torch.arange(first, first + n))
        c.store(torch.zeros(1, 2, D, dtype=BF), torch.full((1, 2, D), pick[0], dtype=BF), [23])
        c.check()


def test_every_bf16_value_rounds_to_its_nearest_code(dev):
    """All 65536 patterns, a row of 64 of one exponent range each, and ties among them."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(BF).view(-1, 1, 64)
    c = Caches(dev, 32, 32, 1, 64)
    c.store(bits, bits.flip(0), torch.arange(1024))
    c.check()


def test_strided_rows_and_a_head_range(dev):
    """K and V as parts of fused projection rows."""
    g = torch.Generator().manual_seed(8)
    fused = values(50, 9, 128, g).to(dev)
    k, v = fused[:, 4:6], fused[:, 7:9]
    kc, vc = (torch.zeros(2, 64, 2 * 128 + PAD, dtype=U8, device=dev) for _ in range(2))
    slots = torch.arange(10, 60, dtype=I32, device=dev)
    nkv.scaled_store_kvcache(k, v, kc, vc, slots)
    ref = [torch.zeros(2, 64, 2 * 128 + PAD, dtype=U8) for _ in range(2)]
    scaled_store_ref(k.cpu(), v.cpu(), *ref, slots.cpu())
    same_cache(kc, ref[0], 2, 128)
    same_cache(vc, ref[1], 2, 128)


# ---------------------------------------------------------------- reading back
def read_ref(k, v, bt, cu, n, Hk, D, starts, fill=7.0):
    out = [torch.full((n, Hk, D), fill, dtype=BF) for _ in range(2)]
    for i, (a, b) in enumerate(zip(cu, cu[1:])):
        s = starts[i] if starts else 0
        if 0 <= a < b <= n and s >= 0:
            for o, c, is_v in ((out[0], k, False), (out[1], v, True)):
                o[a:b] = scaled_rows_ref(c, is_v, bt[i].tolist(), b - a, Hk, D, s).to(BF)
    return out


def check_read(dev, k, v, bt, cu, n, Hk, D, starts=None):
    out = tuple(torch.full((n, Hk, D), 7.0, dtype=BF, device=dev) for _ in range(2))
    i32 = dict(dtype=I32, device=dev)
    got = nkv.scaled_read_kvcache(k.to(dev), v.to(dev), bt.to(dev), torch.tensor(cu, **i32), n, Hk,
                                  starts=None if starts is None else torch.tensor(starts, **i32),
                                  out=out)
    assert got is out
    for a, b in zip(got, read_ref(k, v, bt, cu, n, Hk, D, starts)):
        assert torch.equal(a.cpu().isnan(), b.isnan())
        assert torch.equal(a.cpu().nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("Hk,D,B", [(1, 64, 32), (3, 64, 64), (1, 128, 96), (2, 128, 32), (8, 64, 32)])
def test_read_any_bytes(dev, Hk, D, B):
    """Caches of random bytes: every code and scale byte there is."""
    g = torch.Generator().manual_seed(9)
    lens = [1, 70, 0, 33, 32, 95]
    bt, NB = tables_of(lens, B)
    k, v = (torch.randint(0, 256, (NB, B, Hk * D + PAD), generator=g, dtype=U8) for _ in range(2))
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    check_read(dev, k, v, bt, cu, cu[-1], Hk, D)
    # from a position on, some rows of no sequence
    starts = [0, 13, 5, 1, 31, 64]
    cu = [3]
    for n, s in zip(lens, starts):
        cu.append(cu[-1] + max(0, n - s))
    check_read(dev, k, v, bt, cu, cu[-1] + 4, Hk, D, starts)


def test_read_what_is_not_there(dev):
    """No valid block, past the table, cu_seqlens outside the rows, positions below zero: zeros, or
    rows left as they are."""
    g = torch.Generator().manual_seed(10)
    k, v = (torch.randint(0, 256, (3, 32, 64 + PAD), generator=g, dtype=U8) for _ in range(2))
    bt = torch.tensor([[0, -1, 2], [3, 1, -9], [1, 1, 1]], dtype=I32)
    check_read(dev, k, v, bt, [0, 96, 150, 200], 200, 1, 64)
    check_read(dev, k, v, bt, [0, 96, 150, 350], 350, 1, 64, [0, 40, 5])   # past the table
    check_read(dev, k, v, bt, [-5, 20, 60, 201], 200, 1, 64)
    check_read(dev, k, v, bt, [50, 20, 20, 60], 200, 1, 64)
    check_read(dev, k, v, bt, [0, 20, 40, 60], 60, 1, 64, [-1, 2 ** 31 - 5, 3])


def test_many_short_sequences(dev):
    g = torch.Generator().manual_seed(11)
    lens = [i % 5 for i in range(300)]
    bt, NB = tables_of(lens, 32)
    k, v = (torch.randint(0, 256, (NB, 32, 2 * 64 + PAD), generator=g, dtype=U8) for _ in range(2))
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    check_read(dev, k, v, bt, cu, cu[-1], 2, 64)


def test_read_of_nothing(dev):
    k = torch.zeros(2, 32, 64 + PAD, dtype=U8, device=dev)
    cu = torch.zeros(1, dtype=I32, device=dev)
    bt = torch.zeros(1, 1, dtype=I32, device=dev)
    a, b = nkv.scaled_read_kvcache(k, k, bt, cu, 0, 1)
    assert a.shape == b.shape == (0, 1, 64)
    a, _ = nkv.scaled_read_kvcache(k, k, bt, torch.zeros(2, dtype=I32, device=dev), 5, 1)
    assert a.shape == (5, 1, 64)


def test_captured_and_on_another_stream(dev):
    """Store and read in a graph, replayed over changing rows, against eager calls."""
    g = torch.Generator().manual_seed(12)
    Hk, D, n = 2, 128, 5
    x, y = values(n, Hk, D, g).to(dev), values(n, Hk, D, g).to(dev)
    slots = torch.tensor([40, 41, -1, 96, 127], dtype=I32, device=dev)
    bt = torch.tensor([[1, 3, 0]], dtype=I32, device=dev)
    cu = torch.tensor([0, 96], dtype=I32, device=dev)
    kc, vc = (torch.zeros(4, 32, Hk * D + PAD, dtype=U8, device=dev) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nkv.scaled_store_kvcache(x, y, kc, vc, slots)
        nkv.scaled_read_kvcache(kc, vc, bt, cu, 96, Hk)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nkv.scaled_store_kvcache(x, y, kc, vc, slots)
        out = nkv.scaled_read_kvcache(kc, vc, bt, cu, 96, Hk)
    ke, ve = kc.clone(), vc.clone()
    for i in range(4):
        x.copy_(values(n, Hk, D, g) * 4.0 ** i)
        y.copy_(values(n, Hk, D, g))
        graph.replay()
        nkv.scaled_store_kvcache(x, y, ke, ve, slots)
        want = nkv.scaled_read_kvcache(ke, ve, bt, cu, 96, Hk)
        torch.cuda.synchronize()
        assert torch.equal(kc, ke) and torch.equal(vc, ve)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_past_four_gib(dev):
    """Slots and blocks whose bytes lie past 2^32."""
    Hk, D, B = 8, 128, 256
    NB = (1 << 32) // (B * (Hk * D + PAD)) + 40
    kc, vc = (torch.zeros(NB, B, Hk * D + PAD, dtype=U8, device=dev) for _ in range(2))
    g = torch.Generator().manual_seed(13)
    x, y = values(40, Hk, D, g).to(dev), values(40, Hk, D, g).to(dev)
    slots = torch.arange((NB - 1) * B, (NB - 1) * B + 40, dtype=I32, device=dev)
    nkv.scaled_store_kvcache(x, y, kc, vc, slots)
    small = [torch.zeros(1, B, Hk * D + PAD, dtype=U8, device=dev) for _ in range(2)]
    nkv.scaled_store_kvcache(x, y, *small, slots - (NB - 1) * B)
    assert torch.equal(kc[-1:], small[0]) and torch.equal(vc[-1:], small[1])
    bt = torch.tensor([[NB - 1]], dtype=I32, device=dev)
    cu = torch.tensor([0, 40], dtype=I32, device=dev)
    got = nkv.scaled_read_kvcache(kc, vc, bt, cu, 40, Hk)
    want = nkv.scaled_read_kvcache(*small, torch.zeros_like(bt), cu, 40, Hk)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
