"""Block-scaled caches: sizes at the ends of what the calls take and values at the ends of what a tile holds,
none of which needs a GPU."""
import math
import struct

import pytest
import torch

from oracle.scaled_ref import PAD, codes_of, exponent, scaled_rows_ref, scaled_store_ref
from test_scaled_checks import BF, I32, L, P, PREFILL, STORE, U8


def _args(base, **kw):
    a = dict(base, **kw)
    scale = [a.pop("scale")] if "scale" in a else []
    args = [0 if x is None else x for x in (*a.values(), None)] + scale  # the stream: NULL
    return struct.pack(f"{len(args) - len(scale)}q{len(scale)}d", *args)


@pytest.mark.parametrize("n,tq,mq,hq,hk,d", [(1, 8, 8, 4, 1, 64), (1, 8, 8, 32, 8, 128), (1, 500, 500, 4, 1, 64),
                                             (3, 24, 8, 8, 1, 128), (40, 40, 1, 4, 1, 64)])
def test_split_prefill_positions_stay_within_32_bits(n, tq, mq, hq, hk, d):
    """A split launch counts every key at 9 a tile at most, at 5 at least, and 192 more a tile, and its
    positions are 32 bits: longer streams are launched whole, which needs no workspace."""
    f = L.lib().nkv_scaled_prefill_workspace_bytes
    tiles = n * -(-mq * hq // hk // 192)  # at least
    seen = set()
    for keys in (10 ** 5, 10 ** 6, 33_500_000, 33_600_000, 10 ** 8, 111_111_111, 120_000_000, 306_783_000,
                 306_784_000, 1 << 29, (1 << 30) - 1, 1 << 30, (1 << 31) - 1):
        split = f(n, tq, mq, keys, hq, hk, d) > 0
        assert not split or 5 * tiles * (keys + 192) < 1 << 31, keys
        seen.add(split)
    assert seen == {False, True}
    assert f(n, tq, mq, (1 << 31) - 1, hq, hk, d) == 0


def test_split_prefill_takes_long_streams_that_fit():
    f = L.lib().nkv_scaled_prefill_workspace_bytes
    assert f(1, 8, 8, 111_110_000, 4, 1, 64) > 0 == f(1, 8, 8, 111_112_000, 4, 1, 64)


@pytest.mark.parametrize("n", [(1 << 27) - 1023, 1 << 27, (1 << 31) - 1])
def test_store_refuses_more_tokens_than_a_launch_holds(n):
    """Four waves to a workgroup, a workgroup for eight tokens: threads of a launch are 32 bits."""
    assert L.lib().nkv_scaled_store(_args(STORE, n=n)) == -4
    assert b"at most" in L.lib().nkv_last_error()


@pytest.mark.parametrize("kw", [
    dict(n=1 << 20, tq=1 << 20, mq=1, hq=16, hk=16, qrs=1024, ors=1024),   # a tile for each row and head
    dict(n=2, tq=1 << 30, mq=1 << 30, hq=8, hk=8)])
def test_prefill_refuses_more_tiles_than_a_launch_holds(kw):
    assert L.lib().nkv_scaled_prefill(_args(PREFILL, **kw)) == -4
    assert b"too many tiles" in L.lib().nkv_last_error()


# ---------------------------------------------------------------- what the header says of precision
@pytest.mark.parametrize("top", [1.0, 3.5e4, 448.0, 449.0, 1.7e-20, 2.9e38])
def test_values_far_below_their_tile_s_largest(top):
    """Down to 2^-13 of it four significant bits are kept (E4M3's normal codes begin at 2^-6 of the scale, the
    largest value is below 448 of it: 2^-14.9); below 2^-19 nothing is (half of 2^-9, over 224: 2^-17.9)."""
    top = torch.tensor(top, dtype=BF).item()
    e = exponent(top)
    kept = [m * 2.0 ** (math.floor(math.log2(top)) - 3 - k) for m in range(8, 16) for k in range(1, 13)]
    kept = torch.tensor([v for v in kept if top * 2.0 ** -13 <= v <= top], dtype=torch.float64)
    assert kept.numel() > 80
    back = codes_of(kept[:, None], e).view(torch.float8_e4m3fn).double() * 2.0 ** e
    assert torch.equal(back[:, 0], kept)
    assert not bool((codes_of(torch.tensor([[top * 2.0 ** -19, -top * 2.0 ** -25]]).double(), e) & 0x7f).any())


def test_rows_that_are_rounded_again_at_each_growth():
    """32 tokens stored one at a time, the scale raised by each: what the first ones hold moves by less than
    one subnormal step of the last scale. A rollback leaves the scale; the tile's first row takes it back."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(32, 1, 64, generator=g).double()
    x *= 2.0 ** (torch.arange(32).double() * 0.6).view(32, 1, 1)
    x = x.to(BF)
    c = torch.zeros(1, 32, 64 + PAD, dtype=U8)
    held, scales = [], []
    for i in range(32):
        scaled_store_ref(x[i:i + 1], x[i:i + 1], c, c.clone(), torch.tensor([i], dtype=I32))
        held.append(scaled_rows_ref(c, False, [0], i + 1, 1, 64)[i])
        scales.append(int(c.view(-1)[32 * 64]) - 127)
    assert len(set(scales)) > 15
    step = 2.0 ** (scales[-1] - 9)
    moved = (scaled_rows_ref(c, False, [0], 32, 1, 64) - torch.stack(held)).abs().max().item()
    assert 0 < moved < step
    scaled_store_ref(x[3:4], x[3:4], c, c.clone(), torch.tensor([3], dtype=I32))  # rolled back to three
    assert int(c.view(-1)[32 * 64]) - 127 == scales[-1]
    scaled_store_ref(x[:1], x[:1], c, c.clone(), torch.tensor([0], dtype=I32))
    assert int(c.view(-1)[32 * 64]) - 127 == scales[0]
