"""Block-scaled caches: sizes at the ends of what the calls take, none of which needs a GPU."""
import struct

import pytest

from test_scaled_checks import L, P, PREFILL, STORE


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
