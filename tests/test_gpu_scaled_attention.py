"""Attention over block-scaled caches, of single tokens and of prompts, against the definition in 64 bits.

The tolerance, from the roundings that the kernels make. Codes widen exactly to bf16, and q is bf16: the
products of a score are exact, its sum is off by at most D steps of 2^-24 of sum |q_d k_d|, and scale and
log2(e) by three more; with m = scale * max_k sum_d |q_d k_d| a weight is off by (D + 3) 2^-24 m of itself
through its score, and as much through the row's maximum, which divides out. A weight then rounds to
bf16, by at most u = eps / 2 = 2^-8 of itself. Weights off by r of themselves, and their sum that of the
weights as they are off, move an output by at most r (sum_k p_k |v_k| + |o|) (1 + 2 r); the output rounds by
u |o|. fp32 sums over the keys and exp2 add less than 2^-16 of sum_k p_k |v_k|.
"""
import importlib
import random

import pytest
import torch

from oracle.scaled_ref import PAD, TILE, attention_rows_ref, scaled_rows_ref
from scaled_util import BF, I32, U8, cache_of, tables_of, values

pytestmark = pytest.mark.gpu

nkv = importlib.import_module("nanokv-llm_amd")
L = importlib.import_module("nanokv-llm_amd._lib")
U = torch.finfo(BF).eps / 2


def reference(q, k, v, scale):
    """-> (o, tolerance) of causal rows q [Lq, Hq, D] over k, v [Lk, Hk, D] in 64 bits."""
    D, Hq, Hk = q.size(2), q.size(1), k.size(1)
    o = attention_rows_ref(q, k, v, scale)
    spread = attention_rows_ref(q, k, v.abs(), scale)  # sum_k p_k |v_k|
    big = torch.zeros(q.size(0), Hq, 1, dtype=torch.float64)
    if k.size(0):
        for h in range(Hq):
            kk = k[:, h * Hk // Hq].nan_to_num().abs()
            big[:, h, 0] = (q[:, h].double().abs() @ kk.t()).amax(1) * scale
    r = U + 2 * (D + 3) * 2.0 ** -24 * big
    return o, r * (1 + 2 * r) * (spread + o.abs()) + U * o.abs() + 2.0 ** -16 * spread + 1e-30


def close(got, want, tol, what=""):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), what
    bad = ((got - want).abs() > tol) & ~want.isnan()
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / tol).nan_to_num()
                                                             .max()))


def make(dev, lens, Hk, D, B, seed=0, width=None, spare=2, garbage=True):
    """Caches that hold each sequence's rows; behind their ends, and in spare blocks, any bytes."""
    g = torch.Generator().manual_seed(seed)
    bt, NB = tables_of(lens, B, seed, width, spare)
    c = {}
    for name, is_v in (("k", False), ("v", True)):
        cache = cache_of(values(NB * B, Hk, D, g).view(NB, B, Hk, D), is_v)
        if garbage:  # codes of NaN behind the ends
            from oracle.scaled_ref import places
            mem, place = cache.view(NB, B // TILE, -1), places(D)[int(is_v)]
            for i, n in enumerate(lens):
                for p in range(n, -(-n // B) * B):
                    t = mem[int(bt[i, p // B]), p % B // TILE]
                    t[:TILE * Hk * D].view(Hk, -1)[:, place[p % TILE]] = 0x7f
        c[name] = cache
    return dict(c, bt=bt, lens=lens, Hk=Hk, D=D, B=B, g=g)


def rows(c, i, n, zeros=False):
    return [scaled_rows_ref(c[x], x == "v", c["bt"][i].tolist(), n, c["Hk"], c["D"], zeros=zeros)
            for x in "kv"]


def gpu(dev, c):
    return c["k"].to(dev), c["v"].to(dev), c["bt"].to(dev)


# ---------------------------------------------------------------- single tokens
def check_decode(dev, c, Hq, scale=None, lens=None, **kw):
    lens = c["lens"] if lens is None else lens
    D = c["D"]
    scale = D ** -0.5 if scale is None else scale
    q = values(len(lens), Hq, D, c["g"], outliers=False)
    k, v, bt = gpu(dev, c)
    got = nkv.scaled_paged_decode(q.to(dev), k, v, torch.tensor(lens, dtype=I32, device=dev), bt, scale,
                                  **kw)
    for i, n in enumerate(lens):
        n = min(max(n, 0), bt.size(1) * c["B"])
        close(got[i:i + 1], *reference(q[i:i + 1], *rows(c, i, n), scale), what=(i, n))
    return got


DECODES = [
    # lens, Hq, Hk, D, B
    ([1], 1, 1, 64, 32), ([1, 0, 2], 2, 1, 128, 32), ([31, 32, 33, 64, 65], 4, 2, 64, 32),
    ([31, 32, 33, 64, 65], 8, 2, 128, 32), ([127, 0, 128, 129, 300], 6, 6, 64, 64),
    ([500, 3, 777], 40, 8, 128, 96), ([900, 100], 16, 1, 128, 32), ([333, 20, 64], 17, 1, 64, 64),
    ([200, 47], 40, 1, 128, 32), ([90, 161], 256, 1, 64, 32), ([100, 95], 66, 2, 128, 32),
    ([1500], 7, 1, 64, 32), ([2100], 32, 8, 64, 32), ([10] * 70, 2, 2, 64, 32),
    ([0, 0, 0], 4, 2, 64, 32), (list(range(1, 40)), 4, 4, 64, 32),
]


@pytest.mark.parametrize("lens,Hq,Hk,D,B", DECODES)
def test_decode(dev, lens, Hq, Hk, D, B):
    check_decode(dev, make(dev, lens, Hk, D, B, seed=len(lens)), Hq)


def test_decode_long_one_over_every_wave(dev):
    """One sequence cut over the whole chip: as many partials as there are."""
    c = make(dev, [20000], 1, 64, 256, garbage=False)
    check_decode(dev, c, 8)


def test_decode_scales(dev):
    for scale in (1e-3, 0.3, 3.0):  # flat, and one key that takes all
        check_decode(dev, make(dev, [70, 200, 33], 2, 128, 32, seed=3), 4, scale)


def test_decode_blocks_that_are_not_there(dev):
    """An invalid block's keys are left out, lengths past the table end with it, below 0 none."""
    c = make(dev, [150, 96, 64, 40, 96], 2, 64, 32, width=5)
    c["bt"][0, 1] = -1
    c["bt"][0, 4] = 10 ** 6
    c["bt"][1, :] = -1                      # nothing at all: zeros
    c["bt"][4, 2] = c["k"].size(0)
    got = check_decode(dev, c, 4, lens=[150, 96, 10 ** 6, -3, 96])
    assert not bool(got[1].any()) and not bool(got[3].any())


def test_decode_rows_apart_and_a_given_workspace(dev):
    """q and out as parts of wider rows; the workspace holds whatever the call before left."""
    c = make(dev, [100, 33, 290], 2, 128, 32, seed=5)
    k, v, bt = gpu(dev, c)
    lens = torch.tensor(c["lens"], dtype=I32, device=dev)
    q = values(3, 8, 128, c["g"], outliers=False).to(dev)
    want = nkv.scaled_paged_decode(q[:, 2:6].contiguous(), k, v, lens, bt, 0.1)
    nbytes = L.lib().nkv_paged_decode_workspace_bytes(3, 4, 128, bt.size(1), 32)
    ws = torch.full((nbytes,), 255, dtype=U8, device=dev)
    out = torch.full((5, 8, 128), 3.0, dtype=BF, device=dev)
    for _ in range(2):
        nkv.scaled_paged_decode(q[:, 2:6], k, v, lens, bt, 0.1, out=out[1:4, 4:], workspace=ws)
    assert torch.equal(out[1:4, 4:], want)
    assert bool((out[:, :4] == 3).all()) and bool((out[[0, 4]] == 3).all())


def test_decode_nan_and_infinite_values_that_are_seen(dev):
    """A row that sees NaN is NaN; the other sequences and heads are not."""
    c = make(dev, [40, 70, 33], 2, 64, 32, seed=6)
    from oracle.scaled_ref import places
    t = c["k"].view(c["k"].size(0), -1, TILE * (2 * 64 + PAD))[int(c["bt"][1, 1]), 0]
    t[places(64)[0][5, 7]] = 0xff           # key 37 of sequence 1, head 0
    t = c["v"].view(c["v"].size(0), -1, TILE * (2 * 64 + PAD))[int(c["bt"][0, 1]), 0]
    t[TILE * 64 + places(64)[1][3, 9]] = 0x7f  # value 35 of sequence 0, head 1, dim 9
    got = check_decode(dev, c, 4)
    assert bool(got[1, :2].isnan().all()) and not bool(got[1, 2:].isnan().any())
    assert bool(got[0, 2:, 9].isnan().all()) and int(got[0].isnan().sum()) == 2


def test_decode_captured(dev):
    c = make(dev, [100, 33, 64, 1], 2, 128, 32, seed=7, width=6)
    k, v, bt = gpu(dev, c)
    lens = torch.tensor(c["lens"], dtype=I32, device=dev)
    q = values(4, 8, 128, c["g"], outliers=False).to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nkv.scaled_paged_decode(q, k, v, lens, bt, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nkv.scaled_paged_decode(q, k, v, lens, bt, 0.1)
    for i in range(4):
        q.copy_(values(4, 8, 128, c["g"], outliers=False))
        lens.copy_(torch.tensor([96 - 30 * i, 33 - i, 64 - 20 * i, i], dtype=I32))
        graph.replay()
        want = nkv.scaled_paged_decode(q, k, v, lens, bt, 0.1)
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))  # NaN among them


# ---------------------------------------------------------------- prompts
def check_prefill(dev, c, new, Hq, scale=None, split=True, lens=None):
    lens = c["lens"] if lens is None else lens
    D = c["D"]
    scale = D ** -0.5 if scale is None else scale
    cu_q, cu_k = [0], [0]
    for a, b in zip(new, lens):
        cu_q.append(cu_q[-1] + a)
        cu_k.append(cu_k[-1] + b)
    N = cu_q[-1]
    q = values(N + 3, Hq, D, c["g"], outliers=False)
    k, v, bt = gpu(dev, c)
    i32 = dict(dtype=I32, device=dev)
    out = torch.full((N + 3, Hq, D), 3.0, dtype=BF, device=dev)
    got = nkv.scaled_varlen_prefill(q.to(dev), k, v, torch.tensor(cu_q, **i32),
                                    torch.tensor(cu_k, **i32), max(new), scale, bt, out=out,
                                    max_seqlen_k=max(lens) if split else None)
    assert got is out and bool((out[N:] == 3).all())
    for i, (a, b) in enumerate(zip(new, lens)):
        close(got[cu_q[i]:cu_q[i + 1]],
              *reference(q[cu_q[i]:cu_q[i + 1]], *rows(c, i, b, zeros=True), scale), what=(i, a, b))
    return got


PREFILLS = [
    # new, lens, Hq, Hk, D, B
    ([1], [1], 1, 1, 64, 32), ([2, 1], [2, 40], 2, 1, 128, 32),
    ([31, 32, 33], [31, 32, 33], 4, 2, 64, 32), ([31, 32, 33], [64, 100, 33], 4, 2, 128, 32),
    ([70, 1, 0, 5], [70, 130, 0, 64], 6, 6, 64, 64), ([100], [165], 40, 8, 64, 96),
    ([20, 3], [300, 40], 24, 1, 128, 32), ([9], [70], 128, 1, 64, 32), ([5, 7], [40, 90], 65, 1, 128, 32),
    ([200, 130], [200, 260], 2, 2, 64, 32), ([129], [129], 1, 1, 128, 256),
    ([1] * 20, list(range(1, 21)), 4, 2, 64, 32), ([6], [1300], 8, 2, 64, 32),
    ([3, 4, 1], [900, 20, 400], 8, 1, 128, 64),
]


@pytest.mark.parametrize("split", [True, False])
@pytest.mark.parametrize("new,lens,Hq,Hk,D,B", PREFILLS)
def test_prefill(dev, new, lens, Hq, Hk, D, B, split):
    check_prefill(dev, make(dev, lens, Hk, D, B, seed=len(new)), new, Hq, split=split)


def test_prefill_row_groups(dev):
    """Enough tiles for the larger ones: some of a tile's rows past the sequence's end."""
    for D in (64, 128):
        check_prefill(dev, make(dev, [37] * 40, 8, D, 64, seed=D, garbage=False), [37] * 40, 16)


@pytest.mark.parametrize("new,lens,Hq,Hk,D", [
    ([50, 200, 90], [400, 230, 90], 512, 8, 128),  # three row groups a wave, longest first
    ([200, 5, 210], [200, 300, 211], 256, 8, 64),  # two
    ([3] * 70, [3 + 5 * i for i in range(70)], 32, 2, 128),  # more sequences than are sorted
])
def test_prefill_more_tiles_than_the_chip_holds(dev, new, lens, Hq, Hk, D):
    check_prefill(dev, make(dev, lens, Hk, D, 64, seed=D + len(new), garbage=False), new, Hq)


@pytest.mark.parametrize("n,D", [(65, 128), (70, 64), (200, 64), (4200, 64)])
def test_prefill_many_sequences_of_few_and_of_many_tiles(dev, n, D):
    """More sequences than a wave has lanes, some with more tiles than one, some without a query."""
    rng = random.Random(n)
    new = [rng.choice([0, 1, 1, 1, 2, 9, rng.randint(1, 30)]) if i % (n // 65) == 0 else rng.choice([0, 0, 1])
           for i in range(n)]
    new[-1], new[0] = 25, 17
    lens = [a + rng.choice([0, 1, 5, 40]) for a in new]
    check_prefill(dev, make(dev, lens, 1, D, 32, seed=n, garbage=False), new, 8)


@pytest.mark.parametrize("new,lens,Hq,Hk,D", [
    ([100, 130], [2000, 1500], 64, 8, 128), ([100, 130], [2000, 1500], 64, 8, 64),
    ([1] * 70 + [9], [7 * i + 1 for i in range(70)] + [1000], 4, 1, 64),
    ([65, 1, 0, 4, 66], [65, 1200, 0, 4, 900], 4, 2, 128),
])
def test_prefill_ranges_of_many_units(dev, new, lens, Hq, Hk, D):
    """Ranges that hold whole units and parts of others, of sequences past a wave's lanes too."""
    assert L.lib().nkv_scaled_prefill_workspace_bytes(len(new), sum(new) + 3, max(new), max(lens), Hq,
                                                      Hk, D) > 0
    check_prefill(dev, make(dev, lens, Hk, D, 64, seed=D + len(new)), new, Hq)


@pytest.mark.parametrize("split", [True, False])
def test_prefill_rows_that_see_nothing(dev, split):
    """More queries than keys: the first rows see no key and are zeros."""
    c = make(dev, [3, 0, 40, 600], 2, 64, 32, seed=8)
    got = check_prefill(dev, c, [7, 2, 41, 601], 4, split=split)
    assert not bool(got[:4].any()) and not bool(got[7:9].any()) and not bool(got[9].any())
    assert bool(got[4].any())


@pytest.mark.parametrize("D", [64, 128])
def test_prefill_nan_among_keys_that_rows_do_not_see(dev, D):
    """NaN in K and in V of a prompt's later keys: rows before them are as if it were not there."""
    from oracle.scaled_ref import places
    Hk = 2
    c = make(dev, [150, 80], Hk, D, 32, seed=9)
    mem = {x: c[x].view(c[x].size(0), -1) for x in "kv"}
    for i, p, h, dim, x in ((0, 100, 0, 3, "v"), (0, 133, 1, D - 1, "v"), (0, 120, 1, 5, "k"),
                            (1, 79, 0, 0, "v"), (1, 70, 1, 17, "v")):
        at = h * TILE * D + int(places(D)[int(x == "v")][p % TILE, dim])
        mem[x][int(c["bt"][i, p // 32]), at] = 0x7f
    for split in (True, False):
        got = check_prefill(dev, c, [120, 70], 4, split=split)
        assert not bool(got[:70].isnan().any()) and bool(got[189].isnan().any())


@pytest.mark.parametrize("split", [True, False])
def test_prefill_blocks_that_are_not_there(dev, split):
    """Zeros in their place, as in varlen_prefill; a length past the table as well."""
    c = make(dev, [150, 96, 700], 2, 64, 32, width=22, seed=10)
    c["bt"][0, 1] = -1
    c["bt"][1, :] = 10 ** 6
    c["bt"][2, 20] = -5
    check_prefill(dev, c, [50, 96, 6], 4, split=split, lens=[150, 96, 720])


def splits(new, lens, Hq, Hk, D):
    return L.lib().nkv_scaled_prefill_workspace_bytes(len(new), sum(new) + 3, max(new), max(lens), Hq,
                                                      Hk, D) > 0


def test_prefill_ranges_of_rows_that_see_nothing(dev):
    new, lens = [7, 2, 41, 1301, 5], [3, 0, 40, 1300, 1000]
    assert splits(new, lens, 4, 2, 64)
    got = check_prefill(dev, make(dev, lens, 2, 64, 32, seed=18), new, 4)
    assert not bool(got[:4].any()) and not bool(got[7:9].any()) and not bool(got[9].any())
    assert not bool(got[50].any()) and bool(got[51].any())


@pytest.mark.parametrize("D", [64, 128])
def test_prefill_ranges_of_keys_that_rows_do_not_see(dev, D):
    """NaN in later keys, of units that one wave takes a row group of and of those that two share."""
    from oracle.scaled_ref import places
    Hk, lens, new = 2, [1100, 900, 1000], [20, 70, 5]
    assert splits(new, lens, 4, Hk, D)
    c = make(dev, lens, Hk, D, 32, seed=19)
    mem = {x: c[x].view(c[x].size(0), -1) for x in "kv"}
    for i, p, h, dim, x in ((0, 1091, 0, 3, "v"), (0, 1095, 1, D - 1, "v"), (0, 1097, 1, 5, "k"),
                            (1, 860, 0, 0, "v"), (1, 897, 1, 17, "k"), (2, 999, 1, 1, "v")):
        at = h * TILE * D + int(places(D)[int(x == "v")][p % TILE, dim])
        mem[x][int(c["bt"][i, p // 32]), at] = 0x7f
    got = check_prefill(dev, c, new, 4)
    assert not bool(got[:11].isnan().any()) and bool(got[19].isnan().any())
    assert not bool(got[20:50].isnan().any()) and bool(got[89].isnan().any())
    assert not bool(got[90:94].isnan().any()) and bool(got[94].isnan().any())


def test_prefill_ranges_over_blocks_that_are_not_there(dev):
    new, lens = [50, 96, 6], [150, 96, 1320]
    assert splits(new, lens, 4, 2, 64)
    c = make(dev, [150, 96, 1300], 2, 64, 32, width=41, seed=20)
    c["bt"][0, 1] = -1
    c["bt"][1, :] = 10 ** 6
    c["bt"][2, 20:23] = -5
    check_prefill(dev, c, new, 4, lens=lens)


def test_two_streams_at_once(dev):
    """Calls that overlap, each with what it allocates: as one after the other."""
    new, lens = [9, 70, 1, 5], [1500, 1300, 900, 1100]
    c = make(dev, lens, 2, 64, 32, seed=21, garbage=False)
    k, v, bt = gpu(dev, c)
    i32 = dict(dtype=I32, device=dev)
    q = values(sum(new), 8, 64, c["g"], outliers=False).to(dev)
    cu_q, cu_k = ([sum(x[:i]) for i in range(len(x) + 1)] for x in (new, lens))
    args = (torch.tensor(cu_q, **i32), torch.tensor(cu_k, **i32), max(new), 0.1, bt)
    ctx = torch.tensor(lens, **i32)
    want = (nkv.scaled_varlen_prefill(q, k, v, *args, max_seqlen_k=max(lens)),
            nkv.scaled_paged_decode(q[:4], k, v, ctx, bt, 0.1))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, nkv.scaled_varlen_prefill(q, k, v, *args, max_seqlen_k=max(lens))
                            if i < 2 else nkv.scaled_paged_decode(q[:4], k, v, ctx, bt, 0.1)))
    torch.cuda.synchronize()
    for i, x in got:
        assert torch.equal(x, want[i == 2])


def test_prefill_sequences_outside_the_rows(dev):
    """cu_seqlens_q that names rows which q does not have: left out, nothing else touched."""
    c = make(dev, [40, 40, 40], 2, 64, 32, seed=11)
    k, v, bt = gpu(dev, c)
    q = values(60, 4, 64, c["g"], outliers=False).to(dev)
    i32 = dict(dtype=I32, device=dev)
    cu_k = torch.tensor([0, 40, 80, 120], **i32)
    for mk in (None, 100000):
        want = nkv.scaled_varlen_prefill(q, k, v, torch.tensor([0, 30, 60, 60], **i32), cu_k, 40, 0.1,
                                         bt)
        for cu in ([0, 30, 60, 100], [-20, 30, 60, 61]):
            out = torch.full_like(q, 3.0)
            nkv.scaled_varlen_prefill(q, k, v, torch.tensor(cu, **i32), cu_k, 40, 0.1, bt, out=out,
                                      max_seqlen_k=mk)
            ok = slice(0, 60) if cu[0] == 0 else slice(30, 60)
            assert torch.equal(out[ok], want[ok]) and bool((out[:ok.start] == 3).all())


def test_prefill_rows_apart_and_a_given_workspace(dev):
    c = make(dev, [900, 300], 2, 128, 32, seed=12, garbage=False)
    k, v, bt = gpu(dev, c)
    i32 = dict(dtype=I32, device=dev)
    cu_q, cu_k = torch.tensor([0, 3, 8], **i32), torch.tensor([0, 900, 1200], **i32)
    q = values(8, 8, 128, c["g"], outliers=False).to(dev)
    want = nkv.scaled_varlen_prefill(q[:, 2:6].contiguous(), k, v, cu_q, cu_k, 5, 0.1, bt,
                                     max_seqlen_k=900)
    nbytes = L.lib().nkv_scaled_prefill_workspace_bytes(2, 8, 5, 900, 4, 2, 128)
    assert nbytes > 0
    ws = torch.full((nbytes,), 255, dtype=U8, device=dev)
    out = torch.full((10, 8, 128), 3.0, dtype=BF, device=dev)
    for _ in range(2):
        nkv.scaled_varlen_prefill(q[:, 2:6], k, v, cu_q, cu_k, 5, 0.1, bt, out=out[1:9, 4:],
                                  max_seqlen_k=900, workspace=ws)
    assert torch.equal(out[1:9, 4:], want)
    assert bool((out[:, :4] == 3).all()) and bool((out[[0, 9]] == 3).all())


def test_prefill_of_nothing(dev):
    c = torch.zeros(1, 32, 64 + PAD, dtype=U8, device=dev)
    z, bt = torch.zeros(1, dtype=I32, device=dev), torch.zeros(1, 1, dtype=I32, device=dev)
    q = torch.zeros(0, 2, 64, dtype=BF, device=dev)
    assert nkv.scaled_varlen_prefill(q, c, c, z, z, 0, 0.1, bt).shape == q.shape
    assert nkv.scaled_paged_decode(q, c, c, z, bt, 0.1).shape == q.shape


@pytest.mark.parametrize("new,lens", [([40, 1], [100, 70]), ([3, 2], [900, 500])])
def test_prefill_captured(dev, new, lens):
    c = make(dev, lens, 2, 64, 32, seed=13)
    k, v, bt = gpu(dev, c)
    i32 = dict(dtype=I32, device=dev)
    cu_q = torch.tensor([0, new[0], sum(new)], **i32)
    cu_k = torch.tensor([0, lens[0], sum(lens)], **i32)
    q = values(sum(new), 4, 64, c["g"], outliers=False).to(dev)
    args = (k, v, cu_q, cu_k, max(new), 0.1, bt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        nkv.scaled_varlen_prefill(q, *args, max_seqlen_k=max(lens))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nkv.scaled_varlen_prefill(q, *args, max_seqlen_k=max(lens))
    for i in range(4):
        q.copy_(values(sum(new), 4, 64, c["g"], outliers=False))
        cu_k.copy_(torch.tensor([0, lens[0] - 7 * i, sum(lens) - 20 * i], dtype=I32))
        graph.replay()
        want = nkv.scaled_varlen_prefill(q, *args, max_seqlen_k=max(lens))
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))  # NaN among them


def test_past_four_gib(dev):
    """Blocks whose bytes lie past 2^32: the same results as from a small cache."""
    Hk, D, B = 8, 128, 256
    NB = (1 << 32) // (B * (Hk * D + PAD)) + 40
    c = make(dev, [300, 100], Hk, D, B, seed=14, garbage=False)
    k, v, bt = gpu(dev, c)
    big = [torch.zeros(NB, B, Hk * D + PAD, dtype=U8, device=dev) for _ in range(2)]
    for x, y in zip(big, (k, v)):
        x[-k.size(0):] = y
    far = torch.where(bt >= 0, bt + NB - k.size(0), bt)
    lens = torch.tensor([300, 100], dtype=I32, device=dev)
    q = values(2, 16, D, c["g"], outliers=False).to(dev)
    assert torch.equal(nkv.scaled_paged_decode(q, *big, lens, far, 0.1),
                       nkv.scaled_paged_decode(q, k, v, lens, bt, 0.1))
    cu_q = torch.tensor([0, 70, 80], dtype=I32, device=dev)
    cu_k = torch.tensor([0, 300, 400], dtype=I32, device=dev)
    q = values(80, 16, D, c["g"], outliers=False).to(dev)
    assert torch.equal(nkv.scaled_varlen_prefill(q, *big, cu_q, cu_k, 70, 0.1, far, max_seqlen_k=300),
                       nkv.scaled_varlen_prefill(q, k, v, cu_q, cu_k, 70, 0.1, bt, max_seqlen_k=300))
