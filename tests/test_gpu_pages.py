"""PagedSequences against the sequential oracle: state, statuses, slots and every copied byte.

All outputs are whole numbers or copied rows, so every comparison is for equality.
"""
import copy
import gc
import importlib
import random

import pytest
import torch

from oracle.attention_ref import paged_decode_ref
from oracle.pages_ref import PagedSequencesRef
from test_pages_checks import free_page_listed

pytestmark = pytest.mark.gpu

nkv = importlib.import_module("nanokv-llm_amd")
I32 = torch.int32


def ints(x, dev):
    return torch.tensor(x, dtype=I32, device=dev)


class Pair:
    """The operators and the oracle over equal pools; every call is made on both and compared."""

    def __init__(self, dev, layers=2, pages=40, block=16, heads=2, dim=64, rows=8, width=6,
                 dtype=torch.bfloat16, seed=0):
        g = torch.Generator().manual_seed(seed)
        raw = torch.randint(-100, 100, (2, layers, pages, block, heads, dim), generator=g)
        self.bits = torch.int8 if dtype == torch.float8_e4m3fn else torch.int16
        self.ref = PagedSequencesRef(raw.to(self.bits), rows, width)
        self.kv = raw.to(self.bits).to(dev).view(dtype)
        self.seqs = nkv.PagedSequences(self.kv, rows, width)
        self.dev, self.S, self.B = dev, rows, block

    def check(self, got, want):
        assert got.cpu().tolist() == list(want)
        assert torch.equal(self.seqs.state.cpu(), self.ref.state())
        assert torch.equal(self.kv.view(self.bits).cpu(), self.ref.kv)

    def append(self, rows, counts=None):
        if counts is None:
            slots, status = self.seqs.append(ints(rows, self.dev))
            want_slots, want = self.ref.append(rows)
        else:
            cu = [0]
            for c in counts:
                cu.append(cu[-1] + c)
            return self.append_cu(rows, cu, cu[-1])
        assert slots.cpu().tolist() == want_slots
        self.check(status, want)
        return want

    def append_cu(self, rows, cu, n_tokens):
        slots, status = self.seqs.append(ints(rows, self.dev), ints(cu, self.dev), n_tokens)
        want_slots, want = self.ref.append(rows, cu=cu, n_tokens=n_tokens)
        assert slots.cpu().tolist() == want_slots
        self.check(status, want)
        return want

    def truncate(self, rows, lens, pages=None):
        got = self.seqs.truncate(ints(rows, self.dev), ints(lens, self.dev),
                                 None if pages is None else ints(pages, self.dev))
        want = self.ref.truncate(rows, lens, pages or ())
        self.check(got, want)
        return want

    def fork(self, parents, children, share=True):
        got = self.seqs.fork(ints(parents, self.dev), ints(children, self.dev), share)
        want = self.ref.fork(parents, children, share)
        self.check(got, want)
        return want

    def compact(self, max_moves):
        info, moves = self.seqs.compact(max_moves)
        want_info, want_moves = self.ref.compact(max_moves)
        assert moves.cpu().tolist() == want_moves
        self.check(info, want_info)
        return want_info


def test_append_one_token_each(dev):
    p = Pair(dev)
    for _ in range(40):
        p.append(list(range(8)))
    assert p.ref.lens == [40] * 8


def test_append_lengths_around_a_page(dev):
    p = Pair(dev, rows=6, width=4)
    assert p.append([0, 1, 2, 3, 4, 5], [0, 1, 15, 16, 17, 64]) == [1] * 6
    assert p.append([5, 4, 0], [1, 0, 3]) == [0, 1, 1]  # row 5 is at its table's width
    assert p.append([1, 2, 3], [16, 1, 32]) == [1, 1, 1]


def test_append_refuses_in_order_when_pages_run_out(dev):
    p = Pair(dev, pages=5, rows=5, width=6)
    assert p.append([0, 1, 2, 3], [32, 20, 33, 1]) == [1, 1, 0, 0]
    assert p.append([1, 2, 0], [10, 1, 1]) == [1, 1, 0]  # row 1 has room in its page
    assert p.append([3, 1], [0, 2]) == [1, 1]


def test_lists_with_padding_repeats_and_rows_outside(dev):
    p = Pair(dev)
    assert p.append([-1, 3, 3, 8, 2, -7, 2 ** 30], [4, 5, 6, 7, 8, 1, 1]) == [0, 1, 0, 0, 1, 0, 0]
    assert p.append([3, -1, 3]) == [1, 0, 0]
    assert p.fork([3, 3, 2, 9, -1], [4, 4, -1, 5, 6]) == [1, 0, 0, 0, 0]
    assert p.truncate([-1, 2, 2, 77], [0, 3, 1, 0]) == [0, 1, 0, 0]


@pytest.mark.parametrize("cu,n_tokens", [([0, 5, 3, 9], 9), ([-1, 2, 3, 4], 9),
                                         ([0, 2, 5, 10], 9), ([0, 0, 2 ** 30, 4], 9)])
def test_append_refuses_cu_seqlens_out_of_order_or_range(dev, cu, n_tokens):
    assert Pair(dev).append_cu([0, 1, 2], cu, n_tokens) == [0, 0, 0]


def test_append_slots_outside_cu_seqlens_are_padding(dev):
    p = Pair(dev)
    assert p.append_cu([0, 1], [3, 5, 25], 31) == [1, 1]
    assert p.append_cu([], [0], 7) == []
    assert p.append([]) == []
    assert p.append([0, 1], [0, 0]) == [1, 1]


def test_truncate_frees_and_rolls_back(dev):
    p = Pair(dev)
    p.append([0, 1, 2], [50, 33, 16])
    assert p.truncate([0, 1, 2], [51, -1, 16]) == [0, 0, 1]  # more than there is; nothing dropped
    assert p.truncate([0, 1], [17, 32]) == [1, 1]
    assert p.truncate([2, 0], [0, 0]) == [1, 1]
    assert p.append([3], [60]) == [1]


def test_truncate_inside_a_shared_page_copies_it(dev):
    p = Pair(dev)
    p.append([0], [40])
    p.fork([0, 0], [1, 2])
    assert p.truncate([1], [20]) == [1]      # its page of its own now
    assert p.truncate([0, 2], [7, 7]) == [1, 1]  # both leave the page they share
    p.append([0, 1, 2], [30, 30, 30])
    p.truncate([0, 1, 2], [0, 0, 0])
    assert sum(p.ref.refs) == 0


def test_truncate_refuses_a_copy_without_a_free_page(dev):
    p = Pair(dev, pages=3, rows=4)
    p.append([0], [32])
    p.fork([0], [1])
    assert p.append([2]) == [1]  # the last free page
    assert p.truncate([0, 1, 2], [20, 16, 0]) == [0, 1, 1]
    assert p.truncate([0, 1], [20, 0]) == [1, 1]


def test_truncate_drops_listed_pages(dev):
    p = Pair(dev)
    p.append([0, 1], [64, 40])
    t = p.ref.tables
    # freed by a compression step: listed pages, padding, one twice, one free, ids outside the pool
    assert p.truncate([1], [3], [t[0][3], -1, t[0][3], 39, 40, -9, 2 ** 30]) == [1]
    assert p.truncate([], [], [t[0][2]]) == []
    p.truncate([], [], [])


def test_fork_shares_full_pages_and_copies_the_last(dev):
    p = Pair(dev)
    p.append([0, 1, 2], [35, 32, 5])
    assert p.fork([0, 1, 2, 0], [3, 4, 5, 6]) == [1] * 4
    assert p.fork([3, 7, 0], [0, 7, 1]) == [0, 1, 0]  # children in use; an empty parent
    for _ in range(20):
        p.append([0, 1, 2, 3, 4, 5, 6])


def test_fork_without_sharing_copies_every_page(dev):
    p = Pair(dev)
    p.append([0, 1], [70, 16])
    assert p.fork([0, 1], [2, 3], share=False) == [1, 1]
    assert all(c <= 1 for c in p.ref.refs)


def test_fork_of_an_empty_child_in_the_same_call(dev):
    p = Pair(dev)
    p.append([0], [20])
    assert p.fork([0, 1], [1, 2]) == [1, 1]  # row 1 is empty before the call, so row 2 stays empty
    assert p.ref.lens[:3] == [20, 20, 0]


@pytest.mark.parametrize("max_moves", [0, 1, 5, 100])
def test_compact_moves_the_highest_pages_down(dev, max_moves):
    p = Pair(dev, rows=9)
    p.append(list(range(8)), [80, 16, 64, 3, 50, 33, 20, 41])
    p.fork([4], [8])
    p.truncate([0, 2, 5], [0, 10, 0])
    p.compact(max_moves)
    p.append([0, 2, 5], [30, 30, 30])
    assert p.compact(max_moves)[1] == 0 or max_moves < 100


def test_compact_of_empty_full_and_packed_pools(dev):
    p = Pair(dev, pages=8, rows=3, width=8)
    assert p.compact(8) == [0, 0]
    p.append([0, 1], [64, 64])
    assert p.compact(8) == [8, 0]
    p.truncate([1], [0])
    assert p.compact(8) == [4, 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float8_e4m3fn])
@pytest.mark.parametrize("layers,block,heads,dim", [(1, 16, 1, 64), (3, 48, 2, 128), (2, 256, 8, 128),
                                                    (5, 32, 3, 64)])
def test_random_programs(dev, dtype, layers, block, heads, dim):
    rng = random.Random(layers * 1000 + block)
    p = Pair(dev, layers, 37, block, heads, dim, rows=11, width=7, dtype=dtype, seed=block)
    for _ in range(40):
        rows = [rng.randrange(-2, 13) for _ in range(rng.randint(0, 9))]
        op = rng.choice(["one", "many", "many", "truncate", "truncate", "fork", "fork", "copy",
                         "compact"])
        if op == "one":
            p.append(rows)
        elif op == "many":
            p.append(rows, [rng.choice([0, 1, block - 1, block, rng.randint(0, 3 * block)])
                            for _ in rows])
        elif op == "truncate":
            keep = [rng.randint(-1, p.ref.lens[r] + 1) if 0 <= r < 11 else 0 for r in rows]
            p.truncate(rows, keep)
        elif op == "compact":
            p.compact(rng.choice([0, 1, 3, 50]))
        else:
            p.fork([rng.randrange(-1, 12) for _ in rows], rows, op == "fork")


def test_many_rows_and_pages(dev):
    """More list entries than the plan has threads, and more pages than one step of its walk."""
    p = Pair(dev, layers=1, pages=40_000, block=16, heads=1, dim=8, rows=3000, width=20)
    rng = random.Random(3)
    rows = list(range(3000))
    rng.shuffle(rows)
    p.append(rows, [rng.randint(0, 200) for _ in rows])
    p.append(rows)
    p.truncate(rows[:1500], [rng.choice([0, p.ref.lens[r] // 2]) for r in rows[:1500]])
    p.compact(3000)
    p.compact(40_000)
    empty = [r for r in range(3000) if p.ref.lens[r] == 0]
    p.fork([rng.choice(rows) for _ in empty], empty)
    p.append([r for r in rows for _ in (0, 1)])  # every row twice: 6000 entries


def test_a_pool_object_and_a_kept_state(dev):
    pool = nkv.layers.kv_cache.KVCachePool(2, 2, 64, 16, num_blocks=10, device=dev)
    pool.kv_cache.zero_()
    seqs = nkv.PagedSequences(pool, 4, 5)
    seqs.append(ints([0, 1], dev), ints([0, 20, 25], dev), 25)
    kept = seqs.state.clone()
    seqs.truncate(ints([0], dev), ints([0], dev))
    again = nkv.PagedSequences(pool, 4, 5, state=kept)
    assert again.context_lens.tolist() == [20, 5, 0, 0]
    assert again.ref_counts.tolist() == [1, 1, 1] + [0] * 7
    assert again.block_tables[:2].tolist() == [[0, 1, -1, -1, -1], [2, -1, -1, -1, -1]]
    assert seqs.context_lens.tolist() == [0, 5, 0, 0]


def test_calls_on_another_stream(dev):
    p = Pair(dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        p.append([0, 1, 2], [30, 40, 50])
        p.fork([0, 2], [3, 4])
        p.truncate([0, 2], [9, 33])
        p.compact(10)
    s.synchronize()


def test_a_decode_step_captured_in_a_graph(dev):
    """append, store, attention in one graph, replayed with eager calls between: each replay's
    slots, state and outputs are those of the same steps made one after another."""
    H, Hk, D, B, S = 4, 2, 64, 16, 5
    g = torch.Generator().manual_seed(4)
    p = Pair(dev, layers=1, pages=30, block=B, heads=Hk, dim=D, rows=S, width=6)
    p.kv.copy_(torch.randn(p.kv.shape, generator=g).to(torch.bfloat16))
    p.ref.kv = p.kv.view(torch.int16).cpu()
    rows = ints([3, 0, -1, 2, 1], dev)
    q = torch.randn(S, H, D, generator=g).to(torch.bfloat16).to(dev)
    k, v = (torch.randn(S, Hk, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    kc, vc = p.kv[0, 0], p.kv[1, 0]
    p.append([0, 1, 2, 3, 4], [14, 33, 1, 15, 8])
    ws = nkv.layers.attention.paged_decode_workspace(q, kc, p.seqs.block_tables)

    def step():
        slots, status = p.seqs.append(rows)
        nkv.store_kvcache(k, v, kc, vc, slots)
        out = nkv.paged_decode(q, kc, vc, p.seqs.context_lens, p.seqs.block_tables, D ** -0.5,
                               workspace=ws)
        return slots, status, out

    kept, kv = p.seqs.state.clone(), p.kv.clone()
    step()  # warm-up
    torch.cuda.synchronize()
    p.seqs.state.copy_(kept)
    p.kv.copy_(kv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots, status, out = step()
    for i in range(6):
        graph.replay()
        torch.cuda.synchronize()
        want_slots, want = p.ref.append([3, 0, -1, 2, 1])
        assert slots.cpu().tolist() == want_slots and status.cpu().tolist() == want
        flat = p.ref.kv.view(2, -1, Hk, D)
        for t, s in enumerate(want_slots):
            if s >= 0:
                flat[0, s], flat[1, s] = k[t].view(torch.int16).cpu(), v[t].view(torch.int16).cpu()
        p.check(status, want)
        refs = p.ref.kv.view(torch.bfloat16)
        lens = torch.tensor(p.ref.lens, dtype=I32)
        ref = paged_decode_ref(q.float().cpu(), refs[0, 0], refs[1, 0], lens,
                               torch.tensor(p.ref.tables, dtype=I32), D ** -0.5)
        # weights and the output rounded to bf16 (half a step 2^-9 of values up to 4 each)
        assert (out.float().cpu() - ref).abs().max() <= 2 * 4 * 2.0 ** -8
        if i == 2:  # eager work between the replays
            p.truncate([0, 3], [5, 16])
        if i == 3:
            p.fork([1], [4]) if p.ref.lens[4] == 0 else p.truncate([4], [0])


def test_compression_beside_shared_sequences(dev):
    """A copy of a sequence is compressed in place: its freed blocks go back through truncate, the
    shared pages of the others stay as they were, and new tokens take the freed pages."""
    cu = importlib.import_module("nanokv-llm_amd.layers.compress_utils")
    B, Hk, D, W, keep = 256, 2, 128, 4, 257
    g = torch.Generator().manual_seed(9)
    kv = torch.randn(2, 1, 24, B, Hk, D, generator=g).to(torch.bfloat16).to(dev)
    seqs = nkv.PagedSequences(kv, 5, 8)
    n = 5 * B + 20
    seqs.append(ints([0], dev), ints([0, n], dev), n)
    assert seqs.fork(ints([0], dev), ints([1], dev)).tolist() == [1]
    assert seqs.fork(ints([0], dev), ints([2], dev), share_pages=False).tolist() == [1]
    before = kv.clone()
    base = seqs.context_lens.clone()
    q = torch.randn(5, 4, D, generator=g).to(torch.bfloat16).to(dev)
    events = torch.empty(1, 4 + 8, dtype=I32, device=dev)
    cu.compress_step(q, kv[0, 0], kv[1, 0], seqs.block_tables, base, seqs.context_lens,
                     ints([2], dev), W, keep, D ** -0.5, events=events)
    empty = ints([], dev)
    seqs.truncate(empty, empty, pages=events[0, 4:].contiguous())
    held = seqs.block_tables.cpu()
    assert seqs.context_lens.tolist() == [n, n, n - W * B + keep, 0, 0]
    assert seqs.ref_counts.tolist() == [int((held == p).sum()) for p in range(24)]
    for r in (0, 1):
        pages = held[r][held[r] >= 0].long().to(dev)
        assert torch.equal(kv[:, :, pages], before[:, :, pages])
    free = int((seqs.ref_counts == 0).sum())
    slots, status = seqs.append(ints([3], dev), ints([0, free * B], dev), free * B) \
        if free <= 8 else seqs.append(ints([3], dev), ints([0, 8 * B], dev), 8 * B)
    assert status.tolist() == [1] and bool((slots >= 0).all())


def test_two_objects_at_once_on_two_streams(dev):
    """Objects of their own share nothing: their calls may overlap."""
    a, b = Pair(dev, seed=1), Pair(dev, seed=2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s, p in zip(streams, (a, b)):
        with torch.cuda.stream(s):
            out = [p.seqs.append(ints([0, 1, 2], dev), ints([0, 40, 77, 80], dev), 80)[1],
                   p.seqs.fork(ints([0, 1], dev), ints([3, 4], dev)),
                   p.seqs.truncate(ints([0, 3], dev), ints([20, 33], dev)),
                   p.seqs.compact(20)[0]]
            got.append(out)
    torch.cuda.synchronize()
    for p, out in zip((a, b), got):
        want = [p.ref.append([0, 1, 2], cu=[0, 40, 77, 80], n_tokens=80)[1],
                p.ref.fork([0, 1], [3, 4]), p.ref.truncate([0, 3], [20, 33]), p.ref.compact(20)[0]]
        assert [x.tolist() for x in out] == want
        p.check(out[3], want[3])


def test_pages_past_4_gib(dev):
    """Copies whose byte offsets pass 32 bits, in the last plane of a large pool."""
    kv = torch.empty(2, 3, 1300, 256, 8, 128, dtype=torch.bfloat16, device=dev)  # 4.1 GB
    kv.view(torch.int16).fill_(7)
    seqs = nkv.PagedSequences(kv, 3, 1300)
    n = 1296 * 256 + 100
    assert seqs.append(ints([0], dev), ints([0, n], dev), n)[1].tolist() == [1]
    kv[:, :, 1296].view(torch.int16).copy_(
        torch.arange(256 * 8 * 128, device=dev).to(torch.int16).view(256, 8, 128))
    assert seqs.fork(ints([0], dev), ints([1], dev)).tolist() == [1]
    assert seqs.block_tables[1, 1296].item() == 1297
    same = kv[:, :, 1297].view(torch.int16) == kv[:, :, 1296].view(torch.int16)
    assert bool(same[:, :, :100].all())
    assert bool((kv[:, :, 1297, 100:].view(torch.int16) == 7).all())
    assert bool((kv[:, :, 1298:].view(torch.int16) == 7).all())


def test_a_kept_state_taken_back_in_place(dev):
    """state.copy_(kept): views, calls and the next tokens' pages are those of the kept state."""
    p = Pair(dev)
    p.append([0, 1, 2], [20, 33, 5])
    kept, oracle = p.seqs.state.clone(), copy.deepcopy(p.ref)
    views = p.seqs.context_lens, p.seqs.block_tables
    p.append([0, 3], [40, 16])
    p.truncate([1], [0])
    p.seqs.state.copy_(kept)
    p.ref = oracle
    assert p.append([1, 3, 0], [1, 50, 13]) == [1, 1, 1]
    assert views[0].tolist() == p.ref.lens and views[1].tolist() == p.ref.tables


def test_a_graph_replayed_after_its_object_is_dropped(dev):
    """The plan's workspace stays the graph's: what is allocated afterwards keeps its contents, and
    the replays go on with the state and pool that the caller holds."""
    p = Pair(dev, rows=5)
    rows = ints([0, 2, 3], dev)
    p.append([0, 1, 2, 3], [14, 33, 1, 15])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots, status = p.seqs.append(rows)
    state, size = p.seqs.state, p.seqs._workspace.numel()
    p.seqs = None
    gc.collect()
    torch.cuda.synchronize()
    others = [torch.full((size,), 7, dtype=torch.uint8, device=dev) for _ in range(8)]
    for _ in range(6):
        graph.replay()
        torch.cuda.synchronize()
        want_slots, want = p.ref.append([0, 2, 3])
        assert slots.cpu().tolist() == want_slots and status.cpu().tolist() == want
        assert torch.equal(state.cpu(), p.ref.state())
        assert all(bool((x == 7).all()) for x in others)
    del graph
    assert nkv.release_retired_decode_workspaces() >= 1


def test_a_listed_page_that_was_free_keeps_its_new_row(dev):
    free_page_listed(Pair(dev))


def test_listed_pages_among_many_copies(dev):
    """Every page of the pool listed beside 40 copies: those in use before lose a reference, the new
    ones keep theirs."""
    p = Pair(dev, pages=200, rows=90, width=4)
    p.append(list(range(40)), [33 + r % 20 for r in range(40)])
    p.fork(list(range(40)), list(range(40, 80)))
    p.truncate(list(range(40, 80)), [17 + r % 15 for r in range(40)], pages=list(range(200)))
    assert [p.ref.refs[p.ref.tables[r][1]] for r in range(40, 80)] == [1] * 40
