"""Block-scaled caches as they are used: a pool, layers over it, and sequences that share its pages.
Outputs are held to the definition over what the cache holds (the tolerance:
test_gpu_scaled_attention.py), and the caches' contents to the oracle's."""
import importlib
import types

import pytest
import torch

from oracle.pages_ref import PagedSequencesRef
from oracle.scaled_ref import PAD, scaled_rows_ref, scaled_store_ref
from scaled_util import BF, I32, U8, values
from test_gpu_scaled_attention import close, reference
from test_gpu_scaled_store import same_cache

pytestmark = pytest.mark.gpu

nkv = importlib.import_module("nanokv-llm_amd")
Hq, Hk, D, B = 8, 2, 64, 32


def layer(scale=0.2):
    cfg = types.SimpleNamespace(kv_compress_enabled=False)
    return nkv.Attention(Hq, D, scale, Hk, cfg, 2)


class Model:
    """Two layers over a pool, and the oracle's sequences and caches beside them."""

    def __init__(self, dev, blocks=40, rows=6, width=8):
        self.pool = nkv.ScaledKVCachePool(2, Hk, D, B, num_blocks=blocks, device=dev)
        self.layers = [layer(), layer()]
        assert self.pool.bind(self.layers) == 2
        self.seqs = nkv.PagedSequences(self.pool, rows, width)
        # the oracle's copies whole pages: what lies behind a sequence's end is nobody's
        self.ref = PagedSequencesRef(torch.zeros(2, 2, blocks, B, 1, Hk * D + PAD, dtype=U8), rows,
                                     width)
        copy = self.ref._copy
        self.ref._copy = lambda src, dst, n: copy(src, dst, -(-n // 32) * 32)
        self.dev, self.g = dev, torch.Generator().manual_seed(1)

    def i32(self, x):
        return torch.tensor(x, dtype=I32, device=self.dev)

    def cache(self, layer, is_v):
        return self.ref.kv[int(is_v), layer].view(-1, B, Hk * D + PAD)

    def step(self, rows, counts, tables=True):
        """New tokens for rows: counts None: one each, decoded; else a prefill."""
        decode = counts is None
        n = [1] * len(rows) if decode else counts
        cu = [sum(n[:i]) for i in range(len(n) + 1)]
        if decode:
            slots, ok = self.seqs.append(self.i32(rows))
            want, _ = self.ref.append(rows)
        else:
            slots, ok = self.seqs.append(self.i32(rows), self.i32(cu), cu[-1])
            want, _ = self.ref.append(rows, cu=cu, n_tokens=cu[-1])
        assert slots.tolist() == want and bool(ok.all())
        lens = self.seqs.context_lens[self.i32(rows).long()]
        bt = self.seqs.block_tables[self.i32(rows).long()]
        total = [self.ref.lens[r] for r in rows]
        cu_k = [sum(total[:i]) for i in range(len(n) + 1)]
        nkv.set_context(decode, self.i32(cu), self.i32(cu_k), max(n), max(total), slots, lens,
                        bt if tables else None)
        try:
            for at, l in enumerate(self.layers):
                q = values(cu[-1], Hq, D, self.g, outliers=False)
                fused = values(cu[-1], 2 * Hk, D, self.g)
                k, v = fused[:, :Hk], fused[:, Hk:]
                o = l(q.to(self.dev), fused.to(self.dev)[:, :Hk], fused.to(self.dev)[:, Hk:], at)
                scaled_store_ref(k, v, self.cache(at, False), self.cache(at, True),
                                 torch.tensor(want))
                o = o.squeeze(1) if decode else o
                for i, r in enumerate(rows):
                    part = slice(cu[i], cu[i + 1])
                    kv = [scaled_rows_ref(self.cache(at, x), x, self.ref.tables[r], total[i], Hk, D)
                          for x in (False, True)] if tables else [k[part].double(), v[part].double()]
                    close(o[part], *reference(q[part], *kv, 0.2), what=(at, r))
        finally:
            nkv.reset_context()

    def check(self):
        """What every row holds, and the bookkeeping."""
        assert torch.equal(self.seqs.state.cpu(), self.ref.state())
        for at in range(2):
            for r, n in enumerate(self.ref.lens):
                if n == 0:
                    continue
                table = self.seqs.block_tables[r:r + 1]
                got = nkv.scaled_read_kvcache(self.layers[at].k_cache, self.layers[at].v_cache, table,
                                              self.i32([0, n]), n, Hk)
                for x, is_v in zip(got, (False, True)):
                    want = scaled_rows_ref(self.cache(at, is_v), is_v, self.ref.tables[r], n, Hk, D)
                    assert torch.equal(x.cpu().double(), want), (at, r, is_v)


def test_prompts_forks_steps_and_rollbacks(dev):
    m = Model(dev)
    m.step([0, 1], [45, 70], tables=False)      # first prompts attend their own rows
    m.check()
    m.step([0, 2], [30, 33])                    # a chunk behind a prefix, a prompt over the cache
    m.step([0, 1, 2], None)
    m.check()
    kids = m.seqs.fork(m.i32([0, 1, 0]), m.i32([3, 4, 5]))
    assert kids.tolist() == m.ref.fork([0, 1, 0], [3, 4, 5])
    for _ in range(3):
        m.step([5, 0, 3, 4, 1], None)           # beams go their own ways in the same page's copies
    m.check()
    m.step([2, 3, 0], [1, 6, 1])                # drafts beside steps
    ok = m.seqs.truncate(m.i32([3, 1, 4, 0]), m.i32([77, 66, 0, 40]))
    assert ok.tolist() == m.ref.truncate([3, 1, 4, 0], [77, 66, 0, 40])
    m.check()
    for _ in range(2):
        m.step([0, 1, 3, 5], None)
    fork = m.seqs.fork(m.i32([5]), m.i32([4]), share_pages=False)
    assert fork.tolist() == m.ref.fork([5], [4], False)
    info, moves = m.seqs.compact(40)
    ref_info, ref_moves = m.ref.compact(40)
    assert info.tolist() == ref_info and moves.tolist() == ref_moves
    m.step([4, 5, 0], None)
    m.check()


def test_a_decode_loop_in_a_graph(dev):
    """Append, store and attention captured once and replayed, against eager calls on a copy."""
    pool, twin = (nkv.ScaledKVCachePool(1, Hk, D, B, num_blocks=20, device=dev) for _ in range(2))
    a, b = layer(), layer()
    pool.bind([a])
    twin.bind([b])
    rows = torch.arange(3, dtype=I32, device=dev)
    cu = torch.tensor([0, 20, 50, 51], dtype=I32, device=dev)
    g = torch.Generator().manual_seed(2)
    seqs = [nkv.PagedSequences(p, 3, 6) for p in (pool, twin)]
    x = values(51, Hk, D, g).to(dev)
    for p, s in zip((a, b), seqs):
        slots, _ = s.append(rows, cu, 51)
        nkv.scaled_store_kvcache(x, x, p.k_cache, p.v_cache, slots)
    q, k = values(3, Hq, D, g).to(dev), values(3, Hk, D, g).to(dev)

    def step(s, l):
        slots, _ = s.append(rows)
        nkv.set_context(True, slot_mapping=slots, context_lens=s.context_lens,
                        block_tables=s.block_tables)
        out = l(q, k, k, 0)
        nkv.reset_context()
        return out

    nkv.reserve_decode_workspace(dev, 3, Hq, 6, B, D)
    step(seqs[1], b)
    kept = seqs[0].state.clone(), pool.kv_cache.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seqs[0], a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(seqs[0], a)
    for _ in range(20):
        q.copy_(values(3, Hq, D, g))
        k.copy_(values(3, Hk, D, g))
        graph.replay()
        want = step(seqs[1], b)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(seqs[0].state, seqs[1].state)
    assert bool(kept[0].ne(seqs[0].state).any())
    same_cache(pool.kv_cache[0, 0], twin.kv_cache[0, 0].cpu(), Hk, D)
    del graph, seqs
    nkv.release_retired_decode_workspaces()


def test_a_pool_sized_by_the_memory(dev):
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()  # a pool leaves room for the peak so far
    pool = nkv.ScaledKVCachePool(4, 8, 128, 256, gpu_memory_utilization=0.05, device=dev)
    assert pool.num_blocks * pool.block_bytes == pool.kv_cache.numel()
    assert 0 < pool.kv_cache.numel() < 0.05 * torch.cuda.get_device_properties(0).total_memory
