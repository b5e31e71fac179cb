"""Varlen differential attention (prompts, chunks, decode rows among them) against the definition in
64 bits, and the layer that calls it.

Tolerances are test_gpu_diff_decode.py's: the kernel rounds each weight once to 16 bits (off by at
most u of itself) and sums the rounded ones, so A_m = sum w v / sum w is off by at most 2 u max|v|: twice
that bound's d.
"""
import importlib

import pytest
import torch

from oracle.diff_attention_ref import diff_attention_ref, gather_rows
from oracle.fp8_ref import fp8_quantize_ref
from test_gpu_diff_decode import BF, F16, FP8, I32, KS, VS, tolerance

pytestmark = pytest.mark.gpu

nkv = importlib.import_module("nanokv-llm_amd")
da = importlib.import_module("nanokv-llm_amd.layers.diff_attention")


def make(dev, new, ctx, hq, hk, d, B=16, dtype=BF, kv=None, seed=0, spread=1.0):
    """Sequences of ctx[i] keys with new[i] queries at their end, in pages and as rows."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // B) for n in ctx]
    NB = sum(counts) + 2
    ids = torch.randperm(NB, generator=g)
    bt, at = torch.full((len(ctx), max(counts) + 1), -1, dtype=I32), 0
    for i, c in enumerate(counts):
        bt[i, :c] = ids[at:at + c]
        at += c
    k = torch.randn(NB, B, hk, d, generator=g)
    v = torch.randn(NB, B, hk, d, generator=g) + 0.3
    if kv is FP8:
        k, v = (k / KS).to(FP8), (v / VS).to(FP8)
    else:
        k, v = k.to(dtype), v.to(dtype)
    q = (torch.randn(sum(new), hq, d, generator=g) * spread).to(dtype)
    lambdas = torch.randn(4, d, generator=g) * 0.1
    weight = (1 + 0.2 * torch.randn(2 * d, generator=g)).to(dtype)
    cu = [torch.tensor([0] + list(x), dtype=torch.int64).cumsum(0).to(I32) for x in (new, ctx)]
    return dict(q=q, k=k, v=v, bt=bt, new=new, ctx=ctx, cu_q=cu[0], cu_k=cu[1], lambdas=lambdas,
                weight=weight, init=0.43, scale=d ** -0.5, B=B, fp8=kv is FP8, dev=dev)


def run(c, split=True, **kw):
    dev = c["dev"]
    ks, vs = (KS, VS) if c["fp8"] else (1.0, 1.0)
    kw.setdefault("norm_weight", c["weight"].to(dev))
    return nkv.diff_varlen_prefill(
        c["q"].to(dev), c["k"].to(dev), c["v"].to(dev), c["cu_q"].to(dev), c["cu_k"].to(dev),
        max(c["new"], default=0), c["scale"], c["lambdas"].to(dev), c["init"],
        block_tables=c["bt"].to(dev), max_seqlen_k=max(c["ctx"]) if split else None, k_scale=ks,
        v_scale=vs, **kw)


def reference(c, weight="own", eps=1e-5, zeros=True):
    ks, vs = (KS, VS) if c["fp8"] else (1.0, 1.0)
    weight = c["weight"] if isinstance(weight, str) else weight
    outs, tols, at = [], [], 0
    for i, (lq, lk) in enumerate(zip(c["new"], c["ctx"])):
        k = gather_rows(c["k"], c["bt"][i], lk, c["B"], zeros, ks)
        v = gather_rows(c["v"], c["bt"][i], lk, c["B"], zeros, vs)
        o = diff_attention_ref(c["q"][at:at + lq], k, v, c["scale"], c["lambdas"], c["init"],
                               weight, eps)
        at += lq
        vmax = float(v.abs().max()) if len(v) else 0.0
        outs.append(o)
        tols.append(tolerance(o, 2 * vmax, c["lambdas"], c["init"], weight, eps, c["q"].dtype))
    return torch.cat(outs), torch.cat(tols)


def check(out, c, **kw):
    ref, tol = reference(c, **kw)
    err = (out.double().cpu() - ref).abs()
    assert out.shape == ref.shape and bool((err <= tol).all()), \
        f"off by up to {float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("dtype,kv", [(BF, None), (F16, None), (BF, FP8)])
@pytest.mark.parametrize("hq,hk,d", [(2, 2, 64), (4, 2, 128), (16, 8, 64), (32, 8, 128), (6, 6, 64),
                                     (40, 8, 128), (20, 2, 64), (12, 2, 128), (128, 2, 64)])
def test_types_heads_and_lengths(dev, dtype, kv, hq, hk, d):
    """One token to several tiles; prompts from nothing and after a prefix; decode rows among them."""
    c = make(dev, [1, 65, 16, 1, 130, 2], [1, 65, 80, 300, 131, 64], hq, hk, d, dtype=dtype, kv=kv,
             seed=hq + d)
    check(run(c), c)


@pytest.mark.parametrize("d,hq", [(64, 2), (64, 6), (128, 2), (128, 10)])
def test_query_counts_around_a_tile(dev, d, hq):
    qt = {64: 96, 128: 128}[d] // (hq // 2)
    new = [qt - 1, qt, qt + 1, 2 * qt, 1]
    c = make(dev, new, [n + 7 for n in new], hq, 2, d, seed=hq)
    check(run(c), c)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B", [16, 48, 80, 256])
def test_pages_that_end_inside_a_step(dev, d, B):
    c = make(dev, [100, 3], [517, 1300], 4, 2, d, B=B, seed=B)
    check(run(c), c)


@pytest.mark.parametrize("kv", [None, FP8])
@pytest.mark.parametrize("d", [64, 128])
def test_split_keys_against_whole_ones(dev, d, kv):
    """Few tiles over long contexts: the keys are split, and every range count gives the row."""
    c = make(dev, [40, 1, 7], [4500, 2100, 520], 8, 4, d, seed=d, kv=kv)
    q, k = c["q"].to(dev), c["k"].to(dev)
    assert da.diff_prefill_workspace(q, k, 3, 40, 4500) is not None
    check(run(c), c)
    check(run(c, split=False), c)


def test_more_sequences_than_lanes(dev):
    n = [(5 * i) % 4 for i in range(150)]  # some bring no token
    c = make(dev, n, [x + (3 * i) % 40 for i, x in enumerate(n)], 4, 2, 64, seed=3)
    check(run(c), c)


@pytest.mark.parametrize("d", [64, 128])
def test_many_short_prompts_over_long_contexts(dev, d):
    """More prompts than lanes, their tiles cut into ranges."""
    new = [2 + i % 4 for i in range(75)]
    c = make(dev, new, [n + (97 * i) % 1400 for i, n in enumerate(new)], 2, 2, d, seed=25)
    check(run(c), c)


def test_rows_that_see_no_key_are_zero(dev):
    """More queries than keys: the first ones see nothing; a sequence without keys."""
    c = make(dev, [20, 5, 3], [8, 0, 50], 4, 2, 64, seed=4)
    out = run(c)
    assert bool((out[:12] == 0).all()) and bool((out[20:25] == 0).all())
    check(out, c)


def test_sharp_maps(dev):
    c = make(dev, [150], [300], 8, 4, 64, seed=6, spread=12.0)
    check(run(c), c)


def test_scores_that_rise_late(dev):
    """Keys that grow along the context: the running maximum is raised step after step."""
    c = make(dev, [70, 40], [700, 1100], 4, 2, 64, seed=16, spread=3.0)
    for i, n in enumerate(c["ctx"]):
        for t in range(0, n, 16):
            b = int(c["bt"][i, t // 16])
            c["k"][b] = c["k"][b] * (0.1 + t / 200)
    check(run(c), c)


def test_without_a_norm_weight_and_other_eps(dev):
    c = make(dev, [50, 7], [50, 90], 4, 2, 128, seed=7)
    check(run(c, norm_weight=None, eps=0.5), c, weight=None, eps=0.5)


def test_infinity_in_one_map_stays_in_it(dev):
    c = make(dev, [9], [33], 4, 2, 64, seed=10)
    c["q"][:, 1::2] = c["q"][:, 1::2].abs()
    c["k"][c["bt"][0, 0], 5, 1] = -float("inf")
    check(run(c), c)


def test_rows_behind_a_context_are_not_read(dev):
    c = make(dev, [5, 18], [21, 70], 4, 2, 64, seed=11)
    clean = c["k"].clone(), c["v"].clone()
    c["k"][:], c["v"][:] = float("nan"), float("nan")
    for i, n in enumerate(c["ctx"]):
        for t in range(n):
            b = int(c["bt"][i, t // 16])
            c["k"][b, t % 16], c["v"][b, t % 16] = clean[0][b, t % 16], clean[1][b, t % 16]
    check(run(c), c)


def test_invalid_blocks_read_as_zeros(dev):
    c = make(dev, [30, 40], [60, 70], 4, 2, 64, seed=12)
    c["bt"][0, 1], c["bt"][1, 2] = -1, 10 ** 6
    check(run(c), c)
    c["bt"] = c["bt"][:, :3].contiguous()  # keys past the table
    check(run(c), c)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("d", [64, 128])
def test_contiguous_rows_of_a_projection(dev, d, dtype):
    hq, hk = 8, 4
    c = make(dev, [33, 1, 140], [33, 1, 140], hq, hk, d, dtype=dtype, seed=13)
    rows = torch.cat([torch.cat([gather_rows(c[x], c["bt"][i], n, 16) for x in ("k", "v")], dim=1)
                      for i, n in enumerate(c["ctx"])])
    fused = torch.zeros(174, (hq + 2 * hk) * d, dtype=dtype)
    fused[:, :hq * d] = c["q"].flatten(1)
    fused[:, hq * d:] = rows.flatten(1).to(dtype)
    f = fused.to(dev)
    q = f[:, :hq * d].unflatten(1, (hq, d))
    k = f[:, hq * d:(hq + hk) * d].contiguous().unflatten(1, (hk, d))  # roped: its own tensor
    v = f[:, (hq + hk) * d:].unflatten(1, (hk, d))
    out = nkv.diff_varlen_prefill(q, k, v, c["cu_q"].to(dev), c["cu_k"].to(dev), 140, c["scale"],
                                  c["lambdas"].to(dev), c["init"], c["weight"].to(dev),
                                  max_seqlen_k=140)
    check(out, c)


def test_rows_of_out_behind_the_last_sequence_stay(dev):
    c = make(dev, [30, 11], [90, 20], 4, 2, 64, seed=14)
    q = torch.cat([c["q"], c["q"][:9]]).to(dev)  # a padded batch
    out = torch.full((50, 2, 128), 7.0, dtype=BF, device=dev)
    got = nkv.diff_varlen_prefill(q, c["k"].to(dev), c["v"].to(dev), c["cu_q"].to(dev),
                                  c["cu_k"].to(dev), 30, c["scale"], c["lambdas"].to(dev), c["init"],
                                  c["weight"].to(dev), block_tables=c["bt"].to(dev), out=out,
                                  max_seqlen_k=90)
    check(got[:41], c)
    assert bool((out[41:] == 7).all())


def test_cu_seqlens_past_the_rows_of_q_write_nothing(dev):
    c = make(dev, [30, 11], [90, 20], 4, 2, 64, seed=15)
    q = c["q"][:35].to(dev)  # the second sequence does not fit
    out = torch.full((35, 2, 128), 7.0, dtype=BF, device=dev)
    nkv.diff_varlen_prefill(q, c["k"].to(dev), c["v"].to(dev), c["cu_q"].to(dev),
                            c["cu_k"].to(dev), 30, c["scale"], c["lambdas"].to(dev), c["init"],
                            c["weight"].to(dev), block_tables=c["bt"].to(dev), out=out)
    ref, tol = reference(c)
    assert bool(((out[:30].double().cpu() - ref[:30]).abs() <= tol[:30]).all())
    assert bool((out[30:] == 7).all())


def test_equal_results_call_after_call_and_on_a_stream(dev):
    c = make(dev, [200, 1, 33], [1200, 900, 33], 8, 4, 128, seed=17)
    first = run(c)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        again = run(c)
    s.synchronize()
    assert torch.equal(first, again) and torch.equal(first, run(c))


def test_empty_batches(dev):
    c = make(dev, [1], [1], 4, 2, 64)
    for cu, rows in (([0], 0), ([0, 0], 0), ([0, 0], 3)):
        cu = torch.tensor(cu, dtype=I32, device=dev)
        out = torch.full((rows, 2, 128), 7.0, dtype=BF, device=dev)
        nkv.diff_varlen_prefill(c["q"].to(dev).repeat(rows, 1, 1), c["k"].to(dev), c["v"].to(dev),
                                cu, cu, 0, 0.1, c["lambdas"].to(dev), 0.2,
                                block_tables=c["bt"].to(dev), out=out)
        assert bool((out == 7).all())


@pytest.mark.parametrize("kv", [BF, F16, FP8])
def test_the_layer_over_shared_pages(dev, kv):
    """The operators together, as a sampling program uses them: a prompt, two samples forked from it,
    steps of all three, one rolled back and one ended, the pool closed up, more steps; every
    output against 64 bits over the rows that were stored."""
    hq, hk, d, B, S = 8, 4, 64, 16, 4
    dtype = F16 if kv is F16 else BF
    ks, vs = (KS, VS) if kv is FP8 else (1.0, 1.0)
    g = torch.Generator().manual_seed(18)
    pool = nkv.layers.kv_cache.KVCachePool(2, hk, d, B, kv, num_blocks=24, device=dev, k_scale=ks,
                                           v_scale=vs)
    pool.kv_cache.view(torch.uint8).zero_()
    seqs = nkv.PagedSequences(pool, S, 6)
    layers = [nkv.DifferentialAttention(hq, d, d ** -0.5, hk, nkv.lambda_init_of(i)).to(dev)
              for i in range(2)]
    for m in layers:
        m.lambdas.copy_(torch.randn(4, d, generator=g) * 0.1)
        m.norm_weight.data = (1 + 0.2 * torch.randn(2 * d, generator=g)).to(dtype).to(dev)
    assert pool.bind(layers) == 2
    stored = [[[] for _ in range(S)] for _ in layers]  # (k, v) rows as the cache holds them

    def ints(x):
        return torch.tensor(x, dtype=I32, device=dev)

    def held(x, scale):
        return fp8_quantize_ref(x, scale).view(FP8).double() * scale if kv is FP8 else x.double()

    def step(rows, counts, decode):
        n = sum(counts)
        cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
        slots, status = seqs.append(ints(rows), *(() if decode else (ints(cu), n)))
        assert status.tolist() == [1] * len(rows)
        at = ints(rows).long()
        lens, bt = seqs.context_lens[at], seqs.block_tables[at]
        cu_k = torch.cat([lens.new_zeros(1), lens.cumsum(0).to(I32)])
        nkv.set_context(decode, ints(cu), cu_k, max(counts), int(lens.max()), slots, lens, bt)
        for i, m in enumerate(layers):
            q = torch.randn(n, hq, d, generator=g).to(dtype)
            k, v = (torch.randn(n, hk, d, generator=g).to(dtype) for _ in range(2))
            out = m(q.to(dev), k.to(dev), v.to(dev), i).reshape(n, hq // 2, 2 * d).double().cpu()
            for r, c, a in zip(rows, counts, cu):
                stored[i][r] += [(held(k[t], ks), held(v[t], vs)) for t in range(a, a + c)]
                kk = torch.stack([x[0] for x in stored[i][r]])
                vv = torch.stack([x[1] for x in stored[i][r]])
                w, l = m.norm_weight.cpu(), m.lambdas.cpu()
                ref = diff_attention_ref(q[a:a + c], kk, vv, d ** -0.5, l, m.lambda_init, w)
                tol = tolerance(ref, 2 * float(vv.abs().max()), l, m.lambda_init, w, 1e-5, dtype)
                assert bool(((out[a:a + c] - ref).abs() <= tol).all())
        nkv.reset_context()

    step([0], [37], False)
    assert seqs.fork(ints([0, 0]), ints([1, 2])).tolist() == [1, 1]
    for i in range(2):
        stored[i][1], stored[i][2] = list(stored[i][0]), list(stored[i][0])
    for _ in range(14):
        step([0, 1, 2], [1, 1, 1], True)
    assert seqs.truncate(ints([1, 0]), ints([20, 0])).tolist() == [1, 1]
    for i in range(2):
        stored[i][1], stored[i][0] = stored[i][1][:20], []
    info, _ = seqs.compact()
    assert info.tolist()[0] == int((seqs.ref_counts > 0).sum())
    assert int(seqs.block_tables.max()) < info.tolist()[0]
    step([2, 3, 1], [1, 25, 9], False)  # a mixed step
    for _ in range(3):
        step([1, 3, 2], [1, 1, 1], True)


@pytest.mark.parametrize("d,hq,hk", [(64, 32, 4), (128, 32, 4), (128, 128, 2)])
@pytest.mark.parametrize("prefix", [0, 700])
def test_large_tiles(dev, d, hq, hk, prefix):
    """More small tiles than CUs, so that the waves take as many row groups as they can: whole tiles,
    and (over a prefix) tiles cut into ranges."""
    n = {64: 600, 128: 1100}[d] if hq < 128 else 300
    c = make(dev, [n, 33], [n + prefix, 33], hq, hk, d, seed=d + prefix)
    check(run(c), c)


@pytest.mark.parametrize("d", [64, 128])
def test_length_bounds_that_are_not(dev, d):
    """max_seqlen_q and max_seqlen_k only choose the launch: a plan for a few long prompts meets many
    short ones, one for decode rows meets prompts, and bounds below the lengths."""
    c = make(dev, [30] * 20, [90] * 20, 8, 4, d, seed=21)
    want = reference(c)
    dev_args = [c[x].to(dev) for x in ("q", "k", "v", "cu_q", "cu_k")]
    for max_q, max_k in ((600, 9000), (581, 700), (2, 10 ** 6), (1, 5000), (30, 1), (0, 0)):
        out = nkv.diff_varlen_prefill(*dev_args, max_q, c["scale"], c["lambdas"].to(dev), c["init"],
                                      c["weight"].to(dev), block_tables=c["bt"].to(dev),
                                      max_seqlen_k=max_k)
        assert bool(((out.double().cpu() - want[0]).abs() <= want[1]).all()), (max_q, max_k)


@pytest.mark.parametrize("kv", [None, FP8])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_rows_among_prompts_in_any_place(dev, d, kv):
    """Rows of one token (streamed apart) before, between and behind prompts, some without keys,
    invalid blocks and keys past the table among their contexts."""
    new = [1, 40, 1, 1, 0, 1, 70, 1]
    ctx = [500, 700, 1, 0, 30, 90, 70, 2000]
    c = make(dev, new, ctx, 20, 4, d, seed=22 + d, kv=kv)
    c["bt"][0, 3], c["bt"][5, 0] = -1, 10 ** 7
    check(run(c), c)
    check(run(c, split=False), c)
    c["bt"] = c["bt"][:, :100].contiguous()  # the last row's keys end past the table
    check(run(c), c)


def test_captured_prefill_and_decode(dev):
    """Both operators in one graph, replayed over new inputs with eager calls between the replays."""
    a = make(dev, [40, 1, 90], [900, 1500, 90], 8, 4, 64, seed=23)
    b = make(dev, [40, 1, 90], [900, 1500, 90], 8, 4, 64, seed=24)
    put = {x: a[x].to(dev) for x in ("q", "k", "v", "bt", "cu_q", "cu_k", "lambdas", "weight")}
    lens = a["cu_k"].diff().to(dev)

    def both():
        p = nkv.diff_varlen_prefill(put["q"], put["k"], put["v"], put["cu_q"], put["cu_k"], 90,
                                    a["scale"], put["lambdas"], a["init"], put["weight"],
                                    block_tables=put["bt"], max_seqlen_k=1500)
        d = nkv.diff_paged_decode(put["q"][:3], put["k"], put["v"], lens, put["bt"], a["scale"],
                                  put["lambdas"], a["init"], put["weight"])
        return p, d

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p, d = both()
    for c in (a, b, a, b):
        for x in put:
            put[x].copy_(c[x])
        graph.replay()
        torch.cuda.synchronize()
        check(p, c)
        eager = both()
        assert torch.equal(eager[0], p) and torch.equal(eager[1], d)


@pytest.mark.parametrize("kv", [None, FP8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_rows_that_see_no_key_beside_values_that_are_not_finite(dev, bad, d, kv):
    """More queries than keys, and a value that is not finite in a key that only the last one sees:
    those that see none are zero all the same, in tiles of others that see some too."""
    if kv is FP8 and bad == float("inf"):
        bad = float("nan")  # e4m3fn has no infinity
    c = make(dev, [40, 20], [13, 600], 4, 2, d, seed=30, kv=kv)
    c["v"][c["bt"][0, 0], 12] = bad
    for split in (False, True):
        out = run(c, split=split)
        assert bool((out[:27] == 0).all())
        assert not bool(torch.isfinite(out[39].float()).any())
        ref, tol = reference(c)
        assert bool(((out[40:].double().cpu() - ref[40:]).abs() <= tol[40:]).all())


def test_a_cache_past_4_gib(dev):
    """Pages whose byte offset passes 32 bits: whole tiles, cut ones and a decode row."""
    B, hk, d = 256, 8, 128
    NB = (5 << 30) // (B * hk * d * 2)
    g = torch.Generator().manual_seed(32)
    k = torch.empty(NB, B, hk, d, dtype=BF, device=dev)
    v = torch.empty(NB, B, hk, d, dtype=BF, device=dev)
    bt = torch.tensor([[NB - 1, 0, NB - 2], [NB - 3, 1, -1]], dtype=I32)
    at = [NB - 1, 0, NB - 2, NB - 3, 1]
    rows = torch.randn(2, 5, B, hk, d, generator=g).to(BF)
    k[at], v[at] = rows[0].to(dev), rows[1].to(dev)
    q = torch.randn(91, 16, d, generator=g).to(BF)
    lambdas = torch.randn(4, d, generator=g) * 0.1
    cu_q, cu_k = torch.tensor([0, 90, 91], dtype=I32), torch.tensor([0, 700, 1000], dtype=I32)
    for max_k in (700, None):
        out = nkv.diff_varlen_prefill(q.to(dev), k, v, cu_q.to(dev), cu_k.to(dev), 90, d ** -0.5,
                                      lambdas.to(dev), 0.2, block_tables=bt.to(dev),
                                      max_seqlen_k=max_k)
        for a, b, first, n in ((0, 90, 0, 700), (90, 91, 3, 300)):
            kk, vv = (x[first:].flatten(0, 1)[:n] for x in rows)
            ref = diff_attention_ref(q[a:b], kk, vv, d ** -0.5, lambdas, 0.2)
            tol = tolerance(ref, 2 * float(vv.abs().max()), lambdas, 0.2, None, 1e-5, BF)
            assert bool(((out[a:b].double().cpu() - ref).abs() <= tol).all())


@pytest.mark.parametrize("kv", [None, FP8])
def test_the_layer_captured_over_a_reserved_workspace(dev, kv):
    """Workspace reserved for heads of 2 head_dim, a decode step of the layer in one graph, replayed
    over new inputs with eager steps and a regrowth of the shared workspace between the replays."""
    hq, hk, d, B = 8, 4, 64, 16
    g = torch.Generator().manual_seed(33)
    c = make(dev, [1] * 5, [60, 1, 33, 700, 16], hq, hk, d, B=B, kv=kv, seed=33)
    m = nkv.DifferentialAttention(hq, d, c["scale"], hk, c["init"]).to(dev)
    m.lambdas.copy_(c["lambdas"])
    m.norm_weight.data = c["weight"].to(dev)
    m.k_cache, m.v_cache = c["k"].to(dev), c["v"].to(dev)
    if kv is FP8:
        m.k_scale, m.v_scale = KS, VS
    bt, lens = c["bt"].to(dev), torch.tensor(c["ctx"], dtype=I32, device=dev)
    slots = torch.tensor([int(c["bt"][i, (n - 1) // B]) * B + (n - 1) % B
                          for i, n in enumerate(c["ctx"])], dtype=I32, device=dev)
    q = torch.empty(5, hq, d, dtype=BF, device=dev)
    k, v = (torch.empty(5, hk, d, dtype=BF, device=dev) for _ in range(2))
    nkv.reserve_decode_workspace(dev, 5, hq, bt.size(1), B, head_dim=2 * d)

    def fill():
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g).to(BF))

    def expect(out):
        now = dict(c, q=q.cpu(), k=m.k_cache.cpu(), v=m.v_cache.cpu())
        check(out.squeeze(1), now, zeros=False)

    nkv.set_context(True, slot_mapping=slots, context_lens=lens, block_tables=bt)
    try:
        graph = torch.cuda.CUDAGraph()
        fill()
        m(q, k, v)  # warm-up
        with torch.cuda.graph(graph):
            out = m(q, k, v)
        for i in range(5):
            fill()
            graph.replay()
            torch.cuda.synchronize()
            expect(out)
            held = m.k_cache.view(torch.uint8).clone()
            assert torch.equal(m(q, k, v), out)  # the same step again, eagerly
            assert torch.equal(m.k_cache.view(torch.uint8), held)
            if i == 2:
                shared = importlib.import_module("nanokv-llm_amd.layers.attention")
                ws = shared.shared_decode_workspace(q.device, 0)
                nkv.reserve_decode_workspace(dev, 64, 64, 4096, B, head_dim=2 * d)
                assert shared.shared_decode_workspace(q.device, 0).numel() >= ws.numel()
    finally:
        nkv.reset_context()
