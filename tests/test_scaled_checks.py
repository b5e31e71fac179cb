"""Block-scaled caches: the oracle's own rules, and the refusals that need no GPU."""
import importlib
import random
import struct
import types

import pytest
import torch

from oracle.scaled_ref import (E_MAX, E_MIN, PAD, TILE, attention_rows_ref, codes_of, exponent,
                               places, scaled_rows_ref, scaled_store_ref)
from scaled_util import cache_of

nkv = importlib.import_module("nanokv-llm_amd")
sc = importlib.import_module("nanokv-llm_amd.layers.scaled_cache")
pages = importlib.import_module("nanokv-llm_amd.engine.pages")
L = importlib.import_module("nanokv-llm_amd._lib")
BF, I32, U8 = torch.bfloat16, torch.int32, torch.uint8
P = 0x10000


# ---------------------------------------------------------------- the oracle
@pytest.mark.parametrize("D", [64, 128])
def test_places_are_every_byte_once(D):
    for p in places(D):
        assert p.flatten().sort().values.tolist() == list(range(TILE * D))


def test_exponents():
    assert exponent(0.0) == E_MIN and exponent(448.0) == 0 and exponent(448.0001) == 1
    assert exponent(224.0) == -1 and exponent(1.0) == -8 and exponent(0.875) == -9
    assert exponent(float(torch.finfo(BF).max)) == E_MAX
    for a in (1e-38, 0.3, 5.0, 7e20):
        e = exponent(a)
        assert (a <= 448 * 2.0 ** e or e == E_MAX) and (e == E_MIN or a > 448 * 2.0 ** (e - 1))


def test_a_store_reads_back_within_half_a_step():
    """E4M3 rounds by at most 2^-4 of the value, or half a subnormal step of the tile's scale."""
    g = torch.Generator().manual_seed(0)
    key, value = torch.randn(40, 2, 64, generator=g).to(BF), torch.randn(40, 2, 64, generator=g).to(BF)
    kc, vc = (torch.zeros(2, 64, 2 * 64 + PAD, dtype=U8) for _ in range(2))
    scaled_store_ref(key, value, kc, vc, torch.arange(40, dtype=I32))
    for x, c, is_v in ((key, kc, False), (value, vc, True)):
        got = scaled_rows_ref(c, is_v, [0], 40, 2, 64)
        x = x.double()
        for lo, hi in ((0, 32), (32, 40)):
            step = x[lo:hi].abs().amax((0, 2)) / 448 * 2 * 2.0 ** -10  # scale < 2 * max / 448
            bound = torch.maximum(x[lo:hi].abs() * 2.0 ** -4, step[None, :, None])
            assert bool(((got[lo:hi] - x[lo:hi]).abs() <= bound).all())


def test_a_scale_that_grows_keeps_the_rows_before():
    key = torch.zeros(3, 1, 64, dtype=BF)
    key[0], key[1], key[2] = 1.0, 2.0 ** 12, 0.5
    c = torch.zeros(1, 32, 64 + PAD, dtype=U8)
    for i in range(2):
        scaled_store_ref(key[i:i + 1], key[i:i + 1], c, c.clone(), torch.tensor([i], dtype=I32))
    assert scaled_rows_ref(c, False, [0], 2, 1, 64)[:, 0, 0].tolist() == [1.0, 4096.0]
    # the tile's first row written again: it begins anew, with a smaller scale
    scaled_store_ref(key[2:], key[2:], c, c.clone(), torch.tensor([0], dtype=I32))
    assert int(c.view(-1)[32 * 64]) == exponent(0.5) + 127
    assert scaled_rows_ref(c, False, [0], 1, 1, 64)[0, 0, 0] == 0.5


def test_cache_of_is_what_a_store_writes():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 32, 2, 64, generator=g).to(BF)
    kc, vc = (torch.zeros(2, 32, 2 * 64 + PAD, dtype=U8) for _ in range(2))
    scaled_store_ref(x.flatten(0, 1), x.flatten(0, 1), kc, vc, torch.arange(64, dtype=I32))
    assert torch.equal(kc, cache_of(x, False)) and torch.equal(vc, cache_of(x, True))


def test_special_values():
    x = torch.tensor([[float("nan"), float("inf"), -float("inf"), 3.0]], dtype=torch.float64)
    assert codes_of(x, 0).tolist() == [[0x7f, 0x7e, 0xfe, 0x44]]


def test_reference_attention():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h, 8, generator=g, dtype=torch.float64)
               for n, h in ((3, 4), (5, 2), (5, 2)))
    out = attention_rows_ref(q, k, v, 0.5)
    for j in range(3):
        for h in range(4):
            p = torch.softmax(k[:3 + j, h // 2] @ q[j, h] * 0.5, 0)
            assert torch.allclose(out[j, h], p @ v[:3 + j, h // 2])
    assert bool((attention_rows_ref(q, k[:1], v[:1], 0.5)[:2] == 0).all())
    k[4], v[4] = float("nan"), float("nan")  # seen by the last row alone
    hidden = attention_rows_ref(q, k, v, 0.5)
    assert torch.equal(hidden[:2], out[:2]) and bool(hidden[2].isnan().all())


# ---------------------------------------------------------------- the C entry points' refusals
STORE = dict(k=P, krs=512, v=P, vrs=512, kc=P, vc=P, slots=P, n=10, hk=4, d=64, ns=640)
READ = dict(kc=P, vc=P, bt=P, btrs=8, mb=8, cu=P, starts=None, n=2, nt=100, hk=4, d=64, bs=32, nb=100,
            ko=P, vo=P)
DECODE = dict(q=P, qrs=512, kc=P, vc=P, bt=P, btrs=8, ctx=P, n=2, hq=8, hk=4, d=64, bs=32, mb=8,
              nb=100, scale=0.1, out=P, ors=512, ws=P, wsb=1 << 30)
PREFILL = dict(q=P, qrs=512, tq=10, kc=P, vc=P, cq=P, ck=P, bt=P, btrs=8, mb=8, n=2, mq=10, mk=100,
               hq=8, hk=4, d=64, bs=32, nb=100, scale=0.1, out=P, ors=512, ws=None, wsb=0)
ALL = [(dict(d=96), -4, b"head_dim"), (dict(d=256), -4, b"head_dim"), (dict(kc=None), -1, b"caches"),
       (dict(vc=P + 8), -1, b"caches")]
TABLES = ALL + [(dict(bs=16), -4, b"multiple of 32"), (dict(bs=0), -4, b"multiple of 32"),
                (dict(bs=48), -4, b"multiple of 32"), (dict(btrs=4), -1, b"block table"),
                (dict(mb=0), -1, b"block table"), (dict(bt=None), -1, b"null"),
                (dict(nb=-1), -1, b"sizes"), (dict(n=-1), -1, b"sizes")]
BOTH = TABLES + [(dict(hk=3), -1, b"n_q_heads"), (dict(hq=0), -1, b"n_q_heads"),
                 (dict(scale=0.0), -1, b"scale"), (dict(scale=float("nan")), -1, b"scale"),
                 (dict(scale=float("inf")), -1, b"scale"), (dict(q=P + 8), -1, b"misaligned"),
                 (dict(q=None), -1, b"null"), (dict(out=None), -1, b"null"),
                 (dict(qrs=511), -1, b"strides"), (dict(qrs=516), -1, b"strides"),
                 (dict(ors=510), -1, b"strides"), (dict(ors=513), -1, b"strides")]
CASES = (
    [("nkv_scaled_store", STORE, *c) for c in ALL + [
        (dict(n=-1), -1, b"sizes"), (dict(n=1 << 31), -1, b"sizes"), (dict(ns=-32), -1, b"sizes"),
        (dict(hk=0), -4, b"KV heads"), (dict(hk=513, krs=1 << 20, vrs=1 << 20), -4, b"KV heads"),
        (dict(ns=650), -1, b"whole tiles"), (dict(slots=None), -1, b"null"), (dict(k=None), -1, b"null"),
        (dict(v=P + 2), -1, b"misaligned"), (dict(krs=255), -1, b"strides"),
        (dict(vrs=260), -1, b"strides"), (dict(n=0, k=None), 0, b"")]]
    + [("nkv_scaled_read", READ, *c) for c in TABLES + [
        (dict(nt=-1), -1, b"sizes"), (dict(nt=(1 << 27) + 1), -4, b"at most"),
        (dict(n=(1 << 20) + 1), -4, b"at most"), (dict(hk=0), -4, b"KV heads"),
        (dict(cu=None), -1, b"null"), (dict(ko=P + 2), -1, b"misaligned"), (dict(vo=None), -1, b"null"),
        (dict(n=0, cu=None), 0, b""), (dict(nt=0), 0, b"")]]
    + [("nkv_scaled_decode", DECODE, *c) for c in BOTH + [
        (dict(hk=0), -4, b"KV heads"), (dict(hq=257 * 4), -4, b"above 256"), (dict(ctx=None), -1, b"null"),
        (dict(ws=None), -3, b"workspace"), (dict(ws=P + 4), -3, b"workspace"),
        (dict(wsb=100), -3, b"workspace"), (dict(mb=1 << 26, btrs=1 << 26), -4, b"too large"),
        (dict(n=1 << 24, mb=1 << 10, btrs=1 << 10), -4, b"too many"), (dict(n=0, ws=None), 0, b"")]]
    + [("nkv_scaled_prefill", PREFILL, *c) for c in BOTH + [
        (dict(hk=0), -4, b"KV heads"), (dict(hq=129 * 4), -4, b"above 128"), (dict(cq=None), -1, b"null"),
        (dict(ck=None), -1, b"null"), (dict(tq=-1), -1, b"sizes"), (dict(tq=1 << 31), -1, b"sizes"),
        (dict(mq=-1), -1, b"sizes"), (dict(out=P + 4), -1, b"misaligned"),
        (dict(ors=514), -1, b"strides"), (dict(nb=1 << 31), -4, b"too large"),
        (dict(mb=1 << 27, btrs=1 << 27), -4, b"too large"), (dict(n=1 << 30, mq=1 << 20), -4, b"too many"),
        (dict(ws=P, wsb=100, mk=100000), -3, b"workspace"),
        (dict(ws=P + 8, wsb=1 << 40, mk=100000), -3, b"workspace"),
        (dict(n=0), 0, b""), (dict(tq=0), 0, b""), (dict(mq=0), 0, b"")]]
)


@pytest.mark.parametrize("name,base,kw,code,msg", CASES)
def test_entry_points_refuse(name, base, kw, code, msg):
    a = dict(base, **kw)
    scale = [a.pop("scale")] if "scale" in a else []
    args = [0 if x is None else x for x in (*a.values(), None)] + scale  # the stream: NULL
    rc = getattr(L.lib(), name)(struct.pack(f"{len(args) - len(scale)}q{len(scale)}d", *args))
    assert rc == code and msg in L.lib().nkv_last_error(), (rc, L.lib().nkv_last_error())


def test_entry_points_refuse_null_arguments():
    for name in ("store", "read", "decode", "prefill"):
        assert getattr(L.lib(), "nkv_scaled_" + name)(None) == -1
        assert b"null arguments" in L.lib().nkv_last_error()


def test_page_calls_refuse():
    def args(block, row=2 * 64 + PAD):
        return struct.pack("13q", P, 4, 10, block, row, P, P, P, 8, 8, 5, P, 1 << 30)

    f, t = L.lib().nkv_scaled_pages_fork, L.lib().nkv_scaled_pages_truncate
    assert f(args(48), P, P, 1, 1, P, None) == -4 and b"multiple of 32" in L.lib().nkv_last_error()
    assert t(args(16), P, P, 1, None, 0, P, None) == -4
    assert f(None, P, P, 1, 1, P, None) == -4 and t(None, P, P, 1, None, 0, P, None) == -4
    assert f(args(32, 100), P, P, 1, 1, P, None) == -4 and b"16 bytes" in L.lib().nkv_last_error()
    assert f(args(32), P, P, -1, 1, P, None) == -1 and t(args(32), P, P, -1, None, 0, P, None) == -1
    # nothing listed: no launch, and no plan of this call's to go on with
    assert f(args(32), None, None, 0, 1, None, None) == 0
    assert t(args(32), None, None, 0, None, 0, None, None) == 0


def test_workspace_follows_the_chip():
    """(no device here: 256 CUs assumed)"""
    f = L.lib().nkv_scaled_prefill_workspace_bytes
    assert f(0, 10, 10, 100, 8, 4, 64) == f(2, 0, 10, 100, 8, 4, 64) == f(2, 10, 0, 100, 8, 4, 64) == 0
    assert f(2, 10, 10, 100, 7, 4, 64) == f(2, 10, 10, 100, 8, 4, 32) == f(2, 10, 10, 100, 8, 0, 64) == 0
    assert f(1, 500, 500, 500, 0, 4, 64) == f(1, 8, 8, 9000, 129 * 4, 4, 64) == 0
    assert f(1, 8, 8, 9000, 32, 8, 128) > 0 == f(1, 8, 8, 100, 32, 8, 128)
    assert f(1, 8, 8, 10 ** 5, 32, 8, 128) == f(1, 8, 8, 10 ** 7, 32, 8, 128)  # by the chip
    assert f(8, 16384, 2048, 10 ** 5, 32, 8, 128) == 0  # whole tiles fill it
    for n, tq, mq in ((1, 512, 512), (4, 36, 9), (30, 1000, 500), (2000, 2000, 1), (64, 128, 2)):
        for d in (64, 128):
            assert f(n, tq, mq, 10 ** 6, 32, 8, d) < 600e6


def test_prefill_maxima_of_any_size():
    """max_seqlen_q and max_seqlen_k far past what there is: as if they were q's rows and 2^31 keys; more
    tiles than a launch holds are refused, not counted wrongly."""
    f = L.lib().nkv_scaled_prefill_workspace_bytes
    for n, tq in ((1, 8), (4, 36), (16, 64)):
        assert f(n, tq, 1 << 62, 10 ** 6, 32, 8, 128) == f(n, tq, tq, 10 ** 6, 32, 8, 128) > 0
    assert f(1, 8, 8, 1 << 62, 32, 8, 128) == f(1, 8, 8, (1 << 31) - 1, 32, 8, 128)
    assert f(1, 8, 8, -(1 << 62), 32, 8, 128) == 0 == f((1 << 20) + 1, 8, 8, 9000, 32, 8, 128)
    for kw in (dict(n=1 << 20, tq=1 << 30, mq=1 << 62, hk=512, hq=512, qrs=1 << 15, ors=1 << 15),
               dict(n=(1 << 20) + 1), dict(n=1 << 62)):
        test_entry_points_refuse("nkv_scaled_prefill", PREFILL, kw, -4, b"too many")


# ---------------------------------------------------------------- the wrappers' refusals
def _gpu_free(monkeypatch):
    """The checks of the wrappers, with host tensors taken for the GPU's."""
    monkeypatch.setattr(L, "require_device", lambda device, **kw: None)


def test_wrappers_refuse_host_tensors():
    c, x = torch.zeros(2, 32, 2 * 64 + PAD, dtype=U8), torch.zeros(2, 2, 64, dtype=BF)
    i = torch.zeros(3, dtype=I32)
    bt = torch.zeros(2, 2, dtype=I32)
    for call in (lambda: nkv.scaled_store_kvcache(x, x, c, c, i[:2]),
                 lambda: nkv.scaled_read_kvcache(c, c, bt, i, 2, 2),
                 lambda: nkv.scaled_paged_decode(x, c, c, i, bt, 0.1),
                 lambda: nkv.scaled_varlen_prefill(x, c, c, i, i, 1, 0.1, bt)):
        with pytest.raises(ValueError, match="expected GPU"):
            call()


def test_wrappers_refuse_shapes_and_types(monkeypatch):
    _gpu_free(monkeypatch)
    c, x = torch.zeros(2, 32, 2 * 64 + PAD, dtype=U8), torch.zeros(2, 2, 64, dtype=BF)
    i, bt = torch.zeros(3, dtype=I32), torch.zeros(2, 2, dtype=I32)
    bad_caches = [(c.view(torch.int8), c), (c, c[:1]), (c[:, :16], c[:, :16]), (c[..., :-8], c[..., :-8]),
                  (c[:, :, None], c[:, :, None]), (c.transpose(0, 1), c.transpose(0, 1)),
                  (torch.zeros(2, 48, 144, dtype=U8),) * 2, (torch.zeros(2, 0, 144, dtype=U8),) * 2]
    calls = {
        "store": lambda k, v: nkv.scaled_store_kvcache(x, x, k, v, i[:2]),
        "read": lambda k, v: nkv.scaled_read_kvcache(k, v, bt, i, 2, 2),
        "decode": lambda k, v: nkv.scaled_paged_decode(x, k, v, i, bt, 0.1),
        "prefill": lambda k, v: nkv.scaled_varlen_prefill(x, k, v, i, i, 1, 0.1, bt),
    }
    for name, call in calls.items():
        for k, v in bad_caches:
            with pytest.raises(ValueError, match="scaled_"):
                call(k, v)
    f16, wide = x.half(), torch.zeros(2, 2, 128, dtype=BF)[..., :64]
    for y in (f16, wide, x[0], x.transpose(0, 1)[..., ::2]):
        with pytest.raises(ValueError, match="key must be"):
            nkv.scaled_store_kvcache(y, x, c, c, i[:2])
        with pytest.raises(ValueError, match="value"):
            nkv.scaled_store_kvcache(x, y, c, c, i[:2])
        with pytest.raises(ValueError, match="q must be"):
            nkv.scaled_paged_decode(y, c, c, i, bt, 0.1)
        with pytest.raises(ValueError, match="q must be"):
            nkv.scaled_varlen_prefill(y, c, c, i, i, 1, 0.1, bt)
    with pytest.raises(ValueError, match="value shape"):
        nkv.scaled_store_kvcache(x, x[:1], c, c, i[:2])
    with pytest.raises(ValueError, match="3 slots for 2"):
        nkv.scaled_store_kvcache(x, x, c, c, i)
    for s in (i[:1], i[:2].long(), torch.zeros(4, dtype=I32)[::2]):
        with pytest.raises(ValueError, match="slot_mapping"):
            nkv.scaled_store_kvcache(x, x, c, c, s)
    for hk in (0, 3, -1):
        with pytest.raises(ValueError, match="heads"):
            nkv.scaled_read_kvcache(c, c, bt, i, 2, hk)
    with pytest.raises(ValueError, match="starts"):
        nkv.scaled_read_kvcache(c, c, bt, i, 2, 2, starts=i[:1])
    with pytest.raises(ValueError, match="n_tokens"):
        nkv.scaled_read_kvcache(c, c, bt, i, -1, 2)
    with pytest.raises(ValueError, match="cu_seqlens"):
        nkv.scaled_read_kvcache(c, c, bt, i[:0], 2, 2)
    for o in ((x, x.half()), (x[:1], x), (x, torch.zeros(2, 2, 128, dtype=BF)[..., ::2])):
        with pytest.raises(ValueError, match="out must be"):
            nkv.scaled_read_kvcache(c, c, bt, i, 2, 2, out=o)
    for o in (x.half(), x[:1], torch.zeros(2, 2, 128, dtype=BF)[..., :64]):
        with pytest.raises(ValueError, match="out must be"):
            nkv.scaled_paged_decode(x, c, c, i, bt, 0.1, out=o)
        with pytest.raises(ValueError, match="out must be"):
            nkv.scaled_varlen_prefill(x, c, c, i, i, 1, 0.1, bt, out=o)
    for w in (torch.zeros(99), torch.zeros(99, dtype=U8)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            nkv.scaled_paged_decode(x, c, c, i, bt, 0.1, workspace=w)
        with pytest.raises(ValueError, match="workspace"):
            nkv.scaled_varlen_prefill(x, c, c, i, i, 1, 0.1, bt, workspace=w)
    for lens in (i[:1], i.long()):
        with pytest.raises(ValueError, match="context_lens"):
            nkv.scaled_paged_decode(x, c, c, lens, bt, 0.1)
    for t in (bt[:1], bt.long(), bt[:, :0], torch.zeros(2, 4, dtype=I32)[:, ::2]):
        with pytest.raises(ValueError, match="block_tables"):
            nkv.scaled_paged_decode(x, c, c, i, t, 0.1)
        with pytest.raises(ValueError, match="block_tables"):
            nkv.scaled_varlen_prefill(x, c, c, i, i, 1, 0.1, t)
        with pytest.raises(ValueError, match="block_tables"):
            nkv.scaled_read_kvcache(c, c, t, i, 2, 2)
    with pytest.raises(ValueError, match="cu_seqlens"):
        nkv.scaled_varlen_prefill(x, c, c, i, i[:2], 1, 0.1, bt)


def test_pool_refuses():
    pool = nkv.ScaledKVCachePool(3, 2, 64, 32, num_blocks=5, device="cpu")
    assert pool.kv_cache.shape == (2, 3, 5, 32, 2 * 64 + PAD) and not bool(pool.kv_cache.any())
    assert pool.block_bytes * 5 == pool.kv_cache.numel()
    layers = [types.SimpleNamespace(k_cache=None, v_cache=None) for _ in range(3)]
    assert pool.bind(layers + [object()]) == 3
    assert layers[1].v_cache.data_ptr() == pool.kv_cache[1, 1].data_ptr()
    for args in ((1, 2, 96), (1, 0, 64), (1, 513, 64), (0, 2, 64), (1, 2, 64, 48), (1, 2, 64, 0)):
        with pytest.raises(ValueError, match="ScaledKVCachePool"):
            nkv.ScaledKVCachePool(*args, num_blocks=5, device="cpu")
    with pytest.raises(RuntimeError, match="no device memory"):
        nkv.ScaledKVCachePool(1, 2, 64, num_blocks=0, device="cpu")


def test_paged_sequences_refuse():
    with pytest.raises(ValueError, match="multiple of 32"):
        pages.PagedSequences(torch.zeros(2, 1, 4, 48, 144, dtype=U8), 2, 2)
    with pytest.raises(ValueError, match="contiguous"):
        pages.PagedSequences(torch.zeros(2, 1, 4, 32, 144, dtype=torch.int8), 2, 2)
    with pytest.raises(ValueError, match="expected GPU"):
        pages.PagedSequences(nkv.ScaledKVCachePool(1, 2, 64, 32, num_blocks=4, device="cpu"), 2, 2)


def _layer(Hk=2, D=64, enabled=False, Hq=4):
    cfg = types.SimpleNamespace(kv_compress_enabled=enabled, kv_compress_window_blocks=4,
                                kv_compress_keep_blocks=2, kv_compress_keep_extra_tokens=1)
    return nkv.Attention(Hq, D, 0.1, Hk, cfg, 1)


@pytest.mark.parametrize("layer,cache,msg", [
    (_layer(), (2, 32, 4 * 64 + PAD), "must be"), (_layer(), (2, 48, 2 * 64 + PAD), "multiple of 32"),
    (_layer(), (2, 32, 2, 64 + PAD), "must be"), (_layer(D=256), (2, 32, 2 * 256 + PAD), "head_dim"),
    (_layer(enabled=True), (2, 32, 2 * 64 + PAD), "compression"),
])
def test_layer_refuses_another_geometry_than_its_own(layer, cache, msg):
    layer.k_cache = layer.v_cache = torch.zeros(cache, dtype=U8)
    nkv.set_context(True)
    try:
        with pytest.raises(ValueError, match=msg):
            layer(torch.zeros(1, 4, layer.head_dim, dtype=BF), None, None, 0)
    finally:
        nkv.reset_context()


def test_layer_calls_with_q_s_device_as_the_current_one(monkeypatch):
    """Launches and sizes that depend on the chip are made on q's device."""
    inside, seen = [], []

    class Device:
        def __enter__(self):
            inside.append(1)

        def __exit__(self, *a):
            inside.pop()

    monkeypatch.setattr(L, "device_of", lambda index: Device())
    att = importlib.import_module("nanokv-llm_amd.layers.attention")
    for name in ("scaled_store_kvcache", "scaled_paged_decode", "scaled_varlen_prefill",
                 "varlen_prefill", "shared_decode_workspace"):
        monkeypatch.setattr(att, name,
                            lambda *a, n=name, **kw: seen.append((n, len(inside))) or torch.zeros(1))
    layer = _layer()
    layer.k_cache = layer.v_cache = torch.zeros(2, 32, 2 * 64 + PAD, dtype=U8)
    q, kv = torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF)
    lens, bt = torch.ones(2, dtype=I32), torch.zeros(2, 2, dtype=I32)
    try:
        for decode, tables, stored in ((True, bt, False), (False, bt, True), (False, None, False)):
            nkv.set_context(decode, lens, lens, 1, 1, lens, lens, tables)
            layer(q, kv, kv, 0, kv_stored=stored)
    finally:
        nkv.reset_context()
    assert seen == [("scaled_store_kvcache", 1), ("shared_decode_workspace", 1),
                    ("scaled_paged_decode", 1), ("scaled_varlen_prefill", 1),
                    ("scaled_store_kvcache", 1), ("varlen_prefill", 1)]


def test_other_operators_refuse_such_a_cache(monkeypatch):
    """Read as an ordinary cache its bytes would be taken for rows."""
    _gpu_free(monkeypatch)
    c, x = torch.zeros(2, 32, 2 * 64 + PAD, dtype=U8), torch.zeros(2, 2, 64, dtype=BF)
    i, bt = torch.zeros(3, dtype=I32), torch.zeros(2, 2, dtype=I32)
    l = torch.zeros(4, 64)
    for call in (lambda: nkv.store_kvcache(x, x, c, c, i[:2]),
                 lambda: nkv.paged_decode(x, c, c, i, bt, 0.1),
                 lambda: nkv.varlen_prefill(x, c, c, i, i, 1, 0.1, block_tables=bt),
                 lambda: nkv.diff_paged_decode(x, c, c, i, bt, 0.1, l, 0.2),
                 lambda: nkv.qk_norm_rope_store(torch.zeros(2, dtype=torch.int64), x, x, x,
                                                torch.zeros(9, 64), k_cache=c, v_cache=c,
                                                slot_mapping=i[:2])):
        with pytest.raises((ValueError, AssertionError)):
            call()
