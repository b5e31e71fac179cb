"""Differential attention: the reference's own rules, and the refusals that need no GPU."""
import importlib
import math

import pytest
import torch

from oracle.diff_attention_ref import diff_attention_ref, gather_rows

da = importlib.import_module("nanokv-llm_amd.layers.diff_attention")
L = importlib.import_module("nanokv-llm_amd._lib")
BF, I32 = torch.bfloat16, torch.int32
P = 0x10000


def test_reference_against_two_softmaxes():
    """One pair, written out: the difference of torch's softmaxes, the norm, the weight; lambda = 0
    leaves the first map, and a row that sees nothing is zero."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, 2, 8, generator=g, dtype=torch.float64) for n in (3, 5, 5))
    l, w = torch.randn(4, 8, generator=g) * 0.3, torch.randn(16, generator=g)
    lam = math.exp(float(l[0].double() @ l[1].double())) \
        - math.exp(float(l[2].double() @ l[3].double())) + 0.3
    out = diff_attention_ref(q, k, v, 0.5, l, 0.3, w)
    for j in range(3):
        n = 3 + j
        a = [torch.softmax(k[:n, m] @ q[j, m] * 0.5, 0) @ v[:n].flatten(1) for m in (0, 1)]
        o = a[0] - lam * a[1]
        want = 0.7 * o / (o.square().mean() + 1e-5).sqrt() * w.double()
        assert torch.allclose(out[j, 0], want, rtol=1e-12, atol=1e-12)
    zero = torch.zeros(4, 8)
    first = diff_attention_ref(q, k, v, 0.5, zero, 0.0, eps=1e-9)  # lambda = 1 - 1 + 0
    o = torch.softmax(k[:, 0] @ q[2, 0] * 0.5, 0) @ v.flatten(1)
    assert torch.allclose(first[2, 0], o / o.square().mean().sqrt(), rtol=1e-6)
    assert bool((diff_attention_ref(q, k[:2], v[:2], 0.5, l, 0.3, w)[0] == 0).all())


def test_gathered_rows():
    cache = torch.arange(3 * 2, dtype=torch.float32).view(3, 2, 1, 1)
    table = torch.tensor([2, -1, 0])
    assert gather_rows(cache, table, 5, 2).flatten().tolist() == [4, 5, 0]
    assert gather_rows(cache, table, 7, 2, zeros=True).flatten().tolist() == [4, 5, 0, 0, 0, 1, 0]


def test_lambda_init():
    assert da.lambda_init_of(0) == pytest.approx(0.2)
    assert da.lambda_init_of(1000) == pytest.approx(0.8)


def test_layer_refuses_what_the_kernels_do_not_take():
    D = importlib.import_module("nanokv-llm_amd").DifferentialAttention
    D(8, 64, 0.125, 4, 0.2)
    for args in ((8, 32, 0.1, 4, 0.2), (8, 256, 0.1, 4, 0.2), (7, 64, 0.1, 7, 0.2),
                 (8, 64, 0.1, 3, 0.2), (12, 64, 0.1, 8, 0.2), (130, 64, 0.1, 2, 0.2),
                 (8, 64, 0.0, 4, 0.2), (8, 64, 0.1, 4, 0.2, 0.0)):
        with pytest.raises(ValueError, match="DifferentialAttention"):
            D(*args)


def test_layer_refuses_a_compression_step():
    nkv = importlib.import_module("nanokv-llm_amd")
    layer = nkv.DifferentialAttention(8, 64, 0.125, 4, 0.2)
    nkv.set_context(True)
    nkv.get_context().is_compress_step = True
    try:
        with pytest.raises(ValueError, match="compression"):
            layer(None, None, None)
    finally:
        nkv.reset_context()


def test_wrappers_refuse_host_tensors():
    q, kc = torch.zeros(2, 8, 64, dtype=BF), torch.zeros(4, 16, 4, 64, dtype=BF)
    lens, bt, l = torch.ones(2, dtype=I32), torch.zeros(2, 4, dtype=I32), torch.zeros(4, 64)
    with pytest.raises(ValueError, match="expected GPU"):
        da.diff_paged_decode(q, kc, kc, lens, bt, 0.1, l, 0.2)
    with pytest.raises(ValueError, match="expected GPU"):
        da.diff_varlen_prefill(q, kc, kc, lens, lens, 1, 0.1, l, 0.2, block_tables=bt)


DECODE = dict(kv=0, q=P, qrs=512, k=P, v=P, bt=P, btrs=8, ctx=P, n=2, hq=8, hk=4, d=64, bs=16, mb=8,
              nb=100, scale=0.1, ks=1.0, vs=1.0, l=P, init=0.2, w=P, eps=1e-5, out=P, ors=512, ws=P,
              wsb=1 << 30)
PREFILL = dict(kv=0, q=P, qrs=512, tq=10, k=P, v=P, krs=256, vrs=256, cq=P, ck=P, bt=P, btrs=8,
               mb=8, n=2, mq=10, mk=100, hq=8, hk=4, d=64, bs=16, rows=1600, scale=0.1, ks=1.0,
               vs=1.0, l=P, init=0.2, w=P, eps=1e-5, out=P, ors=512, ws=None, wsb=0)
BOTH = [
    (dict(kv=3), -1, b"kv_type"), (dict(hq=7), -1, b"pairs"), (dict(hk=3), -1, b"pairs"),
    (dict(hq=12, hk=8), -1, b"pairs"), (dict(hq=0), -1, b"pairs"), (dict(d=96), -4, b"head_dim"),
    (dict(d=256), -4, b"head_dim"), (dict(hq=260, hk=4), -4, b"above 64"),
    (dict(scale=0.0), -1, b"scales"), (dict(scale=float("nan")), -1, b"scales"),
    (dict(ks=0.0), -1, b"scales"), (dict(vs=float("inf")), -1, b"scales"),
    (dict(init=float("inf")), -1, b"lambda_init"), (dict(eps=0.0), -1, b"eps"),
    (dict(l=None), -1, b"lambdas"), (dict(w=P + 4), -1, b"norm_weight"),
    (dict(out=P + 2), -1, b"8-byte"), (dict(ors=500), -1, b"stride"), (dict(ors=514), -1, b"stride"),
    (dict(q=P + 8), -1, b"16-byte"), (dict(k=P + 8), -1, b"16-byte"),
    (dict(qrs=511), -1, b"stride"), (dict(bs=8), -4, b"multiple of 16"),
    (dict(btrs=4), -1, b"block table"),
]


@pytest.mark.parametrize("name,base", [("nkv_diff_decode", DECODE), ("nkv_diff_prefill", PREFILL)])
@pytest.mark.parametrize("kw,code,msg", BOTH)
def test_entry_points_refuse(name, base, kw, code, msg):
    rc = getattr(L.lib(), name)(*dict(base, **kw).values(), None)
    assert rc == code and msg in L.lib().nkv_last_error(), (rc, L.lib().nkv_last_error())


@pytest.mark.parametrize("kw,code,msg", [
    (dict(q=None), -1, b"null"), (dict(cq=None), -1, b"null"), (dict(out=None), -1, b"null"),
    (dict(n=-1), -1, b"sizes"), (dict(tq=-1), -1, b"sizes"), (dict(tq=1 << 31), -1, b"sizes"),
    (dict(krs=250), -1, b"row strides"), (dict(vrs=1 << 24), -1, b"row strides"),
    (dict(krs=264), -1, b"paged rows"), (dict(kv=2, bt=None), -4, b"paged"),
    (dict(bt=None, rows=1 << 31), -4, b"too many"), (dict(ws=P + 8, wsb=1 << 40), -3, b"workspace"),
    (dict(ws=P, wsb=100, mq=10, mk=100000), -3, b"workspace"),
    (dict(n=0), 0, b""), (dict(tq=0), 0, b""),
])
def test_prefill_refuses(kw, code, msg):
    rc = L.lib().nkv_diff_prefill(*dict(PREFILL, **kw).values(), None)
    assert rc == code and msg in L.lib().nkv_last_error(), (rc, L.lib().nkv_last_error())


@pytest.mark.parametrize("kw,code,msg", [
    (dict(q=None), -1, b"null"), (dict(ctx=None), -1, b"null"), (dict(out=None), -1, b"out must"),
    (dict(n=-1), -1, b"sizes"), (dict(ws=None), -3, b"workspace"), (dict(wsb=100), -3, b"workspace"),
    (dict(mb=1 << 27, btrs=1 << 27), -4, b"too large"), (dict(n=0, out=None), 0, b""),
])
def test_decode_refuses(kw, code, msg):
    rc = L.lib().nkv_diff_decode(*dict(DECODE, **kw).values(), None)
    assert rc == code and msg in L.lib().nkv_last_error(), (rc, L.lib().nkv_last_error())


def test_workspace_sizes_follow_the_chip_not_the_lengths():
    """(no device here: 256 CUs assumed)"""
    f = L.lib().nkv_diff_prefill_workspace_bytes
    assert f(0, 0, 10, 10, 10, 8, 4, 64, 1) == f(0, 2, 10, 10, 100, 7, 4, 64, 1) == 0
    assert f(0, 2, 10, 10, 100, 8, 4, 32, 1) == 0
    # one long chunk: cut; a batch that fills the chip: whole tiles, nothing needed
    assert 0 < f(0, 1, 512, 512, 10 ** 4, 32, 8, 128, 1) == f(0, 1, 512, 512, 10 ** 6, 32, 8, 128, 1)
    assert f(0, 8, 16384, 2048, 10 ** 5, 32, 8, 128, 1) == 0
    for d in (64, 128):
        for n, tq, mq in ((1, 512, 512), (500, 1010, 511), (2000, 2000, 1), (300, 600, 2),
                          (1000, 1600, 100)):
            assert f(0, n, tq, mq, 10 ** 6, 32, 8, d, 1) < 900e6
    assert L.lib().nkv_diff_decode_workspace_bytes(4, 32, 96, 8, 256) == 0
    assert L.lib().nkv_diff_decode_workspace_bytes(4, 32, 64, 8, 256) == \
        L.lib().nkv_paged_decode_workspace_bytes(4, 32, 128, 8, 256)


def test_layer_refuses_another_geometry_than_its_own(monkeypatch):
    """A cache or rows of other heads would be read over the wrong pairs: before anything runs."""
    nkv = importlib.import_module("nanokv-llm_amd")

    def launched(*a, **kw):
        raise AssertionError("launched")

    for name in ("store_kvcache", "diff_paged_decode", "diff_varlen_prefill",
                 "shared_decode_workspace"):
        monkeypatch.setattr(da, name, launched)
    layer = nkv.DifferentialAttention(8, 64, 0.125, 4, 0.2)

    def rows(heads, d=64):
        return torch.zeros(2, heads, d, dtype=BF)

    def cache(hk=4, d=64, B=16):
        return torch.zeros(3, B, hk, d, dtype=BF)

    lens, bt = torch.ones(2, dtype=I32), torch.zeros(2, 3, dtype=I32)
    cu = torch.tensor([0, 1, 2], dtype=I32)
    try:
        for decode, tables in ((True, bt), (False, bt), (False, None)):
            nkv.set_context(decode, cu, cu, 1, 1, lens, lens, tables)
            for stored in (False, True):
                for kc in (cache(2), cache(8), cache(d=128), cache(B=24), cache()[0]):
                    layer.k_cache = layer.v_cache = kc
                    with pytest.raises(ValueError, match="k_cache must be|block_size"):
                        layer(rows(8), rows(4), rows(4), kv_stored=stored)
                layer.k_cache = layer.v_cache = cache()
                for q in (rows(16), rows(4), rows(8, 128), rows(8)[0]):
                    with pytest.raises(ValueError, match="q must be"):
                        layer(q, rows(4), rows(4), kv_stored=stored)
        layer.k_cache = layer.v_cache = torch.tensor([])  # a first prompt without a cache
        with pytest.raises(ValueError, match="k and v must be"):
            layer(rows(8), rows(2), rows(2))
        nkv.set_context(True, cu, cu, 1, 1, lens, lens, bt)
        with pytest.raises(ValueError, match="no cache"):
            layer(rows(8), rows(4), rows(4))
    finally:
        nkv.reset_context()


def test_another_device_than_the_current_one(monkeypatch):
    """Every launch, the store's too, and every size that depends on the chip are made with q's
    device as the current one: a null stream belongs to that."""
    nkv = importlib.import_module("nanokv-llm_amd")
    inside, seen = [], []

    class Device:
        def __enter__(self):
            inside.append(1)

        def __exit__(self, *a):
            inside.pop()

    class Lib:
        def __getattr__(self, name):
            return lambda *a: seen.append((name, bool(inside))) or 0

    attn = importlib.import_module("nanokv-llm_amd.layers.attention")
    lib = Lib()
    monkeypatch.setattr(L, "lib", lambda: lib)
    monkeypatch.setattr(L, "require_device", lambda *a, **kw: None)
    monkeypatch.setattr(L, "device_of", lambda index: Device())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing",
                        lambda: seen.append(("capturing", bool(inside))) or False)
    monkeypatch.setattr(attn, "_SHARED_WS", {})
    layer = nkv.DifferentialAttention(8, 64, 0.125, 4, 0.2)
    layer.norm_weight.data = layer.norm_weight.data.to(BF)
    layer.k_cache = layer.v_cache = torch.zeros(3, 16, 4, 64, dtype=BF)
    q, k = torch.zeros(2, 8, 64, dtype=BF), torch.zeros(2, 4, 64, dtype=BF)
    lens, bt = torch.ones(2, dtype=I32), torch.zeros(2, 3, dtype=I32)
    cu = torch.tensor([0, 1, 2], dtype=I32)
    try:
        for decode, tables in ((True, bt), (False, bt), (False, None)):
            nkv.set_context(decode, cu, cu, 1, 1, lens, lens, tables)
            layer(q, k, k)
    finally:
        nkv.reset_context()
    da.diff_paged_decode(q, layer.k_cache, layer.k_cache, lens, bt, 0.1, layer.lambdas, 0.2)
    names = {n for n, _ in seen}
    assert {"nkv_store_kvcache", "nkv_diff_decode", "nkv_diff_prefill", "capturing",
            "nkv_diff_decode_workspace_bytes", "nkv_diff_prefill_workspace_bytes"} <= names
    assert all(ok for _, ok in seen), [n for n, ok in seen if not ok]


def test_layer_refuses_host_tensors():
    nkv = importlib.import_module("nanokv-llm_amd")
    layer = nkv.DifferentialAttention(8, 64, 0.125, 4, 0.2)
    layer.k_cache = layer.v_cache = torch.zeros(3, 16, 4, 64, dtype=BF)
    q, k = torch.zeros(2, 8, 64, dtype=BF), torch.zeros(2, 4, 64, dtype=BF)
    nkv.set_context(True, None, None, 1, 1, torch.ones(2, dtype=I32), torch.ones(2, dtype=I32),
                    torch.zeros(2, 3, dtype=I32))
    try:
        with pytest.raises(ValueError, match="expected GPU"):
            layer(q, k, k)
    finally:
        nkv.reset_context()


def test_a_device_without_memory_takes_the_launch_that_needs_none(monkeypatch):
    """No workspace left: the prefill runs without one, as without max_seqlen_k."""
    calls = []

    class Lib:
        def nkv_diff_prefill_workspace_bytes(self, *a):
            return 1 << 40

        def nkv_diff_prefill(self, *a):
            calls.append(a)
            return 0

    lib, empty = Lib(), torch.empty

    def no_memory(*size, **kw):
        if size == (1 << 40,):
            raise torch.OutOfMemoryError("no memory")
        return empty(*size, **kw)

    monkeypatch.setattr(L, "lib", lambda: lib)
    monkeypatch.setattr(L, "require_device", lambda *a, **kw: None)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(torch, "empty", no_memory)
    q, kc = torch.zeros(2, 8, 64, dtype=BF), torch.zeros(4, 16, 4, 64, dtype=BF)
    cu, bt, l = torch.tensor([0, 2], dtype=I32), torch.zeros(1, 4, dtype=I32), torch.zeros(4, 64)
    assert da.diff_prefill_workspace(q, kc, 1, 2, 60) is None
    da.diff_varlen_prefill(q, kc, kc, cu, cu, 2, 0.1, l, 0.2, block_tables=bt, max_seqlen_k=60)
    assert calls[0][-3:] == (None, 0, 0)  # workspace, bytes, stream
