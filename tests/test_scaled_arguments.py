"""Block-scaled caches: right arguments reach the library without the checks by name, which are for wrong
ones (they keep the host busy for longer than a small call runs). Host tensors stand in for the GPU's."""
import contextlib
import struct
import types

import pytest
import torch

from test_scaled_checks import BF, I32, L, PAD, U8, nkv, sc, _layer


@pytest.fixture
def calls(monkeypatch):
    """What reached the library: (entry point, its fields)."""
    seen = []

    def entry(name, fmt):
        return lambda packed: seen.append((name, struct.unpack(fmt, packed))) or 0

    lib = types.SimpleNamespace(
        nkv_scaled_store=entry("store", "12q"), nkv_scaled_read=entry("read", "16q"),
        nkv_scaled_decode=entry("decode", "19qd"), nkv_scaled_prefill=entry("prefill", "23qd"),
        nkv_paged_decode_workspace_bytes=lambda *a: 64,
        nkv_scaled_prefill_workspace_bytes=lambda *a: 0)
    monkeypatch.setattr(L, "lib", lambda: lib)
    monkeypatch.setattr(L, "device_of", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(L, "require_device", lambda device, **kw: None)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    sc._decode_bytes.cache_clear()
    yield seen
    sc._decode_bytes.cache_clear()


@pytest.fixture
def no_names(monkeypatch):
    def refuse(what, *a):
        raise AssertionError(f"{what}: checked by name")

    for op in ("store", "read", "decode", "prefill"):
        monkeypatch.setattr(sc, "_refuse_" + op, refuse)


C = torch.zeros(2, 32, 2 * 64 + PAD, dtype=U8)
Q, KV = torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF)
LENS, BT = torch.zeros(3, dtype=I32), torch.zeros(2, 2, dtype=I32)
WS = torch.zeros(256, dtype=U8)


@pytest.mark.parametrize("out", [None, torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 6, 64, dtype=BF)[:, :4]])
@pytest.mark.parametrize("workspace", [None, WS])
def test_attention_with_outputs_and_workspaces(calls, no_names, out, workspace):
    nkv.scaled_paged_decode(Q, C, C, LENS, BT, 0.1, out=out, workspace=workspace)
    nkv.scaled_varlen_prefill(Q, C, C, LENS, LENS, 1, 0.1, BT, out=out, workspace=workspace, max_seqlen_k=9)
    assert [n for n, _ in calls] == ["decode", "prefill"]
    for (_, a), at in zip(calls, (14, 18)):  # out, its stride, workspace, its bytes
        if out is not None:
            assert a[at:at + 2] == (out.data_ptr(), out.stride(0))
        if workspace is not None:
            assert a[at + 2:at + 4] == (WS.data_ptr(), 256)


def test_rows_read_into_outputs(calls, no_names):
    out = (torch.zeros(2, 2, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF))
    assert nkv.scaled_read_kvcache(C, C, BT, LENS, 2, 2, out=out) is out
    assert calls[0][1][13:15] == (out[0].data_ptr(), out[1].data_ptr())


def test_the_layer(calls, no_names, monkeypatch):
    """Its decode passes the workspace that the device's layers share."""
    att = nkv.Attention.forward.__globals__
    monkeypatch.setitem(att, "shared_decode_workspace", lambda device, nbytes: WS)
    layer = _layer()
    layer.k_cache = layer.v_cache = C
    nkv.set_context(True, LENS, LENS, 1, 1, LENS[:2], LENS, BT)
    try:
        layer(Q, KV, KV, 0)
    finally:
        nkv.reset_context()
    assert [n for n, _ in calls] == ["store", "decode"] and calls[1][1][16:18] == (WS.data_ptr(), 256)


@pytest.mark.parametrize("kw", [
    dict(out=torch.zeros(2, 4, 64)), dict(out=torch.zeros(2, 4, 128, dtype=BF)[..., :64]),
    dict(out=torch.zeros(2, 4, 128, dtype=BF)[..., ::2]), dict(out=torch.zeros(1, 4, 64, dtype=BF)),
    dict(workspace=WS[::2]), dict(workspace=torch.zeros(64))])
def test_wrong_outputs_and_workspaces_are_refused(calls, kw):
    what = next(iter(kw))
    with pytest.raises(ValueError, match=what):
        nkv.scaled_paged_decode(Q, C, C, LENS, BT, 0.1, **kw)
    with pytest.raises(ValueError, match=what):
        nkv.scaled_varlen_prefill(Q, C, C, LENS, LENS, 1, 0.1, BT, **kw)
    if what == "out":
        with pytest.raises(ValueError, match="out must be"):
            nkv.scaled_read_kvcache(C, C, BT, LENS, 2, 2, out=(kw["out"], kw["out"]))
    assert calls == []
    rows = torch.zeros(2, 2, 64, dtype=BF)
    for out in ((rows,), (rows, rows, rows)):
        with pytest.raises(ValueError):
            nkv.scaled_read_kvcache(C, C, BT, LENS, 2, 2, out=out)
