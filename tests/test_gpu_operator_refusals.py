"""Refusals of the page and differential-attention wrappers that need tensors on a GPU: each raises
ValueError before anything is launched, and the operators work afterwards."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

nkv = importlib.import_module("nanokv-llm_amd")
BF, F16, FP8, I32 = torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.int32


def test_paged_sequences_refuse(dev):
    kv = torch.zeros(2, 1, 8, 16, 2, 64, dtype=BF, device=dev)
    for kw in (dict(max_seqs=0), dict(max_blocks_per_seq=0),
               dict(state=torch.zeros(10, dtype=I32, device=dev)),
               dict(state=torch.zeros(8 + 4 + 20, dtype=torch.int64, device=dev)),
               dict(state=torch.zeros(8 + 4 + 20, dtype=I32))):
        with pytest.raises(ValueError):
            nkv.PagedSequences(kv, **{**dict(max_seqs=4, max_blocks_per_seq=5), **kw})
    seqs = nkv.PagedSequences(kv, 4, 5)
    rows = torch.zeros(2, dtype=I32, device=dev)
    kept = seqs.state.clone()
    for call in (lambda: seqs.append(rows.long()), lambda: seqs.append(rows.cpu()),
                 lambda: seqs.append(rows[None]), lambda: seqs.append(rows.repeat(2)[::2]),
                 lambda: seqs.append(rows, rows, 5), lambda: seqs.append(rows, n_tokens=3),
                 lambda: seqs.append(rows, torch.zeros(3, dtype=I32, device=dev)),
                 lambda: seqs.truncate(rows, rows[:1]), lambda: seqs.truncate(rows, rows.float()),
                 lambda: seqs.truncate(rows, rows, pages=rows.cpu()),
                 lambda: seqs.fork(rows, rows[:1]), lambda: seqs.compact(-1)):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(seqs.state, kept)
    assert seqs.append(rows)[1].tolist() == [1, 0]


def test_diff_attention_refuses(dev):
    def t(*shape, dtype=BF, device=dev):
        return torch.zeros(*shape, dtype=dtype, device=device)

    good = dict(q=t(2, 8, 64), k=t(4, 16, 4, 64), v=t(4, 16, 4, 64), lens=t(2, dtype=I32),
                bt=t(2, 3, dtype=I32), l=t(4, 64, dtype=torch.float32), w=t(128), out=None, ws=None)
    cu = torch.tensor([0, 1, 2], dtype=I32, device=dev)

    def decode(**kw):
        a = dict(good, **kw)
        return nkv.diff_paged_decode(a["q"], a["k"], a["v"], a["lens"], a["bt"], 0.1, a["l"], 0.2,
                                     a["w"], out=a["out"], workspace=a["ws"])

    def prefill(**kw):
        a = dict(good, **kw)
        return nkv.diff_varlen_prefill(a["q"], a["k"], a["v"], a.get("cu", cu), a.get("ck", cu), 1,
                                       0.1, a["l"], 0.2, a["w"], block_tables=a["bt"], out=a["out"],
                                       workspace=a["ws"])

    shared = [dict(q=t(2, 8, 128)[..., ::2]), dict(q=t(2, 8, 64, dtype=torch.float32)),
              dict(q=t(2, 8, 64, dtype=F16)), dict(q=t(2, 512)), dict(q=t(2, 6, 64)),
              dict(k=t(4, 16, 4, 128), v=t(4, 16, 4, 128)), dict(v=t(4, 16, 2, 64)),
              dict(k=t(4, 4, 16, 64).transpose(1, 2)), dict(v=t(4, 16, 4, 64, dtype=F16)),
              dict(q=t(2, 8, 64, dtype=F16), k=t(4, 16, 4, 64, dtype=FP8),
                   v=t(4, 16, 4, 64, dtype=FP8), w=t(128, dtype=F16)),
              dict(l=t(4, 64)), dict(l=t(4, 128, dtype=torch.float32)),
              dict(l=t(64, 4, dtype=torch.float32).t()), dict(w=t(64)), dict(w=t(128, dtype=F16)),
              dict(w=t(256)[::2]), dict(out=t(2, 8, 64)), dict(out=t(2, 4, 128, dtype=F16)),
              dict(out=t(2, 4, 256)[..., ::2]), dict(bt=t(1, 3, dtype=I32)),
              dict(bt=t(2, 3, dtype=torch.int64)), dict(bt=t(3, 2, dtype=I32).t()),
              dict(ws=t(100, dtype=torch.float32)), dict(l=t(4, 64, dtype=torch.float32,
                                                             device="cpu"))]
    for call, more in ((decode, [dict(lens=t(1, dtype=I32)), dict(lens=t(2, dtype=torch.int64))]),
                       (prefill, [dict(cu=t(2, dtype=I32)), dict(ck=t(2, dtype=I32)),
                                  dict(cu=t(0, dtype=I32), ck=t(0, dtype=I32)),
                                  dict(cu=t(3, dtype=torch.int64))])):
        for kw in shared + more:
            with pytest.raises(ValueError):
                call(**kw)
        assert bool((call() == 0).all())
    with pytest.raises(importlib.import_module("nanokv-llm_amd._lib").NkvError):
        decode(ws=t(16, dtype=torch.uint8))  # too small


def test_paged_sequences_of_a_pool_with_odd_rows(dev):
    with pytest.raises(importlib.import_module("nanokv-llm_amd._lib").NkvError, match="16 bytes"):
        nkv.PagedSequences(torch.zeros(2, 1, 8, 16, 1, 4, dtype=BF, device=dev), 4, 5).compact()
