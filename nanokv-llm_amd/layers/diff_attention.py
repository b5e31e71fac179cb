"""Differential attention over the paged K/V cache: the difference of two softmax maps.

Heads stand in pairs. Query pair h (heads 2h and 2h+1 of q) reads KV pair p = h // G: K heads 2p and
2p+1, and one value of 2 D numbers, V heads 2p and 2p+1 side by side.

    A_m    = softmax(scale * q_{2h+m} . K_{2p+m}) [V_2p | V_2p+1]        m = 0, 1
    lambda = exp(l[0] . l[1]) - exp(l[2] . l[3]) + lambda_init
    o      = A_0 - lambda * A_1
    out_h  = (1 - lambda_init) * o / sqrt(mean(o^2) + eps) * norm_weight

The cache is the one that ``Attention`` uses ([blocks, block_size, Hk, D], Hk the two heads of every
pair), so ``store_kvcache``, ``qk_norm_rope_store``, ``KVCachePool`` and ``PagedSequences`` serve it
as they are. No counterpart in the reference; the layer stands beside its ``Attention``
(nanokvllm/layers/attention.py:42-108).
"""
from __future__ import annotations

import math

import torch
from torch import nn

from .. import _lib
from ..utils.context import get_context
from .attention import shared_decode_workspace, store_kvcache

_FP8 = torch.float8_e4m3fn
_I32 = torch.int32
MAX_GROUP = 64  # include/nkv.h, NKV_DIFF_MAX_GROUP


def lambda_init_of(layer: int) -> float:
    """The usual lambda_init of layer ``layer`` (from 0): 0.8 - 0.6 exp(-0.3 layer)."""
    return 0.8 - 0.6 * math.exp(-0.3 * layer)


def _check(what, q, k, v, lambdas, norm_weight, out, paged, **others):
    """The checks that both operators share -> (rows, Hq, D, Hk, kv_type)."""
    _lib.require_device(q.device, k=k, v=v, lambdas=lambdas, norm_weight=norm_weight, out=out,
                        **others)
    _lib.need(q.dim() == 3 and q.stride(2) == 1 and q.stride(1) == q.size(2),
              f"{what}: q must be [rows, Hq, D], rows of contiguous heads")
    N, Hq, D = q.shape
    f16 = _lib.is_f16(q, f"{what}: q")
    fp8 = paged and k.dtype == _FP8
    _lib.need(k.dim() == (4 if paged else 3) and k.size(-1) == D and v.shape == k.shape
              and v.dtype == k.dtype, f"{what}: k and v must share a shape and a dtype, with q's "
              "head_dim")
    _lib.need(k.dtype == q.dtype or (fp8 and not f16),
              f"{what}: caches must have q's dtype (or fp8 with bf16 q)")
    Hk = k.size(-2)
    if paged:
        _lib.need(k.is_contiguous() and v.is_contiguous(), f"{what}: caches must be contiguous")
    else:
        _lib.need(all(t.stride(1) == D and t.stride(2) == 1 for t in (k, v)),
                  f"{what}: k and v must be rows of contiguous heads")
    _lib.need(Hq > 0 and Hk > 0 and Hq % 2 == 0 and Hk % 2 == 0 and Hq % Hk == 0,
              f"{what}: heads stand in pairs, whole groups of query pairs to a KV pair (got "
              f"Hq={Hq}, Hk={Hk})")
    _lib.need(lambdas.shape == (4, D) and lambdas.dtype == torch.float32
              and lambdas.is_contiguous(), f"{what}: lambdas must be contiguous float32 [4, {D}]")
    _lib.need(norm_weight is None or (norm_weight.shape == (2 * D,) and norm_weight.dtype == q.dtype
                                      and norm_weight.is_contiguous()),
              f"{what}: norm_weight must be contiguous [{2 * D}] in q's dtype")
    _lib.need(out is None or (out.shape == (N, Hq // 2, 2 * D) and out.dtype == q.dtype
                              and out.stride(2) == 1 and out.stride(1) == 2 * D),
              f"{what}: out must be [rows, Hq/2, 2 D] in q's dtype, rows of contiguous heads")
    return N, Hq, D, Hk, (_lib.NKV_KV_FP8 if fp8 else _lib.NKV_KV_F16 if f16 else
                          _lib.NKV_KV_BF16)


def _int32_rows(what, name, t, dims=1):
    _lib.need(t.dtype is _I32 and t.dim() == dims and
              (t.is_contiguous() if dims == 1 else t.stride(1) == 1),
              f"{what}: {name} must be int32, {'contiguous' if dims == 1 else 'contiguous rows'}")


def diff_decode_workspace_bytes(bs: int, n_q_heads: int, max_blocks_per_seq: int, block_size: int,
                                head_dim: int) -> int:
    """Bytes that diff_paged_decode needs (0 for a head_dim that it does not take)."""
    return int(_lib.lib().nkv_diff_decode_workspace_bytes(bs, n_q_heads, head_dim,
                                                          max_blocks_per_seq, block_size))


def diff_paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      context_lens: torch.Tensor, block_tables: torch.Tensor, scale: float,
                      lambdas: torch.Tensor, lambda_init: float,
                      norm_weight: torch.Tensor | None = None, eps: float = 1e-5,
                      out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                      k_scale: float = 1.0, v_scale: float = 1.0) -> torch.Tensor:
    """Differential attention of one new token per sequence: q [bs, Hq, D] -> [bs, Hq/2, 2 D] (q's
    dtype: bf16 or fp16) over caches [NB, B, Hk, D] (q's dtype, or fp8 with bf16 q).

    ``lambdas``: float32 [4, D]; ``norm_weight``: [2 D] in q's dtype, or None for ones. The other
    arguments are ``paged_decode``'s; a sequence of length 0 gives zeros.
    """
    what = "diff_paged_decode"
    bs, Hq, D, Hk, kv_type = _check(what, q, k_cache, v_cache, lambdas, norm_weight, out, True,
                                    block_tables=block_tables, context_lens=context_lens,
                                    workspace=workspace)
    _int32_rows(what, "block_tables", block_tables, 2)
    _int32_rows(what, "context_lens", context_lens)
    _lib.need(block_tables.size(0) >= bs and context_lens.numel() >= bs,
              f"{what}: block_tables and context_lens need a row for each of q's {bs}")
    NB, B, width = k_cache.size(0), k_cache.size(1), block_tables.size(1)
    if out is None:
        out = torch.empty(bs, Hq // 2, 2 * D, dtype=q.dtype, device=q.device)
    if workspace is None:
        workspace = torch.empty(max(diff_decode_workspace_bytes(bs, Hq, width, B, D), 4),
                                dtype=torch.uint8, device=q.device)
    _lib.need(workspace.dtype == torch.uint8 and workspace.is_contiguous(),
              f"{what}: workspace must be contiguous uint8")
    with _lib.device_of(q.get_device()):
        rc = _lib.lib().nkv_diff_decode(
            kv_type, q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(),
            block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), bs, Hq, Hk,
            D, B, width, NB, scale, k_scale, v_scale, lambdas.data_ptr(), lambda_init,
            _lib.ptr(norm_weight), eps, out.data_ptr(), out.stride(0), workspace.data_ptr(),
            workspace.numel(), _lib.stream_of(q))
    if rc:
        _lib.check(rc, what)
    return out
