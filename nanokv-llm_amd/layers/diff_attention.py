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
    """The checks that both operators share -> (rows, Hq, D, Hk, kv_type). One pass over the
    arguments where they are right (messages are made only for the others: building them all took
    as long as a launch)."""
    _lib.require_device(q.device, k=k, v=v, lambdas=lambdas, norm_weight=norm_weight, out=out,
                        **others)
    qs, ks, dt, ct = q.shape, k.shape, q.dtype, k.dtype
    if len(qs) != 3 or q.stride(2) != 1 or q.stride(1) != qs[2]:
        raise ValueError(f"{what}: q must be [rows, Hq, D], rows of contiguous heads")
    N, Hq, D = qs
    f16 = _lib.is_f16(q, what)
    fp8 = paged and ct is _FP8
    if len(ks) != (4 if paged else 3) or ks[-1] != D or v.shape != ks or v.dtype is not ct:
        raise ValueError(f"{what}: k and v must share a shape and a dtype, with q's head_dim")
    if ct is not dt and (not fp8 or f16):
        raise ValueError(f"{what}: caches must have q's dtype (or fp8 with bf16 q)")
    Hk = ks[-2]
    if paged:
        if not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError(f"{what}: caches must be contiguous")
    elif not all(t.stride(1) == D and t.stride(2) == 1 for t in (k, v)):
        raise ValueError(f"{what}: k and v must be rows of contiguous heads")
    if Hq <= 0 or Hk <= 0 or Hq % 2 or Hk % 2 or Hq % Hk:
        raise ValueError(f"{what}: heads stand in pairs, whole groups of query pairs to a KV pair "
                         f"(got Hq={Hq}, Hk={Hk})")
    if lambdas.shape != (4, D) or lambdas.dtype is not torch.float32 \
            or not lambdas.is_contiguous():
        raise ValueError(f"{what}: lambdas must be contiguous float32 [4, {D}]")
    if norm_weight is not None and (norm_weight.shape != (2 * D,) or norm_weight.dtype is not dt
                                    or not norm_weight.is_contiguous()):
        raise ValueError(f"{what}: norm_weight must be contiguous [{2 * D}] in q's dtype")
    if out is not None and (out.shape != (N, Hq // 2, 2 * D) or out.dtype is not dt
                            or out.stride(2) != 1 or out.stride(1) != 2 * D):
        raise ValueError(f"{what}: out must be [rows, Hq/2, 2 D] in q's dtype, rows of contiguous "
                         "heads")
    return N, Hq, D, Hk, (_lib.NKV_KV_FP8 if fp8 else _lib.NKV_KV_F16 if f16 else
                          _lib.NKV_KV_BF16)


def _int32_rows(what, name, t, dims=1):
    if t.dtype is not _I32 or t.dim() != dims or not (t.is_contiguous() if dims == 1
                                                      else t.stride(1) == 1):
        raise ValueError(f"{what}: {name} must be int32, "
                         f"{'contiguous' if dims == 1 else 'contiguous rows'}")


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
    if block_tables.size(0) < bs or context_lens.numel() < bs:
        raise ValueError(f"{what}: block_tables and context_lens need a row for each of q's {bs}")
    NB, B, width = k_cache.size(0), k_cache.size(1), block_tables.size(1)
    if out is None:
        out = torch.empty(bs, Hq // 2, 2 * D, dtype=q.dtype, device=q.device)
    if workspace is not None and (workspace.dtype is not torch.uint8
                                  or not workspace.is_contiguous()):
        raise ValueError(f"{what}: workspace must be contiguous uint8")
    with _lib.device_of(q.get_device()):
        if workspace is None:
            workspace = torch.empty(max(diff_decode_workspace_bytes(bs, Hq, width, B, D), 4),
                                    dtype=torch.uint8, device=q.device)
        rc = _lib.lib().nkv_diff_decode(
            kv_type, q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(),
            block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), bs, Hq, Hk,
            D, B, width, NB, scale, k_scale, v_scale, lambdas.data_ptr(), lambda_init,
            _lib.ptr(norm_weight), eps, out.data_ptr(), out.stride(0), workspace.data_ptr(),
            workspace.numel(), _lib.stream_of(q))
    if rc:
        _lib.check(rc, what)
    return out


def diff_prefill_workspace(q: torch.Tensor, k: torch.Tensor, n_seqs: int, max_seqlen_q: int,
                           max_seqlen_k: int) -> torch.Tensor | None:
    """The workspace for splitting diff_varlen_prefill's keys where that is of use (few query tiles
    over long contexts) and for streaming the sequences that bring one token, else None. Sized by
    the chip and the tiles, not by the lengths; None too where the device has no such memory
    left, since nothing else needs any."""
    kv_type = _lib.NKV_KV_FP8 if k.dtype == _FP8 else _lib.NKV_KV_BF16
    nbytes = _lib.lib().nkv_diff_prefill_workspace_bytes(
        kv_type, n_seqs, q.size(0), int(max_seqlen_q), int(max_seqlen_k), q.size(1), k.size(-2),
        q.size(2), 1 if k.dim() == 4 else 0)
    try:
        return torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    except torch.OutOfMemoryError:
        return None


def diff_varlen_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor,
                        max_seqlen_q: int, scale: float, lambdas: torch.Tensor,
                        lambda_init: float, norm_weight: torch.Tensor | None = None,
                        eps: float = 1e-5, block_tables: torch.Tensor | None = None,
                        out: torch.Tensor | None = None, max_seqlen_k: int | None = None,
                        k_scale: float = 1.0, v_scale: float = 1.0,
                        workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Varlen causal (bottom-right) differential attention: q [sum Lq, Hq, D] -> [sum Lq, Hq/2,
    2 D].

    With ``block_tables`` k and v are the paged caches [NB, B, Hk, D] (q's dtype, or fp8 with bf16
    q); without, they are [sum Lk, Hk, D] rows, each with its own row stride. ``lambdas`` and
    ``norm_weight`` are ``diff_paged_decode``'s, the rest ``varlen_prefill``'s. Given
    ``max_seqlen_k``, the keys are split over the chip where few tiles would leave it idle and
    sequences that bring one token are streamed apart from the tiles, in ``workspace``
    (diff_prefill_workspace) or in memory taken for the call; without, nothing but the output is
    allocated. A row that sees no key gives zeros.
    """
    what = "diff_varlen_prefill"
    paged = block_tables is not None
    N, Hq, D, Hk, kv_type = _check(what, q, k, v, lambdas, norm_weight, out, paged,
                                   cu_seqlens_q=cu_seqlens_q, cu_seqlens_k=cu_seqlens_k,
                                   block_tables=block_tables, workspace=workspace)
    _int32_rows(what, "cu_seqlens_q", cu_seqlens_q)
    _int32_rows(what, "cu_seqlens_k", cu_seqlens_k)
    n_seqs = cu_seqlens_q.numel() - 1
    if n_seqs < 0 or cu_seqlens_k.numel() != n_seqs + 1:
        raise ValueError(f"{what}: cu_seqlens_q and cu_seqlens_k need one entry per sequence + 1")
    if paged:
        _int32_rows(what, "block_tables", block_tables, 2)
        if block_tables.size(0) < n_seqs:
            raise ValueError(f"{what}: block_tables needs a row for each of the {n_seqs} sequences")
        B, rows = k.size(1), k.size(0) * k.size(1)
        k_stride = v_stride = Hk * D
        bt, bt_stride, width = (block_tables.data_ptr(), block_tables.stride(0),
                                block_tables.size(1))
    else:
        B, rows, k_stride, v_stride = 0, k.size(0), k.stride(0), v.stride(0)
        bt, bt_stride, width = None, 0, 0
    if out is None:
        out = torch.empty(N, Hq // 2, 2 * D, dtype=q.dtype, device=q.device)
    if workspace is not None and (workspace.dtype is not torch.uint8
                                  or not workspace.is_contiguous()):
        raise ValueError(f"{what}: workspace must be contiguous uint8")
    with _lib.device_of(q.get_device()):
        if workspace is None and max_seqlen_k is not None:
            workspace = diff_prefill_workspace(q, k, n_seqs, max_seqlen_q, max_seqlen_k)
        rc = _lib.lib().nkv_diff_prefill(
            kv_type, q.data_ptr(), q.stride(0), N, k.data_ptr(), v.data_ptr(), k_stride, v_stride,
            cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), bt, bt_stride, width, n_seqs,
            int(max_seqlen_q), 0 if max_seqlen_k is None else int(max_seqlen_k), Hq, Hk, D, B,
            rows, scale, k_scale, v_scale, lambdas.data_ptr(), lambda_init,
            _lib.ptr(norm_weight), eps, out.data_ptr(), out.stride(0), _lib.ptr(workspace),
            0 if workspace is None else workspace.numel(), _lib.stream_of(q))
    if rc:
        _lib.check(rc, what)
    return out


class DifferentialAttention(nn.Module):
    """One layer's differential attention: store, then prefill or decode, by the context that
    ``Attention`` goes by (same ``k_cache``/``v_cache`` attributes, assigned by
    ``KVCachePool.bind`` or the model runner).

    ``num_heads`` and ``num_kv_heads`` count q's and the cache's heads (both even, two to a pair).
    ``lambdas`` (float32 [4, head_dim]) and ``norm_weight`` ([2 head_dim], the model's dtype)
    are parameters to load; gradients are not computed. There is no compression of such a cache.
    """

    def __init__(self, num_heads: int, head_dim: int, scale: float, num_kv_heads: int,
                 lambda_init: float, norm_eps: float = 1e-5):
        super().__init__()
        _lib.need(head_dim in (64, 128),
                  f"DifferentialAttention: head_dim {head_dim} is not 64 or 128")
        _lib.need(num_heads > 0 and num_kv_heads > 0 and num_heads % 2 == 0
                  and num_kv_heads % 2 == 0 and num_heads % num_kv_heads == 0
                  and num_heads // num_kv_heads <= MAX_GROUP,
                  f"DifferentialAttention: {num_heads} query and {num_kv_heads} KV heads are not "
                  f"pairs with 1 to {MAX_GROUP} query pairs to a KV pair")
        _lib.need(scale > 0 and norm_eps > 0,
                  "DifferentialAttention: scale and norm_eps must be > 0")
        self.num_heads, self.head_dim, self.num_kv_heads = num_heads, head_dim, num_kv_heads
        self.scale, self.lambda_init, self.norm_eps = scale, lambda_init, norm_eps
        self.lambdas = nn.Parameter(torch.zeros(4, head_dim, dtype=torch.float32),
                                    requires_grad=False)
        self.norm_weight = nn.Parameter(torch.ones(2 * head_dim), requires_grad=False)
        self.k_cache = self.v_cache = torch.tensor([])
        self.k_scale = self.v_scale = 1.0
        self._cache_checked = None  # (k_cache data_ptr, shape) whose geometry was checked

    def _check_cache(self):
        """The bound cache's geometry, once per binding."""
        kc = self.k_cache
        key = (kc.data_ptr(), tuple(kc.shape))
        if self._cache_checked == key:
            return
        _lib.need(kc.dim() == 4 and kc.size(2) == self.num_kv_heads and
                  kc.size(3) == self.head_dim,
                  f"DifferentialAttention: k_cache must be [blocks, block_size, "
                  f"{self.num_kv_heads}, {self.head_dim}], got {tuple(kc.shape)}")
        _lib.need(kc.size(1) % 16 == 0,
                  f"DifferentialAttention: block_size {kc.size(1)} is not a multiple of 16")
        self._cache_checked = key

    def forward(self, q: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None, Layer=None,
                kv_stored: bool = False):
        """q [N, Hq, D], k and v [N, Hk, D] -> [N, Hq/2, 2 D] (decode: [N, 1, Hq/2, 2 D], as
        ``Attention``). ``kv_stored=True``: k and v are in the cache already."""
        ctx = get_context()
        _lib.need(not ctx.is_compress_step, "DifferentialAttention: its cache takes no part in "
                  "compression steps")
        if q.dim() != 3 or q.size(1) != self.num_heads or q.size(2) != self.head_dim:
            raise ValueError(f"DifferentialAttention: q must be [rows, {self.num_heads}, "
                             f"{self.head_dim}], got {tuple(q.shape)}")
        kc, vc = self.k_cache, self.v_cache
        paged = ctx.use_decode_kernel or ctx.block_tables is not None
        if kc.numel():
            self._check_cache()
        elif paged:
            raise ValueError("DifferentialAttention: no cache is bound")
        if not paged and (k.dim() != 3 or k.size(1) != self.num_kv_heads
                          or k.size(2) != self.head_dim):
            raise ValueError(f"DifferentialAttention: k and v must be [rows, {self.num_kv_heads}, "
                             f"{self.head_dim}], got {tuple(k.shape)}")
        with _lib.device_of(q.get_device()):
            return self._step(q, k, v, ctx, kv_stored)

    def _step(self, q, k, v, ctx, kv_stored):
        kc, vc = self.k_cache, self.v_cache
        if kc.numel() and not kv_stored:
            store_kvcache(k, v, kc, vc, ctx.slot_mapping, self.k_scale, self.v_scale)
        weights = (self.lambdas, self.lambda_init, self.norm_weight, self.norm_eps)
        if ctx.use_decode_kernel:
            bt = ctx.block_tables
            workspace = shared_decode_workspace(q.device, diff_decode_workspace_bytes(
                q.size(0), q.size(1), bt.size(1), kc.size(1), q.size(2)))
            return diff_paged_decode(q, kc, vc, ctx.context_lens, bt, self.scale, *weights,
                                     workspace=workspace, k_scale=self.k_scale,
                                     v_scale=self.v_scale).unsqueeze(1)
        if ctx.block_tables is not None:
            k, v = kc, vc
        return diff_varlen_prefill(q, k, v, ctx.cu_seqlens_q, ctx.cu_seqlens_k, ctx.max_seqlen_q,
                                   self.scale, *weights, block_tables=ctx.block_tables,
                                   max_seqlen_k=ctx.max_seqlen_k, k_scale=self.k_scale,
                                   v_scale=self.v_scale)
