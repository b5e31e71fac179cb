"""The block-scaled K/V cache: 8-bit codes with a scale for every 32 tokens and head.

The fp8 pool of ``kv_cache`` has one scale per layer, which has to be calibrated. Here a tile of 32 rows
of one head has a scale of its own, a power of two that follows from what is stored: nothing to
calibrate, and heads and tokens of any magnitude keep E4M3's full precision, for 16 bytes a token
(kept beside the codes, so that whoever copies a page copies its scales).

    e     the smallest in [-100, 119] with max |x| <= 448 * 2^e over the tile's rows
    code  E4M3(x * 2^-e), read as code * 2^e

A cache is uint8 ``[blocks, block_size, Hk * D + 16]``, its tiles laid out as include/nkv.h says. q, k,
v and outputs are bf16, head_dim is 64 or 128. No counterpart in the reference; it stands beside the
pool of nanokvllm/engine/model_runner.py:133-152 and the calls of layers/attention.py:33-40, 96-107.
"""
from __future__ import annotations

import torch

from .. import _lib
from .kv_cache import blocks_that_fit

_BF16, _I32, _U8 = torch.bfloat16, torch.int32, torch.uint8
TILE = 32      # tokens under one scale
ROW_PAD = 16   # include/nkv.h, NKV_SCALED_ROW_PAD
MAX_HEADS = 512


class ScaledKVCachePool:
    """One uint8 tensor of block-scaled K/V for every layer: ``kv_cache`` [2, layers, blocks,
    block_size, Hk * D + 16], zeros (nothing written), sized from the free device memory as
    ``KVCachePool`` is. ``PagedSequences`` takes it as it takes a ``KVCachePool``."""

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, block_size: int = 256,
                 gpu_memory_utilization: float = 0.8, num_blocks: int | None = None,
                 device="cuda"):
        if head_dim not in (64, 128) or not 0 < num_kv_heads <= MAX_HEADS or num_layers <= 0:
            raise ValueError(f"ScaledKVCachePool: {num_layers} layers of {num_kv_heads} KV heads of "
                             f"{head_dim} (head_dim 64 or 128, 1 to {MAX_HEADS} heads)")
        if block_size <= 0 or block_size % TILE:
            raise ValueError(f"ScaledKVCachePool: block_size {block_size} is not a multiple of {TILE}")
        row = num_kv_heads * head_dim + ROW_PAD
        self.block_size, self.dtype = block_size, _U8
        self.block_bytes = 2 * num_layers * block_size * row
        if num_blocks is None:
            num_blocks = blocks_that_fit(self.block_bytes, gpu_memory_utilization, device)
        if num_blocks <= 0:
            raise RuntimeError("no device memory left for the K/V pool")
        self.num_blocks = num_blocks
        self.kv_cache = torch.zeros(2, num_layers, num_blocks, block_size, row, dtype=_U8,
                                    device=device)

    def bind(self, modules) -> int:
        """Assign layer i's views to the i-th module with k_cache/v_cache (model_runner.py
        :148-152); returns the number of layers bound."""
        layer = 0
        for m in modules:
            if hasattr(m, "k_cache") and hasattr(m, "v_cache"):
                m.k_cache, m.v_cache = self.kv_cache[0, layer], self.kv_cache[1, layer]
                layer += 1
        return layer


def _caches(what, k_cache, v_cache, row):
    """Blocks and block size of caches whose rows hold ``row`` codes."""
    if not (k_cache.dtype is _U8 and v_cache.dtype is _U8 and k_cache.dim() == 3
            and v_cache.shape == k_cache.shape and k_cache.size(2) == row + ROW_PAD
            and k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"{what}: caches must be contiguous uint8 [blocks, block_size, "
                         f"{row + ROW_PAD}], got {k_cache.dtype} {tuple(k_cache.shape)} and "
                         f"{v_cache.dtype} {tuple(v_cache.shape)}")
    if k_cache.size(1) % TILE or k_cache.size(1) == 0:
        raise ValueError(f"{what}: block_size {k_cache.size(1)} is not a multiple of {TILE}")
    return k_cache.size(0), k_cache.size(1)


def _kv_heads(what, k_cache, D):
    """The KV heads of a cache of head_dim D."""
    row = k_cache.size(-1) - ROW_PAD
    if row <= 0 or row % D:
        raise ValueError(f"{what}: the cache's rows of {row} codes are not heads of {D}")
    return row // D


def _rows(what, name, t, dtype=_BF16):
    if t.dim() != 3 or t.dtype is not dtype or t.stride(2) != 1 or t.stride(1) != t.size(2):
        raise ValueError(f"{what}: {name} must be bf16 [rows, heads, head_dim], rows of contiguous "
                         f"heads, got {t.dtype} {tuple(t.shape)}")


def _int32(what, name, t, n, dims=1):
    """``n``: entries (or rows) needed at least."""
    ok = t.dtype is _I32 and t.dim() == dims and t.size(0) >= n
    if not ok or not (t.is_contiguous() if dims == 1 else t.stride(1) == 1 and t.size(1) > 0):
        raise ValueError(f"{what}: {name} must be int32 with at least {n} "
                         f"{'contiguous entries' if dims == 1 else 'contiguous rows'}, got {t.dtype} "
                         f"{tuple(t.shape)}")


def scaled_store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                         v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Rows key[i] and value[i] ([N, Hk, D]) into row slot_mapping[i]; -1 slots are skipped.

    A call that writes a tile's first row begins the tile anew, with the scale of the rows that it
    writes there; otherwise the scale only grows, and the rows held so far are rounded to it where it
    does. The tokens of one tile must stand next to each other in ``slot_mapping``, as those of a
    sequence do.
    """
    what = "scaled_store_kvcache"
    _lib.require_device(key.device, value=value, k_cache=k_cache, v_cache=v_cache,
                        slot_mapping=slot_mapping)
    _rows(what, "key", key)
    _rows(what, "value", value)
    N, Hk, D = key.shape
    if value.shape != key.shape:
        raise ValueError(f"{what}: value shape differs from key")
    NB, B = _caches(what, k_cache, v_cache, Hk * D)
    _int32(what, "slot_mapping", slot_mapping, N)
    if slot_mapping.numel() != N:
        raise ValueError(f"{what}: {slot_mapping.numel()} slots for {N} rows")
    with _lib.device_of(key.get_device()):
        rc = _lib.lib().nkv_scaled_store(key.data_ptr(), key.stride(0), value.data_ptr(),
                                         value.stride(0), k_cache.data_ptr(), v_cache.data_ptr(),
                                         slot_mapping.data_ptr(), N, Hk, D, NB * B,
                                         _lib.stream_of(key))
    if rc:
        _lib.check(rc, what)


def scaled_read_kvcache(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                        cu_seqlens: torch.Tensor, n_tokens: int, num_kv_heads: int,
                        starts: torch.Tensor | None = None,
                        out: tuple[torch.Tensor, torch.Tensor] | None = None
                        ) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of sequences as bf16 rows, exactly what the codes stand for.

    Sequence i's positions ``starts[i]`` .. (or 0 ..) become rows cu_seqlens[i] .. cu_seqlens[i+1] - 1
    of the outputs [n_tokens, Hk, D] (``out``, or new ones; rows of no sequence are left as they
    are). Positions that its table has no valid block for read as zeros.
    """
    what = "scaled_read_kvcache"
    _lib.require_device(k_cache.device, v_cache=v_cache, block_tables=block_tables,
                        cu_seqlens=cu_seqlens, starts=starts)
    Hk, row = num_kv_heads, k_cache.size(-1) - ROW_PAD
    if Hk <= 0 or row <= 0 or row % Hk:
        raise ValueError(f"{what}: the cache's rows of {row} codes are not {Hk} heads")
    D = row // Hk
    NB, B = _caches(what, k_cache, v_cache, row)
    n_seqs = cu_seqlens.numel() - 1
    if n_seqs < 0 or n_tokens < 0:
        raise ValueError(f"{what}: cu_seqlens needs one entry per sequence + 1, n_tokens >= 0")
    _int32(what, "cu_seqlens", cu_seqlens, n_seqs + 1)
    _int32(what, "block_tables", block_tables, n_seqs, 2)
    if starts is not None:
        _int32(what, "starts", starts, n_seqs)
    shape = (n_tokens, Hk, D)
    if out is None:
        out = tuple(torch.empty(shape, dtype=_BF16, device=k_cache.device) for _ in range(2))
    k, v = out
    _lib.require_device(k_cache.device, k=k, v=v)
    for t in out:
        if t.shape != shape or t.dtype is not _BF16 or not t.is_contiguous():
            raise ValueError(f"{what}: out must be two contiguous bf16 {shape}")
    with _lib.device_of(k_cache.get_device()):
        rc = _lib.lib().nkv_scaled_read(
            k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), block_tables.stride(0),
            block_tables.size(1), cu_seqlens.data_ptr(), _lib.ptr(starts), n_seqs, n_tokens, Hk, D,
            B, NB, k.data_ptr(), v.data_ptr(), _lib.stream_of(k_cache))
    if rc:
        _lib.check(rc, what)
    return out


def _out(what, q, out):
    if out is None:
        return q.new_empty(q.shape)
    if out.shape != q.shape or out.dtype is not _BF16 or out.stride(2) != 1 \
            or out.stride(1) != q.size(2):
        raise ValueError(f"{what}: out must be bf16 and shaped like q, rows of contiguous heads")
    return out


def _workspace_ok(what, workspace):
    if workspace is not None and (workspace.dtype is not _U8 or not workspace.is_contiguous()):
        raise ValueError(f"{what}: workspace must be contiguous uint8")


def scaled_paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        context_lens: torch.Tensor, block_tables: torch.Tensor, scale: float,
                        out: torch.Tensor | None = None, workspace: torch.Tensor | None = None
                        ) -> torch.Tensor:
    """Attention of one new token per sequence: q [bs, Hq, D] -> [bs, Hq, D] (bf16).

    The arguments are ``paged_decode``'s, the workspace's size ``decode_workspace_bytes``; a sequence
    of length 0 gives zeros.
    """
    what = "scaled_paged_decode"
    _lib.require_device(q.device, k_cache=k_cache, v_cache=v_cache, context_lens=context_lens,
                        block_tables=block_tables, out=out, workspace=workspace)
    _rows(what, "q", q)
    bs, Hq, D = q.shape
    Hk = _kv_heads(what, k_cache, D)
    NB, B = _caches(what, k_cache, v_cache, Hk * D)
    _int32(what, "context_lens", context_lens, bs)
    _int32(what, "block_tables", block_tables, bs, 2)
    _workspace_ok(what, workspace)
    out = _out(what, q, out)
    with _lib.device_of(q.get_device()):
        width = block_tables.size(1)
        if workspace is None:
            nbytes = _lib.lib().nkv_paged_decode_workspace_bytes(bs, Hq, D, width, B)
            workspace = torch.empty(max(nbytes, 4), dtype=_U8, device=q.device)
        rc = _lib.lib().nkv_scaled_decode(
            q.data_ptr(), q.stride(0), k_cache.data_ptr(), v_cache.data_ptr(),
            block_tables.data_ptr(), block_tables.stride(0), context_lens.data_ptr(), bs, Hq, Hk, D,
            B, width, NB, scale, out.data_ptr(), out.stride(0), workspace.data_ptr(),
            workspace.numel(), _lib.stream_of(q))
    if rc:
        _lib.check(rc, what)
    return out


def scaled_prefill_workspace(q: torch.Tensor, k_cache: torch.Tensor, n_seqs: int,
                             max_seqlen_q: int, max_seqlen_k: int) -> torch.Tensor | None:
    """The workspace for splitting scaled_varlen_prefill's keys where few query tiles would leave the
    chip idle, else None; None too where the device has no such memory left, since nothing else
    needs any."""
    D = q.size(2)
    nbytes = _lib.lib().nkv_scaled_prefill_workspace_bytes(
        n_seqs, q.size(0), int(max_seqlen_q), int(max_seqlen_k), q.size(1),
        _kv_heads("scaled_varlen_prefill", k_cache, D), D)
    try:
        return torch.empty(nbytes, dtype=_U8, device=q.device) if nbytes else None
    except torch.OutOfMemoryError:
        return None


def scaled_varlen_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                          cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor,
                          max_seqlen_q: int, scale: float, block_tables: torch.Tensor,
                          out: torch.Tensor | None = None, max_seqlen_k: int | None = None,
                          workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Varlen causal (bottom-right) attention: q [sum Lq, Hq, D] -> [sum Lq, Hq, D] (bf16).

    The arguments are ``varlen_prefill``'s with block tables. Given ``max_seqlen_k``, the keys are split
    over the chip where few tiles would leave it idle, in ``workspace`` (scaled_prefill_workspace) or
    in memory taken for the call; without, nothing but the output is allocated. A row that sees no
    key gives zeros; what keys hold that a row does not see has no effect on it.
    """
    what = "scaled_varlen_prefill"
    _lib.require_device(q.device, k_cache=k_cache, v_cache=v_cache, cu_seqlens_q=cu_seqlens_q,
                        cu_seqlens_k=cu_seqlens_k, block_tables=block_tables, out=out,
                        workspace=workspace)
    _rows(what, "q", q)
    N, Hq, D = q.shape
    Hk = _kv_heads(what, k_cache, D)
    NB, B = _caches(what, k_cache, v_cache, Hk * D)
    n_seqs = cu_seqlens_q.numel() - 1
    if n_seqs < 0 or cu_seqlens_k.numel() != n_seqs + 1:
        raise ValueError(f"{what}: cu_seqlens_q and cu_seqlens_k need one entry per sequence + 1")
    _int32(what, "cu_seqlens_q", cu_seqlens_q, n_seqs + 1)
    _int32(what, "cu_seqlens_k", cu_seqlens_k, n_seqs + 1)
    _int32(what, "block_tables", block_tables, n_seqs, 2)
    _workspace_ok(what, workspace)
    out = _out(what, q, out)
    with _lib.device_of(q.get_device()):
        if workspace is None and max_seqlen_k is not None:
            workspace = scaled_prefill_workspace(q, k_cache, n_seqs, max_seqlen_q, max_seqlen_k)
        rc = _lib.lib().nkv_scaled_prefill(
            q.data_ptr(), q.stride(0), N, k_cache.data_ptr(), v_cache.data_ptr(),
            cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), block_tables.data_ptr(),
            block_tables.stride(0), block_tables.size(1), n_seqs, int(max_seqlen_q),
            0 if max_seqlen_k is None else int(max_seqlen_k), Hq, Hk, D, B, NB, scale,
            out.data_ptr(), out.stride(0), _lib.ptr(workspace),
            0 if workspace is None else workspace.numel(), _lib.stream_of(q))
    if rc:
        _lib.check(rc, what)
    return out
