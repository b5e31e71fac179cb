"""The block-scaled K/V cache: 8-bit codes with a scale for every 32 tokens and head.

The fp8 pool of ``kv_cache`` has one scale per layer, which has to be calibrated. Here a tile of 32 rows
of one head has a scale of its own, a power of two that follows from what is stored: nothing to
calibrate, for 16 bytes a token (kept beside the codes, so that whoever copies a page copies its
scales). Values down to 2^-13 of the largest that the tile's 32 tokens hold of the head keep E4M3's four
significant bits, whatever its magnitude; smaller ones keep fewer, and those below 2^-19 become zero.

    e     the smallest in [-100, 119] with max |x| <= 448 * 2^e over the tile's rows
    code  E4M3(x * 2^-e), read as code * 2^e

A cache is uint8 ``[blocks, block_size, Hk * D + 16]``, its tiles laid out as include/nkv.h says. q, k,
v and outputs are bf16, head_dim is 64 or 128. No counterpart in the reference; it stands beside the
pool of nanokvllm/engine/model_runner.py:133-152 and the calls of layers/attention.py:33-40, 96-107.
"""
from __future__ import annotations

import functools
import struct

import torch

from .. import _lib
from .kv_cache import blocks_that_fit

_BF16, _I32, _U8 = torch.bfloat16, torch.int32, torch.uint8
TILE = 32      # tokens under one scale
ROW_PAD = 16   # include/nkv.h, NKV_SCALED_ROW_PAD
MAX_HEADS = 512
_STORE_ARGS, _READ_ARGS = struct.Struct("12q"), struct.Struct("16q")  # include/nkv.h
_DECODE_ARGS, _PREFILL_ARGS = struct.Struct("19qd"), struct.Struct("23qd")


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


# ---------------------------------------------------------------- checks
# Each operator passes its arguments by one expression where they are right, outputs and workspaces that
# it is given among them; only for others does its _refuse_* function look for what is wrong (with
# messages made and checks by name, they kept the host busy for 8 to 20 us a call, longer than a small
# call runs).
def _caches(what, k_cache, v_cache, row):
    if not (k_cache.dtype is _U8 and v_cache.dtype is _U8 and k_cache.dim() == 3
            and v_cache.shape == k_cache.shape and k_cache.size(2) == row + ROW_PAD
            and k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"{what}: caches must be contiguous uint8 [blocks, block_size, "
                         f"{row + ROW_PAD}], got {k_cache.dtype} {tuple(k_cache.shape)} and "
                         f"{v_cache.dtype} {tuple(v_cache.shape)}")
    if k_cache.size(1) % TILE or k_cache.size(1) == 0:
        raise ValueError(f"{what}: block_size {k_cache.size(1)} is not a multiple of {TILE}")


def _heads_of(what, k_cache, D):
    row = k_cache.size(-1) - ROW_PAD
    if row <= 0 or D <= 0 or row % D:
        raise ValueError(f"{what}: the cache's rows of {row} codes are not heads of {D}")
    return row


def _rows(what, name, t):
    if t.dim() != 3 or t.dtype is not _BF16 or t.stride(2) != 1 or t.stride(1) != t.size(2):
        raise ValueError(f"{what}: {name} must be bf16 [rows, heads, head_dim], rows of contiguous "
                         f"heads, got {t.dtype} {tuple(t.shape)}")


def _int32(what, name, t, n, dims=1):
    """``n``: entries (or rows) needed at least."""
    ok = t.dtype is _I32 and t.dim() == dims and t.size(0) >= n
    if not ok or not (t.is_contiguous() if dims == 1 else t.stride(1) == 1 and t.size(1) > 0):
        raise ValueError(f"{what}: {name} must be int32 with at least {n} "
                         f"{'contiguous entries' if dims == 1 else 'contiguous rows'}, got {t.dtype} "
                         f"{tuple(t.shape)}")


def _out_rows(what, q, out):
    if out is not None and (out.shape != q.shape or out.dtype is not _BF16 or out.stride(2) != 1
                            or out.stride(1) != q.size(2)):
        raise ValueError(f"{what}: out must be bf16 and shaped like q, rows of contiguous heads")


def _workspace_ok(what, workspace):
    if workspace is not None and (workspace.dtype is not _U8 or not workspace.is_contiguous()):
        raise ValueError(f"{what}: workspace must be contiguous uint8")


def _refuse_store(what, key, value, k_cache, v_cache, slot_mapping):
    _lib.require_device(key.device, value=value, k_cache=k_cache, v_cache=v_cache,
                        slot_mapping=slot_mapping)
    _rows(what, "key", key)
    _rows(what, "value", value)
    N, Hk, D = key.shape
    if value.shape != key.shape:
        raise ValueError(f"{what}: value shape differs from key")
    _caches(what, k_cache, v_cache, Hk * D)
    _int32(what, "slot_mapping", slot_mapping, N)
    if slot_mapping.numel() != N:
        raise ValueError(f"{what}: {slot_mapping.numel()} slots for {N} rows")


def _refuse_read(what, k_cache, v_cache, block_tables, cu_seqlens, n_tokens, Hk, starts, out):
    _lib.require_device(k_cache.device, v_cache=v_cache, block_tables=block_tables,
                        cu_seqlens=cu_seqlens, starts=starts)
    row = k_cache.size(-1) - ROW_PAD
    if Hk <= 0 or row <= 0 or row % Hk:
        raise ValueError(f"{what}: the cache's rows of {row} codes are not {Hk} heads")
    _caches(what, k_cache, v_cache, row)
    n_seqs = cu_seqlens.numel() - 1
    if n_seqs < 0 or n_tokens < 0:
        raise ValueError(f"{what}: cu_seqlens needs one entry per sequence + 1, n_tokens >= 0")
    _int32(what, "cu_seqlens", cu_seqlens, n_seqs + 1)
    _int32(what, "block_tables", block_tables, n_seqs, 2)
    if starts is not None:
        _int32(what, "starts", starts, n_seqs)
    if out is not None:
        k, v = out
        _lib.require_device(k_cache.device, k=k, v=v)
        shape = (n_tokens, Hk, row // Hk)
        for t in (k, v):
            if t.shape != shape or t.dtype is not _BF16 or not t.is_contiguous():
                raise ValueError(f"{what}: out must be two contiguous bf16 {shape}")


def _refuse_decode(what, q, k_cache, v_cache, context_lens, block_tables, out, workspace):
    _lib.require_device(q.device, k_cache=k_cache, v_cache=v_cache, context_lens=context_lens,
                        block_tables=block_tables, out=out, workspace=workspace)
    _rows(what, "q", q)
    _caches(what, k_cache, v_cache, _heads_of(what, k_cache, q.size(2)))
    _int32(what, "context_lens", context_lens, q.size(0))
    _int32(what, "block_tables", block_tables, q.size(0), 2)
    _workspace_ok(what, workspace)
    _out_rows(what, q, out)


def _refuse_prefill(what, q, k_cache, v_cache, cu_q, cu_k, block_tables, out, workspace):
    _lib.require_device(q.device, k_cache=k_cache, v_cache=v_cache, cu_seqlens_q=cu_q,
                        cu_seqlens_k=cu_k, block_tables=block_tables, out=out, workspace=workspace)
    _rows(what, "q", q)
    _caches(what, k_cache, v_cache, _heads_of(what, k_cache, q.size(2)))
    n_seqs = cu_q.numel() - 1
    if n_seqs < 0 or cu_k.numel() != n_seqs + 1:
        raise ValueError(f"{what}: cu_seqlens_q and cu_seqlens_k need one entry per sequence + 1")
    _int32(what, "cu_seqlens_q", cu_q, n_seqs + 1)
    _int32(what, "cu_seqlens_k", cu_k, n_seqs + 1)
    _int32(what, "block_tables", block_tables, n_seqs, 2)
    _workspace_ok(what, workspace)
    _out_rows(what, q, out)


def _caches_right(k_cache, v_cache, cs, di):
    return (len(cs) == 3 and v_cache.shape == cs and k_cache.dtype is _U8 and v_cache.dtype is _U8
            and k_cache.get_device() == di and v_cache.get_device() == di and cs[1] > 0
            and cs[1] % TILE == 0 and k_cache.is_contiguous() and v_cache.is_contiguous())


def _entries_right(t, di):
    return t.dtype is _I32 and t.get_device() == di and t.dim() == 1 and t.is_contiguous()


def _tables_right(t, shape, di, n):
    return (len(shape) == 2 and shape[0] >= n and shape[1] > 0 and t.dtype is _I32
            and t.get_device() == di and t.stride(1) == 1)


def _out_right(t, shape, di):
    return (t.shape == shape and t.dtype is _BF16 and t.get_device() == di and t.stride(2) == 1
            and t.stride(1) == shape[2])


def _workspace_right(t, di):
    return t.dtype is _U8 and t.get_device() == di and t.is_contiguous()


# ---------------------------------------------------------------- the operators
def scaled_store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                         v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Rows key[i] and value[i] ([N, Hk, D]) into row slot_mapping[i]; -1 slots are skipped.

    A call that writes a tile's first row begins the tile anew, with the scale of the rows that it
    writes there; otherwise the scale only grows, and the rows held so far are rounded to it where it
    does (also by rows that are dropped later, a rejected draft's, which a rollback does not undo). The
    tokens of one tile must stand next to each other in ``slot_mapping``, as those of a
    sequence do, fewer than 32 skipped ones between any two.
    """
    what = "scaled_store_kvcache"
    ks, cs, di = key.shape, k_cache.shape, key.get_device()
    k_st, v_st = key.stride(), value.stride()
    if not (di >= 0 and len(ks) == 3 and value.shape == ks and value.get_device() == di
            and key.dtype is _BF16 and value.dtype is _BF16 and k_st[2] == 1 and v_st[2] == 1
            and k_st[1] == ks[2] and v_st[1] == ks[2] and _caches_right(k_cache, v_cache, cs, di)
            and cs[2] == ks[1] * ks[2] + ROW_PAD and _entries_right(slot_mapping, di)
            and slot_mapping.size(0) == ks[0]):
        _refuse_store(what, key, value, k_cache, v_cache, slot_mapping)
    with _lib.device_of(di):
        rc = _lib.lib().nkv_scaled_store(_STORE_ARGS.pack(
            key.data_ptr(), k_st[0], value.data_ptr(), v_st[0], k_cache.data_ptr(),
            v_cache.data_ptr(), slot_mapping.data_ptr(), *ks, cs[0] * cs[1],
            torch._C._cuda_getCurrentRawStream(di)))
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
    what, Hk = "scaled_read_kvcache", num_kv_heads
    cs, bs, di = k_cache.shape, block_tables.shape, k_cache.get_device()
    row, n = cs[-1] - ROW_PAD, cu_seqlens.numel() - 1
    if not (di >= 0 and _caches_right(k_cache, v_cache, cs, di) and Hk > 0 and row > 0
            and row % Hk == 0 and n >= 0 and n_tokens >= 0 and _entries_right(cu_seqlens, di)
            and _tables_right(block_tables, bs, di, n)
            and (starts is None or _entries_right(starts, di) and starts.size(0) >= n)
            and (out is None or len(out) == 2 and all(
                _out_right(t, (n_tokens, Hk, row // Hk), di) and t.is_contiguous() for t in out))):
        _refuse_read(what, k_cache, v_cache, block_tables, cu_seqlens, n_tokens, Hk, starts, out)
    D = row // Hk
    with _lib.device_of(di):
        if out is None:
            device = k_cache.device
            out = (torch.empty((n_tokens, Hk, D), dtype=_BF16, device=device),
                   torch.empty((n_tokens, Hk, D), dtype=_BF16, device=device))
        rc = _lib.lib().nkv_scaled_read(_READ_ARGS.pack(
            k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(), block_tables.stride(0),
            bs[1], cu_seqlens.data_ptr(), 0 if starts is None else starts.data_ptr(), n, n_tokens,
            Hk, D, cs[1], cs[0], out[0].data_ptr(), out[1].data_ptr(),
            torch._C._cuda_getCurrentRawStream(di)))
    if rc:
        _lib.check(rc, what)
    return out


@functools.lru_cache(maxsize=256)
def _decode_bytes(device: int, *sizes: int) -> int:
    """Workspace bytes on a device (current), a call into the library each where they are new."""
    return max(_lib.lib().nkv_paged_decode_workspace_bytes(*sizes), 4)


def scaled_paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        context_lens: torch.Tensor, block_tables: torch.Tensor, scale: float,
                        out: torch.Tensor | None = None, workspace: torch.Tensor | None = None
                        ) -> torch.Tensor:
    """Attention of one new token per sequence: q [bs, Hq, D] -> [bs, Hq, D] (bf16).

    The arguments are ``paged_decode``'s, the workspace's size ``decode_workspace_bytes``; a sequence
    of length 0 gives zeros.
    """
    what = "scaled_paged_decode"
    qs, cs, bs, di = q.shape, k_cache.shape, block_tables.shape, q.get_device()
    q_st = q.stride()
    if not (di >= 0 and len(qs) == 3 and q.dtype is _BF16 and q_st[2] == 1 and q_st[1] == qs[2] > 0
            and _caches_right(k_cache, v_cache, cs, di) and cs[2] > ROW_PAD
            and (cs[2] - ROW_PAD) % qs[2] == 0 and _entries_right(context_lens, di)
            and context_lens.size(0) >= qs[0] and _tables_right(block_tables, bs, di, qs[0])
            and (out is None or _out_right(out, qs, di))
            and (workspace is None or _workspace_right(workspace, di))):
        _refuse_decode(what, q, k_cache, v_cache, context_lens, block_tables, out, workspace)
    n, Hq, D = qs
    lib = _lib.lib()
    with _lib.device_of(di):
        if out is None:
            out = torch.empty(qs, dtype=_BF16, device=q.device)
        if workspace is None:
            workspace = torch.empty(_decode_bytes(di, n, Hq, D, bs[1], cs[1]), dtype=_U8,
                                    device=q.device)
        rc = lib.nkv_scaled_decode(_DECODE_ARGS.pack(
            q.data_ptr(), q_st[0], k_cache.data_ptr(), v_cache.data_ptr(), block_tables.data_ptr(),
            block_tables.stride(0), context_lens.data_ptr(), n, Hq, (cs[2] - ROW_PAD) // D, D, cs[1],
            bs[1], cs[0], out.data_ptr(), out.stride(0), workspace.data_ptr(), workspace.numel(),
            torch._C._cuda_getCurrentRawStream(di), scale))
    if rc:
        _lib.check(rc, what)
    return out


# Up to so many keys a step is never split: the plan need not be asked.
_WHOLE_KEYS = 768


def scaled_prefill_workspace(q: torch.Tensor, k_cache: torch.Tensor, n_seqs: int,
                             max_seqlen_q: int, max_seqlen_k: int) -> torch.Tensor | None:
    """The workspace for splitting scaled_varlen_prefill's keys where few query tiles would leave the
    chip idle, else None; None too where the device has no such memory left, since nothing else
    needs any."""
    if max_seqlen_k <= _WHOLE_KEYS:
        return None
    D = q.size(2)
    nbytes = _lib.lib().nkv_scaled_prefill_workspace_bytes(
        n_seqs, q.size(0), int(max_seqlen_q), int(max_seqlen_k), q.size(1),
        (k_cache.size(2) - ROW_PAD) // D, D)
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
    qs, cs, bs, di = q.shape, k_cache.shape, block_tables.shape, q.get_device()
    q_st, n = q.stride(), cu_seqlens_q.numel() - 1
    if not (di >= 0 and len(qs) == 3 and q.dtype is _BF16 and q_st[2] == 1 and q_st[1] == qs[2] > 0
            and _caches_right(k_cache, v_cache, cs, di) and cs[2] > ROW_PAD
            and (cs[2] - ROW_PAD) % qs[2] == 0 and n >= 0 and _entries_right(cu_seqlens_q, di)
            and _entries_right(cu_seqlens_k, di) and cu_seqlens_k.size(0) == n + 1
            and _tables_right(block_tables, bs, di, n)
            and (out is None or _out_right(out, qs, di))
            and (workspace is None or _workspace_right(workspace, di))):
        _refuse_prefill(what, q, k_cache, v_cache, cu_seqlens_q, cu_seqlens_k, block_tables, out,
                        workspace)
    D = qs[2]
    with _lib.device_of(di):
        if out is None:
            out = torch.empty(qs, dtype=_BF16, device=q.device)
        if workspace is None and max_seqlen_k is not None:
            workspace = scaled_prefill_workspace(q, k_cache, n, max_seqlen_q, max_seqlen_k)
        rc = _lib.lib().nkv_scaled_prefill(_PREFILL_ARGS.pack(
            q.data_ptr(), q_st[0], qs[0], k_cache.data_ptr(), v_cache.data_ptr(),
            cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), block_tables.data_ptr(),
            block_tables.stride(0), bs[1], n, int(max_seqlen_q),
            0 if max_seqlen_k is None else int(max_seqlen_k), qs[1], (cs[2] - ROW_PAD) // D, D, cs[1],
            cs[0], out.data_ptr(), out.stride(0),
            0 if workspace is None else workspace.data_ptr(),
            0 if workspace is None else workspace.numel(),
            torch._C._cuda_getCurrentRawStream(di), scale))
    if rc:
        _lib.check(rc, what)
    return out
