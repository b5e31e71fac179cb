"""Sequences over one K/V pool whose pages are counted and listed on the device.

The reference keeps its block manager on the host (nanokvllm/engine/block_manager.py:13-138), so
a step's tables and slots are host data. ``PagedSequences`` keeps a reference count per page, and a
length and a block table per row (sequence), in device memory, and changes them with kernels: new
tokens take pages (``append``), sequences end, roll back or shrink (``truncate``), beams and samples
start from a common prefix (``fork``), and the pages in use move to the pool's lower end
(``compact``). No call reads anything back, so a decode loop (append, store, attention, sampling)
can be captured in a HIP graph. ``block_tables`` and ``context_lens`` go to ``set_context`` as they
are (rows are then the batch) or indexed by the step's rows.
"""
from __future__ import annotations

import struct
import weakref

import torch

from .. import _lib
from ..layers import attention
from ..layers.kv_cache import KVCachePool
from ..layers.scaled_cache import TILE, ScaledKVCachePool

_PAGES = struct.Struct("13q")  # nkv_pages
_I32 = torch.int32


class PagedSequences:
    """Up to ``max_seqs`` rows of at most ``max_blocks_per_seq`` pages each over ``kv_cache``, a
    ``KVCachePool`` or its tensor [2, layers, pages, block_size, Hk, D], or a ``ScaledKVCachePool`` or
    its tensor (uint8 [2, layers, pages, block_size, row]; a copy of part of a page then brings whole
    tiles, their scales among them).

    ``state`` is one int32 buffer [pages + max_seqs + max_seqs * max_blocks_per_seq]: the reference
    counts, the lengths (``context_lens``) and the tables (``block_tables``, -1 past a row's
    pages), each a view of it. A new object has all pages free and all rows empty; given a
    ``state`` (another object's, or a clone of one kept before a step) it goes on from there.
    ``state.copy_(kept)`` takes an object back to one; ``state`` and ``kv_cache`` cannot be set.

    Lists are int32 tensors on the pool's device. An entry of -1 is padding, and a row named twice
    counts where it is named first. Pages are taken lowest first and in the list's order: an entry
    is carried out if it needs no page or the pages needed by all entries up to it are free before
    the call, else it is refused and changes nothing. Each call returns a ``status`` (int32, 1:
    carried out, 0: refused or padding). A row's last page, where it is filled in part, belongs to
    that row alone; full pages may be shared, so code that writes rows in place (a compression
    step) needs a fork made with ``share_pages=False``.

    Calls run on the current stream of the pool's device and share the object's state and
    workspace: the caller orders calls of one object that it makes on several streams, captured
    graphs' replays among them. A graph that captured a call needs the pool for as long as it is
    replayed; state and workspace stay allocated after the object is dropped, until
    ``release_retired_decode_workspaces()``.
    """

    def __init__(self, kv_cache: torch.Tensor | KVCachePool | ScaledKVCachePool, max_seqs: int,
                 max_blocks_per_seq: int, state: torch.Tensor | None = None):
        kv = kv_cache.kv_cache if isinstance(kv_cache, (KVCachePool, ScaledKVCachePool)) else kv_cache
        self._scaled = kv.dim() == 5 and kv.dtype is torch.uint8
        if self._scaled and kv.size(3) % TILE:
            raise ValueError(f"PagedSequences: block_size {kv.size(3)} of a block-scaled pool is not "
                             f"a multiple of {TILE}")
        if kv.dim() != (5 if self._scaled else 6) or kv.size(0) != 2 or not kv.is_contiguous():
            raise ValueError("PagedSequences: the pool must be contiguous [2, layers, pages, "
                             f"block_size, Hk, D], got {tuple(kv.shape)}")
        _lib.require_device(kv.device, state=state)
        if max_seqs <= 0 or max_blocks_per_seq <= 0:
            raise ValueError("PagedSequences: max_seqs and max_blocks_per_seq must be > 0")
        _, layers, pages, block = kv.shape[:4]
        n = pages + max_seqs + max_seqs * max_blocks_per_seq
        if state is None:
            state = torch.zeros(n, dtype=_I32, device=kv.device)
            state[pages + max_seqs:].fill_(-1)
        if state.dtype is not _I32 or state.dim() != 1 or state.numel() != n \
                or not state.is_contiguous():
            raise ValueError(f"PagedSequences: state must be {n} contiguous int32")
        nbytes = _lib.lib().nkv_pages_workspace_bytes(pages)
        if nbytes == 0:
            raise ValueError(f"PagedSequences: a pool of {pages} pages (1 to 2^20)")
        self._kv, self._state = kv, state
        self.max_seqs, self.max_blocks, self.block_size = max_seqs, max_blocks_per_seq, block
        self._pages, self._device = pages, kv.get_device()
        self._workspace = torch.empty(nbytes, dtype=torch.uint8, device=kv.device)
        self._streams = {torch._C._cuda_getCurrentRawStream(self._device)}  # the allocations' first
        self._captured = False
        at = state.data_ptr()
        self._args = _PAGES.pack(kv.data_ptr(), 2 * layers, pages, block,
                                 kv.shape[4:].numel() * kv.element_size(), at, at + 4 * pages,
                                 at + 4 * (pages + max_seqs), max_blocks_per_seq,
                                 max_blocks_per_seq, max_seqs, self._workspace.data_ptr(), nbytes)

    def __reduce__(self):  # a copy's calls go to the copied buffers and a workspace of its own
        return type(self), (self._kv, self.max_seqs, self.max_blocks, self._state)

    # The kernels are given the addresses of these two once, so that an attribute set to another
    # tensor would leave them writing to memory that nothing owns any more.
    @property
    def kv_cache(self) -> torch.Tensor:
        return self._kv

    @property
    def state(self) -> torch.Tensor:
        return self._state

    @property
    def ref_counts(self) -> torch.Tensor:
        return self._state[:self._pages]

    @property
    def context_lens(self) -> torch.Tensor:
        return self._state[self._pages:self._pages + self.max_seqs]

    @property
    def block_tables(self) -> torch.Tensor:
        return self._state[self._pages + self.max_seqs:].view(self.max_seqs, self.max_blocks)

    def _list(self, what: str, t: torch.Tensor, n: int | None = None) -> int:
        """The list's length (``n`` entries, if given)."""
        if not (t.get_device() == self._device and t.dtype is _I32 and t.dim() == 1
                and t.is_contiguous() and (n is None or t.numel() == n)):
            raise ValueError(f"{what} must be contiguous int32 [{'n' if n is None else n}] on the "
                             f"pool's device, got {t.dtype} {tuple(t.shape)} on {t.device}")
        return t.numel()

    def _call(self, fn, what, *args):
        with _lib.device_of(self._device):
            stream = torch._C._cuda_getCurrentRawStream(self._device)
            if torch.cuda.is_current_stream_capturing():
                self._keep_for_graphs()
            elif stream not in self._streams:
                self._use_on(stream)
            rc = fn(self._args, *args, stream)
        if rc:
            _lib.check(rc, what)

    def _use_on(self, stream):
        """The buffers' memory, once freed, waits for what still runs on another stream."""
        for t in (self._workspace, self._state):
            t.record_stream(torch.cuda.current_stream())
        self._streams.add(stream)

    def _keep_for_graphs(self):
        """A graph holds the buffers' addresses: dropping the object leaves them allocated until
        release_retired_decode_workspaces()."""
        if not self._captured:
            self._captured = True
            weakref.finalize(self, attention.retire_workspace, self._workspace,
                             self._state).atexit = False

    def append(self, rows: torch.Tensor, cu_seqlens_q: torch.Tensor | None = None,
               n_tokens: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """New tokens: one for each of ``rows``, or ``cu_seqlens_q`` (int32 [n + 1]) in all
        ``n_tokens`` of them. -> (slot_mapping [n_tokens], status [n]): the tokens' slots in the
        order of the list, -1 for refused rows' and for those outside ``cu_seqlens_q``."""
        n = self._list("append: rows", rows)
        if cu_seqlens_q is None:
            if n_tokens is not None and n_tokens != n:
                raise ValueError("append: without cu_seqlens_q there is one token a row")
            n_tokens, cu = n, None
        else:
            self._list("append: cu_seqlens_q", cu_seqlens_q, n + 1)
            if n_tokens is None:
                raise ValueError("append: cu_seqlens_q needs n_tokens, the tokens' number on the "
                                 "host")
            cu = cu_seqlens_q.data_ptr()
        slots, status = rows.new_empty(n_tokens), rows.new_empty(n)
        self._call(_lib.lib().nkv_pages_append, "append", rows.data_ptr(), n, cu, n_tokens,
                   slots.data_ptr(), status.data_ptr())
        return slots, status

    def truncate(self, rows: torch.Tensor, lens: torch.Tensor,
                 pages: torch.Tensor | None = None) -> torch.Tensor:
        """Row ``rows[i]`` keeps its first ``lens[i]`` tokens (0: the sequence ends). Pages that no
        row holds any more are free; one that stays in part while others hold it is copied.
        ``pages``: ids that lose a reference besides, -1 for none (the freed blocks in the events
        of a compression step); those free before the call are passed over. -> status [n]."""
        n = self._list("truncate: rows", rows)
        self._list("truncate: lens", lens, n)
        m = 0 if pages is None else self._list("truncate: pages", pages)
        status = rows.new_empty(n)
        fn = _lib.lib().nkv_scaled_pages_truncate if self._scaled else _lib.lib().nkv_pages_truncate
        self._call(fn, "truncate", rows.data_ptr(), lens.data_ptr(), n,
                   pages.data_ptr() if m else None, m, status.data_ptr())
        return status

    def fork(self, parents: torch.Tensor, children: torch.Tensor,
             share_pages: bool = True) -> torch.Tensor:
        """The empty row ``children[i]`` becomes a copy of row ``parents[i]``: the parent's full
        pages are shared and the one filled in part is copied, or all are copied
        (``share_pages=False``). -> status [n]."""
        n = self._list("fork: parents", parents)
        self._list("fork: children", children, n)
        status = parents.new_empty(n)
        fn = _lib.lib().nkv_scaled_pages_fork if self._scaled else _lib.lib().nkv_pages_fork
        self._call(fn, "fork", parents.data_ptr(), children.data_ptr(), n,
                   1 if share_pages else 0, status.data_ptr())
        return status

    def compact(self, max_moves: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """Moves at most ``max_moves`` pages (default: as many as it takes) from the top of the
        pool to free ones below, so that with enough moves the pages in use are the first ones.
        -> (info int32 [2]: pages in use and moves made, moves int32 [max_moves, 2]: from and to,
        -1 padded)."""
        if max_moves is None:
            max_moves = self._pages
        if not 0 <= max_moves <= 2 ** 20:
            raise ValueError(f"compact: max_moves {max_moves} must be 0 to 2^20")
        out = self._state.new_empty(2 + 2 * max_moves)
        self._call(_lib.lib().nkv_pages_compact, "compact", max_moves, out.data_ptr(),
                   out.data_ptr() + 8)
        return out[:2], out[2:].view(-1, 2)
