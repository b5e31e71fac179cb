"""Sequences over a pool of counted pages, one list entry after the other (plain Python).

The rules of ``PagedSequences`` (block counts as in nanokvllm/engine/block_manager.py:13-138): every
decision is by the state before the call; an entry is granted if the pages needed by all entries up
to it were free before the call; the lowest free pages are taken first.
"""
from __future__ import annotations

import torch


class PagedSequencesRef:
    def __init__(self, kv: torch.Tensor, rows: int, width: int):
        self.kv = kv.clone()  # [2, layers, pages, B, Hk, D], any dtype that copies bit by bit
        self.B, self.NB, self.S, self.W = kv.size(3), kv.size(2), rows, width
        self.refs, self.lens = [0] * self.NB, [0] * rows
        self.tables = [[-1] * width for _ in range(rows)]

    def state(self) -> torch.Tensor:
        return torch.tensor(self.refs + self.lens + [x for t in self.tables for x in t],
                            dtype=torch.int32)

    def _pages(self, n):
        return -(-n // self.B)

    def _firsts(self, rows):
        seen, out = set(), []
        for r in rows:
            out.append(0 <= r < self.S and r not in seen)
            seen.add(r)
        return out

    def _grant(self, fit, need):
        """-> for each entry its pages, or None where it is refused."""
        free = [p for p, c in enumerate(self.refs) if c == 0]
        out, at = [], 0
        for f, n in zip(fit, need):
            n = n if f else 0
            at += n
            out.append((free[at - n:at] if n else []) if f and (n == 0 or at <= len(free))
                       else None)
        return out

    def _copy(self, src, dst, rows):
        self.kv[:, :, dst, :rows] = self.kv[:, :, src, :rows]

    def append(self, rows, counts=None, cu=None, n_tokens=None):
        if cu is not None:
            counts = [b - a for a, b in zip(cu, cu[1:])]
            bad = any(a < 0 or b < a or b > n_tokens for a, b in zip(cu, cu[1:]))
        else:
            counts, bad, cu, n_tokens = [1] * len(rows), False, range(len(rows)), len(rows)
        fit, need = [], []
        for r, c, f in zip(rows, counts, self._firsts(rows)):
            ok = f and not bad and self._pages(self.lens[r] + c) <= self.W
            fit.append(ok)
            need.append(self._pages(self.lens[r] + c) - self._pages(self.lens[r]) if ok else 0)
        slots = [-1] * n_tokens
        got = self._grant(fit, need)
        for i, (r, c, pages) in enumerate(zip(rows, counts, got)):
            if pages is None:
                continue
            t, n = self.tables[r], self.lens[r]
            t[self._pages(n):self._pages(n + c)] = pages
            for p in pages:
                self.refs[p] = 1
            for j in range(c):
                slots[cu[i] + j] = t[(n + j) // self.B] * self.B + (n + j) % self.B
            self.lens[r] = n + c
        return slots, [int(g is not None) for g in got]

    def truncate(self, rows, keeps, pages=()):
        fit, own = [], []
        for r, k, f in zip(rows, keeps, self._firsts(rows)):
            ok = f and 0 <= k <= self.lens[r]
            fit.append(ok)
            own.append(int(ok and k < self.lens[r] and k % self.B > 0
                           and self.refs[self.tables[r][k // self.B]] > 1))
        got = self._grant(fit, own)
        drop = [p for p in pages if 0 <= p < self.NB and self.refs[p] > 0]
        for r, k, new in zip(rows, keeps, got):
            if new is None:
                continue
            t = self.tables[r]
            if new:
                old = t[k // self.B]
                self._copy(old, new[0], k % self.B)
                t[k // self.B] = new[0]
                self.refs[new[0]] = 1
                drop.append(old)
            for j in range(self._pages(k), self._pages(self.lens[r])):
                drop.append(t[j])
                t[j] = -1
            self.lens[r] = k
        for p in drop:
            self.refs[p] = max(0, self.refs[p] - 1)
        return [int(g is not None) for g in got]

    def fork(self, parents, children, share=True):
        lens, fit, need = list(self.lens), [], []
        for p, c, f in zip(parents, children, self._firsts(children)):
            ok = f and 0 <= p < self.S and lens[c] == 0
            fit.append(ok)
            need.append(self._pages(lens[p]) - (lens[p] // self.B if share else 0) if ok else 0)
        got = self._grant(fit, need)
        for p, c, pages in zip(parents, children, got):
            if pages is None:
                continue
            n, full = lens[p], lens[p] // self.B if share else 0
            for j in range(full):
                self.tables[c][j] = self.tables[p][j]
                self.refs[self.tables[p][j]] += 1
            for j, page in enumerate(pages, full):
                self._copy(self.tables[p][j], page, min(self.B, n - j * self.B))
                self.tables[c][j] = page
                self.refs[page] = 1
            self.lens[c] = n
        return [int(g is not None) for g in got]

    def compact(self, max_moves):
        n_live = sum(c > 0 for c in self.refs)
        holes = [p for p in range(n_live) if self.refs[p] == 0]
        above = [p for p in range(self.NB - 1, n_live - 1, -1) if self.refs[p] > 0]
        moves = list(zip(above, holes))[:max_moves]
        for src, dst in moves:
            self._copy(src, dst, self.B)
            self.refs[dst], self.refs[src] = self.refs[src], 0
            self.tables = [[dst if x == src else x for x in t] for t in self.tables]
        return [n_live, len(moves)], [list(m) for m in moves] + [[-1, -1]] * (max_moves -
                                                                              len(moves))
