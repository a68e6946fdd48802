"""CPU oracle for the paged K/V cache and the attention over it.

TEST INFRASTRUCTURE ONLY: imported by ``tests/`` as the checker of the device cache; the
product package never imports it.

``PagedOracle`` restates the rules of include/moe_sm100.h ("paged K/V cache") entry by
entry on Python lists and a float64 numpy pool.  An operation that the device reports
through its error word raises ``OracleError`` here, after leaving the state as the device
leaves it.  ``attend_chunk`` is the definition of the attention in float64.
"""
from __future__ import annotations

import math

import numpy as np


class OracleError(Exception):
    pass


class PagedOracle:
    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 sequences: int, max_blocks: int) -> None:
        self.shape = (layers, pages, kv_heads, page_size, head_dim)
        self.k = np.zeros(self.shape)
        self.v = np.zeros(self.shape)
        self.page = page_size
        self.table = [[-1] * max_blocks for _ in range(sequences)]
        self.lengths = [0] * sequences
        self.refs = [0] * pages

    # -- helpers -----------------------------------------------------------------
    def blocks(self, tokens: int) -> int:
        return -(-tokens // self.page)

    def _check(self, seqs: list[int], unique: bool = True) -> None:
        if any(s < 0 or s >= len(self.lengths) for s in seqs) or \
                (unique and len(set(seqs)) < len(seqs)):
            raise OracleError("sequence")

    def check_invariants(self) -> None:
        """Every page is held by exactly refs[page] table cells, blocks past the end are -1."""
        held = [0] * len(self.refs)
        for row, n in zip(self.table, self.lengths):
            for b, p in enumerate(row):
                assert (p >= 0) == (b < self.blocks(n))
                if p >= 0:
                    held[p] += 1
        assert held == self.refs

    # -- pages -------------------------------------------------------------------
    def reserve(self, seqs: list[int], counts: list[int]) -> None:
        self._check(seqs)
        plan, need = [], 0
        for s, c in zip(seqs, counts):
            n = self.lengths[s]
            if c < 0 or self.blocks(n + c) > len(self.table[s]):
                raise OracleError("length")
            copy = c > 0 and n % self.page > 0 and self.refs[self.table[s][n // self.page]] > 1
            fresh = self.blocks(n + c) - self.blocks(n) + int(copy)
            plan.append((s, c, copy, fresh))
            need += fresh
        free = [p for p, r in enumerate(self.refs) if r == 0]
        if need > len(free):
            raise OracleError("pages")
        for s, c, copy, fresh in plan:
            n = self.lengths[s]
            mine, free = free[:fresh], free[fresh:]
            at = self.blocks(n)
            if copy:
                old, new = self.table[s][at - 1], mine.pop(0)
                for pool in (self.k, self.v):
                    pool[:, new, :, :n % self.page] = pool[:, old, :, :n % self.page]
                self.refs[old] -= 1
                self.refs[new] = 1
                self.table[s][at - 1] = new
            for p in mine:
                self.table[s][at] = p
                self.refs[p] = 1
                at += 1
            self.lengths[s] = n + c

    def fork(self, parents: list[int], children: list[int]) -> None:
        self._check(children)
        self._check(parents, unique=False)
        if set(parents) & set(children):
            raise OracleError("sequence")
        bad = False
        for p, c in zip(parents, children):
            if self.lengths[c]:
                bad = True
                continue
            self.table[c] = list(self.table[p])
            self.lengths[c] = self.lengths[p]
            for x in self.table[p]:
                if x >= 0:
                    self.refs[x] += 1
        if bad:
            raise OracleError("length")

    def truncate(self, seqs: list[int], lengths: list[int]) -> None:
        self._check(seqs)
        bad = False
        for s, n in zip(seqs, lengths):
            if n < 0 or n > self.lengths[s]:
                bad = True
                continue
            for b in range(self.blocks(n), self.blocks(self.lengths[s])):
                self.refs[self.table[s][b]] -= 1
                self.table[s][b] = -1
            self.lengths[s] = n
        if bad:
            raise OracleError("length")

    def copy_pages(self, src: list[int], dst: list[int]) -> None:
        ids = range(len(self.refs))
        if any(p not in ids for p in src + dst) or len(set(dst)) < len(dst) or set(src) & set(dst):
            raise OracleError("page")
        for a, b in zip(src, dst):
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]

    def compact(self, into: "PagedOracle | None" = None) -> None:
        live = [p for p, r in enumerate(self.refs) if r > 0]
        if into is None:
            n = len(live)
            holes = [p for p in range(n) if self.refs[p] == 0]
            to = {p: p for p in live if p < n} | dict(zip([p for p in live if p >= n], holes))
            dst = self
        else:
            if len(live) > len(into.refs):
                raise OracleError("pages")
            to, dst = {p: i for i, p in enumerate(live)}, into
        refs = [0] * len(dst.refs)
        k, v = dst.k.copy(), dst.v.copy()
        for a, b in to.items():
            refs[b] = self.refs[a]
            k[:, b], v[:, b] = self.k[:, a], self.v[:, a]
        table = [[to.get(p, -1) for p in row] for row in self.table]
        lengths = list(self.lengths)
        wide = len(dst.table[0])
        dst.table = [r + [-1] * (wide - len(r)) for r in table] + \
            [[-1] * wide for _ in range(len(dst.table) - len(table))]
        dst.lengths = lengths + [0] * (len(dst.lengths) - len(lengths))
        dst.refs, dst.k, dst.v = refs, k, v

    # -- tokens ------------------------------------------------------------------
    def append(self, layer: int, k: np.ndarray, v: np.ndarray, seqs: list[int],
               starts: list[int]) -> None:
        for i, s in enumerate(seqs):
            m = starts[i + 1] - starts[i]
            for r in range(m):
                pos = self.lengths[s] - m + r
                p = self.table[s][pos // self.page]
                self.k[layer, p, :, pos % self.page] = k[starts[i] + r]
                self.v[layer, p, :, pos % self.page] = v[starts[i] + r]

    def cached(self, layer: int, s: int) -> tuple[np.ndarray, np.ndarray]:
        """[tokens, kv_heads, head_dim] keys and values of a sequence."""
        n, ids = self.lengths[s], self.table[s][:self.blocks(self.lengths[s])]
        out = []
        for pool in (self.k, self.v):
            x = pool[layer, ids].transpose(0, 2, 1, 3).reshape(-1, self.shape[2], self.shape[4])
            out.append(x[:n])
        return out[0], out[1]


def attend_chunk(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float
                 ) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Causal attention of the last ``m`` tokens of a sequence in float64: ``q`` [m, heads,
    dim], ``k`` / ``v`` [n, kv_heads, dim].  Returns out, the log of the sum of the
    exponentials, and sum_j p_j |v_j| (what the roundings of p can move out by)."""
    m, heads, dim = q.shape
    n, kv_heads, _ = k.shape
    out, mag = np.zeros((m, heads, dim)), np.zeros((m, heads, dim))
    lse = np.full((m, heads), -math.inf)
    hidden = np.arange(n)[None, :] > np.arange(n - m, n)[:, None]
    for h in range(heads):
        g = h // (heads // kv_heads)
        s = q[:, h] @ k[:, g].T * scale
        s[hidden] = -math.inf
        rows = np.flatnonzero(~hidden.all(axis=1)) if n else np.zeros(0, int)
        if not len(rows):
            continue
        top = s[rows].max(axis=1, keepdims=True)
        p = np.exp(s[rows] - top)
        total = p.sum(axis=1, keepdims=True)
        out[rows, h] = p @ v[:, g] / total
        mag[rows, h] = p @ np.abs(v[:, g]) / total
        lse[rows, h] = top[:, 0] + np.log(total[:, 0])
    return out, lse, mag
