"""Pages of latent rows for many sequences: the cache that DeepSeek-V2's attention reads while a batch is decoded.

``StaticCache`` (gemq/inference/kv_cache.py:79-114) reserves the full length for every sequence, keys and values of every
head.  ``PagedLatentCache`` holds one row of ``rank + 64`` numbers a token and layer in pages that sequences take as they grow.
Which pages a sequence has is kept on the host; the pages lie in one tensor, and what moves them (a fork's last page, compaction) is
one launch of ``copy_pages`` for all layers.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence

import torch
from torch import Tensor

from ..kernels.latent_attention import ROPE, copy_pages


@dataclass
class LatentPlan:
    """What one step of a batch needs on the device, for all layers.  Sequences lie one behind the other, ``steps`` tokens each in a
    decode step, any number in a prefill; ``slots`` is where their rows go, ``table`` and ``lens`` what each has then."""

    positions: Tensor              # int64 [tokens]
    slots: Tensor                  # int64 [tokens]
    table: Tensor                  # int32 [sequences, pages]
    lens: Tensor                   # int32 [sequences]
    steps: int = 0                 # decode: tokens a sequence; 0: prefill
    cu_q: Optional[Tensor] = None  # prefill: int32 [sequences + 1], tokens and rows before each sequence
    cu_k: Optional[Tensor] = None
    rows: Optional[Tensor] = None  # prefill with rows from before: int64 [all rows], where they lie
    # decode with shared prefixes: table and lens are then what lies behind them
    prefix_table: Optional[Tensor] = None
    prefix_lens: Optional[Tensor] = None
    starts: Optional[Tensor] = None


class PagedLatentCache:
    """``num_pages`` pages of ``page_size`` rows in each of ``num_layers`` layers.  Sequences are numbers that ``new`` and ``fork`` give."""

    def __init__(self, num_layers: int, num_pages: int, page_size: int = 64, rank: int = 512, dtype: torch.dtype = torch.bfloat16,
                 device="cuda"):
        if num_layers <= 0 or num_pages <= 0 or not (page_size in (16, 32) or (page_size > 0 and page_size % 64 == 0)):
            raise ValueError("a cache has a layer and a page at least, and page sizes of 16, 32 or multiples of 64")
        if rank not in (128, 256, 384, 512) or dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("latent rank must be 128, 256, 384 or 512, the type fp16 or bf16")
        self.page_size, self.rank, self.num_pages = page_size, rank, num_pages
        self.pages = torch.zeros((num_layers, num_pages, page_size, rank + ROPE), dtype=dtype, device=device)
        self._free: List[int] = list(range(num_pages - 1, -1, -1))  # the lowest is taken first
        self._users = [0] * num_pages
        self._table: Dict[int, List[int]] = {}
        self._len: Dict[int, int] = {}
        self._next = 0

    def layer(self, i: int) -> Tensor:
        """``[pages, page_size, rank + 64]`` of a layer: the ``cache`` of the latent operators."""
        return self.pages[i]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._len[seq]

    def pages_of(self, seq: int) -> List[int]:
        return list(self._table[seq])

    # ---- sequences ---------------------------------------------------------------------------------
    def new(self) -> int:
        seq, self._next = self._next, self._next + 1
        self._table[seq], self._len[seq] = [], 0
        return seq

    def free(self, seq: int) -> None:
        """The sequence ends; pages that no other has are free again."""
        for page in reversed(self._table.pop(seq)):
            self._release(page)
        del self._len[seq]

    def fork(self, seq: int) -> int:
        """A new sequence that begins with the rows of ``seq``: whole pages are shared, one that is filled in part is copied in all
        layers."""
        table, n = self._table[seq], self._len[seq]
        whole = n // self.page_size
        shared = table[:whole]
        child = []
        if whole < len(table):
            child = self._take(1)
            self._copy([table[whole]], child)
        for page in shared:
            self._users[page] += 1
        new = self.new()
        self._table[new], self._len[new] = shared + child, n
        return new

    def truncate(self, seq: int, length: int) -> None:
        """The sequence keeps its first ``length`` rows (a rejected draft): pages behind them are released.  A page that is then filled in
        part and shared is copied, so that what follows is written to the sequence's own."""
        if not 0 <= length <= self._len[seq]:
            raise ValueError(f"sequence {seq} has {self._len[seq]} rows, not {length}")
        table = self._table[seq]
        keep = -(-length // self.page_size)
        if length % self.page_size and self._users[table[keep - 1]] > 1:
            own = self._take(1)
            self._copy([table[keep - 1]], own)
            self._release(table[keep - 1])
            table[keep - 1] = own[0]
        for page in reversed(table[keep:]):
            self._release(page)
        del table[keep:]
        self._len[seq] = length

    def compact(self) -> int:
        """Moves the pages in use to the front of the pool, in one launch; returns how many moved.  Plans made before do not hold any more."""
        used = [p for p in range(self.num_pages) if self._users[p]]
        n = len(used)
        src = [p for p in used if p >= n]
        dst = [p for p in range(n) if not self._users[p]]
        if src:
            self._copy(src, dst)
            to = dict(zip(src, dst))
            for table in self._table.values():
                table[:] = [to.get(p, p) for p in table]
            for a, b in zip(src, dst):
                self._users[b], self._users[a] = self._users[a], 0
        self._free = list(range(self.num_pages - 1, n - 1, -1))
        return len(src)

    # ---- steps ---------------------------------------------------------------------------------------
    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> List[int]:
        """Room for ``counts[i]`` more rows of ``seqs[i]`` -> their slots, one sequence behind the other.  All or nothing."""
        if len(set(seqs)) != len(seqs) or len(counts) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("every sequence once, with the number of its new rows")
        need = [-(-(self._len[s] + c) // self.page_size) - len(self._table[s]) for s, c in zip(seqs, counts)]
        pages = self._take(sum(need))
        slots, at = [], 0
        for s, c, k in zip(seqs, counts, need):
            self._table[s].extend(pages[at:at + k])
            at += k
            n, table = self._len[s], self._table[s]
            slots += [table[i // self.page_size] * self.page_size + i % self.page_size for i in range(n, n + c)]
            self._len[s] = n + c
        return slots

    def plan_decode(self, seqs: Sequence[int], steps: int = 1, groups: Optional[Sequence[int]] = None) -> LatentPlan:
        """``steps`` new rows for every sequence.  ``groups`` gives the number of sequences of each group that may share a prefix: the pages that all of
        a group begin with are then read once (``latent_decode_shared``)."""
        if steps < 1:
            raise ValueError(f"a decode step has one new row a sequence at least, not {steps}")
        if groups is not None and (sum(groups) != len(seqs) or any(g <= 0 for g in groups) or not groups):
            raise ValueError("groups must cover the sequences, one or more in each")
        slots = self.extend(seqs, [steps] * len(seqs))
        positions = [self._len[s] - steps + i for s in seqs for i in range(steps)]
        tables, lens = [self._table[s] for s in seqs], [self._len[s] for s in seqs]
        plan = LatentPlan(self._ints(positions, torch.int64), self._ints(slots, torch.int64), None, None, steps)
        if groups is not None:
            prefix, at, starts = [], 0, [0]
            for g in groups:
                mine = tables[at:at + g]
                # whole pages that existed before this step: the new rows, and what only some have, stay behind
                least = min((lens[i] - steps) // self.page_size for i in range(at, at + g))
                same = 0
                while g > 1 and same < least and all(t[same] == mine[0][same] for t in mine):
                    same += 1
                prefix.append(mine[0][:same])
                for i in range(at, at + g):
                    tables[i] = tables[i][same:]
                    lens[i] -= same * self.page_size
                at += g
                starts.append(at)
            plan.prefix_table, plan.prefix_lens = self._tables(prefix), self._ints([len(p) * self.page_size for p in prefix], torch.int32)
            plan.starts = self._ints(starts, torch.int32)
        plan.table, plan.lens = self._tables(tables), self._ints(lens, torch.int32)
        return plan

    def plan_prefill(self, seqs: Sequence[int], counts: Sequence[int]) -> LatentPlan:
        """``counts[i]`` new rows of ``seqs[i]``, behind those it has already."""
        before = [self._len[s] for s in seqs]
        slots = self.extend(seqs, counts)
        positions = [n + i for n, c in zip(before, counts) for i in range(c)]
        cu_q, cu_k = [0], [0]
        for n, c in zip(before, counts):
            cu_q.append(cu_q[-1] + c)
            cu_k.append(cu_k[-1] + n + c)
        rows = None
        if any(before):
            page = self.page_size
            rows = self._ints([self._table[s][i // page] * page + i % page for s in seqs for i in range(self._len[s])], torch.int64)
        return LatentPlan(self._ints(positions, torch.int64), self._ints(slots, torch.int64), self._tables([self._table[s] for s in seqs]),
                          self._ints([self._len[s] for s in seqs], torch.int32), 0, self._ints(cu_q, torch.int32), self._ints(cu_k, torch.int32),
                          rows)

    # ---- inside --------------------------------------------------------------------------------------
    def _ints(self, v, dtype) -> Tensor:
        return torch.tensor(v, dtype=dtype, device=self.pages.device)

    def _tables(self, tables) -> Tensor:
        wide = max([len(t) for t in tables] + [1])
        return self._ints([t + [0] * (wide - len(t)) for t in tables], torch.int32).view(len(tables), wide)

    def _take(self, n: int) -> List[int]:
        if n > len(self._free):
            raise RuntimeError(f"the cache is full: {n} pages wanted, {len(self._free)} of {self.num_pages} free")
        taken = [self._free.pop() for _ in range(n)]
        for p in taken:
            self._users[p] = 1
        return taken

    def _release(self, page: int) -> None:
        self._users[page] -= 1
        if not self._users[page]:
            self._free.append(page)

    def _copy(self, src: List[int], dst: List[int]) -> None:
        copy_pages(self.pages, self._ints(src, torch.int64), self._ints(dst, torch.int64))
