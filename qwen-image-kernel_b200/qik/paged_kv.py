"""Paged KV cache: pages of tokens shared between sequences, next to the contiguous prefix
slab of ``qik.kv_cache`` (which holds one prefix per batch entry and cannot grow, share or
free parts of it).

K and V are two allocations ``[layers, pages, heads, page, D]``, so one head's tokens of a page
are contiguous rows, as in the slab.  The host owns the allocation: which pages a sequence
has, how many sequences use a page, which are free.  The device sees a ``PagedStep`` (page
table, lengths, positions, slots of one forward pass, uploaded once for all layers) and page
copies (``copy_pages``).  A page that is not full belongs to one sequence: a fork shares the full
pages and copies the rest of the last one, so that a store never writes to a shared page.
"""
from __future__ import annotations

import heapq

import numpy as np
import torch

from . import _calls


class CacheFull(RuntimeError):
    """Not enough free pages (nothing was changed)."""


def copy_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, moves) -> None:
    """Copy the first tokens of pages to other pages, in every layer and head of both pools.

    k_pages, v_pages: [layers, pages, heads, page, D] (or one layer's [pages, heads, page, D]);
    moves: a list of (from, to, tokens), or an int array or tensor [n, 3].  In a page the tokens of a
    head are contiguous, or the heads of a token and then the tokens (a pool [pages, page, heads, D] seen
    with its heads first); other strides are refused.  The rest of a written page stays as it is.  No page may be written twice or both read and written in one
    call; indices are checked before anything is launched."""
    if not isinstance(moves, (list, tuple)):
        moves = moves.tolist()
    _calls.copy_pages(k_pages, v_pages, moves)


class PagedStep:
    """What one forward pass over a batch of sequences needs, on the device:

    * ``page_table`` int32 [batch, pages of the longest], ``seq_lens`` int32 [batch] (tokens in the
      cache, the new ones among them), ``query_starts`` int32 [batch + 1];
    * ``positions`` and ``slots`` int64 [new tokens]: each new token's place in its sequence and
      in the pools;
    * ``max_new`` and ``max_kv``, on the host.
    """

    def __init__(self, page_table: np.ndarray, seq_lens: np.ndarray, query_starts: np.ndarray, positions: np.ndarray,
                 slots: np.ndarray, device: torch.device):
        B, T = len(seq_lens), len(positions)
        parts = [positions.astype(np.int64).view(np.int32), slots.astype(np.int64).view(np.int32),
                 page_table.astype(np.int32).ravel(), seq_lens.astype(np.int32), query_starts.astype(np.int32)]
        host = torch.from_numpy(np.concatenate(parts))
        if device.type == "cuda":
            host = host.pin_memory()
        all_ = host.to(device, non_blocking=True)  # one copy for the whole step
        ends = np.cumsum([len(p) for p in parts])
        self.positions = all_[:ends[0]].view(torch.int64)
        self.slots = all_[ends[0]:ends[1]].view(torch.int64)
        self.page_table = all_[ends[1]:ends[2]].view(B, -1) if B else all_[:0].view(0, 0)
        self.seq_lens = all_[ends[2]:ends[3]]
        self.query_starts = all_[ends[3]:ends[4]]
        self.max_new = int(np.diff(query_starts).max()) if B else 0
        self.max_kv = int(seq_lens.max()) if B else 0
        self.tokens = T


class PagedKVCache:
    """Pages of ``page_size`` tokens for ``num_layers`` layers, and the sequences that use them."""

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device: torch.device | str = "cuda"):
        if min(num_layers, num_pages, num_kv_heads, head_dim) <= 0:
            raise ValueError("qik: PagedKVCache: sizes must be positive")
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"qik: PagedKVCache: a page is a power of two of 16 to 4096 tokens, got {page_size}")
        shape = (num_layers, num_pages, num_kv_heads, page_size, head_dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=device)
        self.v_pages = torch.empty(shape, dtype=dtype, device=device)
        self.device = self.k_pages.device
        self.num_layers, self.num_pages, self.page_size = num_layers, num_pages, page_size
        self._users = [0] * num_pages            # sequences that have the page
        self._free = list(range(num_pages))      # a heap: the lowest page first
        self._pages: dict[int, list[int]] = {}   # sequence -> its pages in order
        self._length: dict[int, int] = {}
        self._next = 0

    # ---- what there is
    @property
    def free_pages(self) -> int:
        return len(self._free)

    def sequences(self) -> list[int]:
        return list(self._pages)

    def length(self, seq: int) -> int:
        return self._length[self._known(seq)]

    def pages_of(self, seq: int) -> list[int]:
        return list(self._pages[self._known(seq)])

    def layer(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        """One layer's (k_pages, v_pages), each [pages, heads, page, D]."""
        return self.k_pages[i], self.v_pages[i]

    def _known(self, seq: int) -> int:
        if seq not in self._pages:
            raise KeyError(f"qik: PagedKVCache: no sequence {seq}")
        return seq

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise CacheFull(f"qik: PagedKVCache: {n} pages wanted, {len(self._free)} of {self.num_pages} are free")
        got = [heapq.heappop(self._free) for _ in range(n)]
        for p in got:
            self._users[p] = 1
        return got

    def _drop(self, pages: list[int]) -> None:
        for p in pages:
            self._users[p] -= 1
            if self._users[p] == 0:
                heapq.heappush(self._free, p)

    def _copy(self, moves: list[tuple[int, int, int]], taken: list[int]) -> None:
        """copy_pages; the pages taken for it are given back when it fails."""
        try:
            copy_pages(self.k_pages, self.v_pages, moves)
        except BaseException:
            self._drop(taken)
            raise

    # ---- sequences
    def new_sequence(self) -> int:
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._length[seq] = [], 0
        return seq

    def free(self, *seqs: int) -> None:
        """Give up sequences; their pages that no other sequence has become free."""
        if len(set(seqs)) < len(seqs):
            raise ValueError("qik: PagedKVCache.free: the same sequence twice")
        for seq in seqs:
            self._known(seq)
        for seq in seqs:
            self._drop(self._pages.pop(seq))
            del self._length[seq]

    def fork(self, seq: int, count: int = 1) -> list[int]:
        """``count`` new sequences that continue ``seq``: its full pages are shared, a partly
        filled last page is copied for each (one kernel for all children and layers)."""
        pages, length = self._pages[self._known(seq)], self._length[seq]
        if count < 0:
            raise ValueError(f"qik: PagedKVCache.fork: {count} children")
        full, rest = divmod(length, self.page_size)
        own = self._take(count) if rest else []
        if own:
            self._copy([(pages[full], p, rest) for p in own], own)
        children = []
        for i in range(count):
            child = self.new_sequence()
            self._pages[child] = pages[:full] + ([own[i]] if rest else [])
            self._length[child] = length
            for p in pages[:full]:
                self._users[p] += 1
            children.append(child)
        return children

    def truncate(self, seq: int, length: int) -> None:
        """Forget the tokens of ``seq`` behind its first ``length`` (drafted ones that were
        rejected).  A shared page that is no longer full is copied, to a page that the call itself
        gives up where no other is free; raises CacheFull, with nothing changed, when there is neither."""
        pages = self._pages[self._known(seq)]
        if not 0 <= length <= self._length[seq]:
            raise ValueError(f"qik: PagedKVCache.truncate: {length} tokens of {self._length[seq]}")
        full, rest = divmod(length, self.page_size)
        keep = pages[:full + (1 if rest else 0)]
        if rest and self._users[keep[-1]] > 1:
            own = [p for p in pages[full + 1:] if self._users[p] == 1]
            if self._free or not own:
                new = self._take(1)[0]
                self._copy([(keep[-1], new, rest)], [new])
            else:
                new = own[0]
                self._copy([(keep[-1], new, rest)], [])
                self._users[new] += 1  # (it stays the sequence's)
            self._drop(pages[full:])
            keep[-1] = new
        else:
            self._drop(pages[len(keep):])
        self._pages[seq], self._length[seq] = keep, length

    def step(self, seqs: list[int], new_tokens: list[int]) -> PagedStep:
        """Make room for ``new_tokens[i]`` more tokens of ``seqs[i]`` and return the forward pass
        that stores and reads them.  Raises CacheFull, with nothing changed, when the free pages
        do not suffice."""
        if len(seqs) != len(new_tokens) or len(set(seqs)) < len(seqs):
            raise ValueError("qik: PagedKVCache.step: one count for each of distinct sequences")
        size = self.page_size
        want = []
        for seq, n in zip(seqs, new_tokens):
            if n < 0:
                raise ValueError(f"qik: PagedKVCache.step: {n} new tokens")
            want.append(max(0, -(-(self._length[self._known(seq)] + n) // size) - len(self._pages[seq])))
        got = self._take(sum(want))
        at = 0
        for seq, n, w in zip(seqs, new_tokens, want):
            self._pages[seq].extend(got[at:at + w])
            self._length[seq] += n
            at += w
        width = max((len(self._pages[s]) for s in seqs), default=0)
        table = np.zeros((len(seqs), width), np.int32)
        positions, slots = [], []
        for i, (seq, n) in enumerate(zip(seqs, new_tokens)):
            row = np.asarray(self._pages[seq], np.int64)
            table[i, :len(row)] = row
            pos = np.arange(self._length[seq] - n, self._length[seq], dtype=np.int64)
            positions.append(pos)
            slots.append(row[pos // size] * size + pos % size if n else pos)
        empty = np.zeros(0, np.int64)
        return PagedStep(table, np.asarray([self._length[s] for s in seqs], np.int64),
                         np.concatenate(([0], np.cumsum(new_tokens, dtype=np.int64))) if seqs else np.zeros(1, np.int64),
                         np.concatenate(positions or [empty]), np.concatenate(slots or [empty]), self.device)

    def compact(self) -> int:
        """Move the pages in use down into the free ones below them, so that they are the first
        pages of the pools; returns how many moved.  Steps made before no longer hold."""
        live = self.num_pages - len(self._free)
        holes = sorted(p for p in self._free if p < live)
        high = [p for p in range(live, self.num_pages) if self._users[p]]
        if not high:
            return 0
        filled = {}
        for seq, pages in self._pages.items():
            for i, p in enumerate(pages):
                filled[p] = max(filled.get(p, 0), min(self.page_size, max(0, self._length[seq] - i * self.page_size)))
        copy_pages(self.k_pages, self.v_pages, [(a, b, filled[a]) for a, b in zip(high, holes)])
        to = dict(zip(high, holes))
        for seq, pages in self._pages.items():
            self._pages[seq] = [to.get(p, p) for p in pages]
        for a, b in to.items():
            self._users[b], self._users[a] = self._users[a], 0
        self._free = list(range(live, self.num_pages))
        heapq.heapify(self._free)
        return len(to)
