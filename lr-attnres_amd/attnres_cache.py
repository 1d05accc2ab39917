"""A decoder's key-value cache in pages, for generation with the HIP kernels.

The reference's attention keeps its cache as a tensor that every new token concatenates to (``model.py:430-569``).
Here each layer's keys and values lie in pages of ``page_size`` tokens that are handed out as sequences grow, so that a
step moves nothing that is cached and sequences of different lengths share one allocation.  All layers use one block
table: a page number stands for that page of every layer.

The host keeps the lengths and the free pages; the device has the block table and the counts that the operators read
(``attnres_ops.qkv_norm_rotary_cached``, ``cached_attention``, ``evict_cached_tokens``), so a step needs no
synchronization.  What a call changes on the device it changes in the order of the current stream.

A step captured in a HIP graph advances the device's counts at every replay, and the host's once, at its capture: that
one is the first replay's.  So reserve the pages of all of them before the capture, and tell the host of every replay
after the first with ``replayed``.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor


def send(numbers, like: Tensor) -> Tensor:
    """Whole numbers of the host as an int32 tensor on ``like``'s device, in its stream's order: from pinned memory, so that
    nothing waits for the GPU.  Not while a graph is captured, whose replays would read that memory again."""
    t = torch.as_tensor(numbers, dtype=torch.int32)
    if not like.is_cuda:
        return t.to(like.device)
    check_no_capture(like)
    return t.pin_memory().to(like.device, non_blocking=True)


def check_no_capture(like: Tensor) -> None:
    if like.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a captured step takes no pages and no counts of its own: reserve its pages before the capture, and "
                           "give every sequence the same number of tokens")


class PagedCache:
    """Pages of ``layers`` layers for ``batch`` sequences of at most ``max_tokens`` cached tokens.

    ``pages``: how many there are in all (enough for every sequence's ``max_tokens``, and ``spare_tokens`` more for a copy
    while ``evict`` moves tokens, unless given).  With ``weights`` the attention that each cached token receives is added up
    in fp32, which ``evict`` goes by.

    ``k``, ``v`` [layers, pages, kv_heads, page_size, head_dim]; ``weights`` [layers, pages, kv_heads, page_size] or None;
    ``table`` [batch, pages of a sequence], ``cached`` and ``positions`` [batch] (int32): each sequence's pages, the tokens
    it has in the cache, and the position of its next one (further on, once tokens were evicted).
    """

    def __init__(self, layers: int, kv_heads: int, head_dim: int, batch: int, max_tokens: int, page_size: int = 64,
                 pages: Optional[int] = None, spare_tokens: int = 0, dtype=torch.bfloat16, device="cuda",
                 weights: bool = False):
        if min(layers, kv_heads, head_dim, batch, max_tokens, page_size) < 1:
            raise ValueError("layers, kv_heads, head_dim, batch, max_tokens and page_size must be >= 1")
        per = -(-max_tokens // page_size)
        self.page_size, self.max_tokens = page_size, max_tokens
        self.pages = batch * (per + -(-spare_tokens // page_size)) if pages is None else pages
        if self.pages < 1:
            raise ValueError("pages must be >= 1")
        shape = (layers, self.pages, kv_heads, page_size)
        self.k = torch.empty((*shape, head_dim), dtype=dtype, device=device)
        self.v = torch.empty((*shape, head_dim), dtype=dtype, device=device)
        self.weights = torch.zeros(shape, dtype=torch.float32, device=device) if weights else None
        self.table = torch.full((batch, per), -1, dtype=torch.int32, device=device)
        self.cached = torch.zeros((batch,), dtype=torch.int32, device=device)
        self.positions = torch.zeros((batch,), dtype=torch.int32, device=device)
        # the host's side of the same
        self.lengths = [0] * batch
        self.next_positions = [0] * batch
        self._owned = [[] for _ in range(batch)]
        self._free = list(range(self.pages - 1, -1, -1))

    @property
    def batch(self) -> int:
        return len(self.lengths)

    def _write_table(self):
        rows = torch.full(tuple(self.table.shape), -1, dtype=torch.int32)
        for b, owned in enumerate(self._owned):
            rows[b, :len(owned)] = torch.tensor(owned, dtype=torch.int32)
        self.table.copy_(send(rows, self.table))

    def _counts(self, fresh) -> list:
        new = [fresh] * self.batch if isinstance(fresh, int) else [int(n) for n in fresh]
        if len(new) != self.batch or min(new) < 0:
            raise ValueError(f"new tokens must be a count, or {self.batch} of them, >= 0, got {fresh}")
        return new

    def reserve(self, fresh) -> None:
        """Pages for ``fresh`` more tokens of each sequence (a count, or one a sequence); raises, with nothing taken, where
        there are none."""
        new = self._counts(fresh)
        need = []
        for b, n in enumerate(new):
            total = self.lengths[b] + n
            if total > self.max_tokens:
                raise RuntimeError(f"sequence {b} would have {total} cached tokens, above max_tokens {self.max_tokens}")
            need.append(max(0, -(-total // self.page_size) - len(self._owned[b])))
        if sum(need) > len(self._free):
            raise RuntimeError(f"{sum(need)} pages are needed and {len(self._free)} of {self.pages} are free")
        if any(need):
            check_no_capture(self.table)
            for b, n in enumerate(need):
                self._owned[b] += [self._free.pop() for _ in range(n)]
            self._write_table()

    def advance(self, fresh) -> None:
        """``fresh`` tokens of each sequence have been written (into reserved pages)."""
        new = self._counts(fresh)
        step = new[0] if len(set(new)) == 1 else send(new, self.cached)
        self.replayed(new)
        self.cached += step
        self.positions += step

    def replayed(self, fresh) -> None:
        """As ``advance``, the device's counts being advanced already: by a replay of a captured step after its first (which the
        capture itself has counted)."""
        new = self._counts(fresh)
        for b, n in enumerate(new):
            if self.lengths[b] + n > len(self._owned[b]) * self.page_size:
                raise RuntimeError(f"sequence {b} has no pages for {n} more tokens: reserve them first")
        for b, n in enumerate(new):
            self.lengths[b] += n
            self.next_positions[b] += n

    def pages_in_use(self) -> int:
        """Pages of the longest sequence: ``table[:, :pages_in_use()]`` holds all that attention reads."""
        return max(1, max(len(o) for o in self._owned))

    def drop(self, sequence: int) -> None:
        """Forgets a sequence: its pages are free, its next token is its first."""
        check_no_capture(self.table)
        self._free += reversed(self._owned[sequence])
        self._owned[sequence] = []
        self.lengths[sequence] = self.next_positions[sequence] = 0
        self.cached[sequence].zero_()
        self.positions[sequence].zero_()
        self._write_table()

    def check_budget(self, budget: int, recent: int) -> None:
        """Raises where ``evict`` could not go by them."""
        if self.weights is None:
            raise RuntimeError("evict goes by the attention that tokens received: PagedCache(weights=True)")
        if budget < 1 or not 0 <= recent <= budget:
            raise ValueError(f"budget {budget} and recent {recent} must be budget >= 1 and 0 <= recent <= budget")

    def evict(self, ops, budget: int, recent: int = 0) -> list:
        """Brings every sequence of more than ``budget`` tokens back to ``budget``: the last ``recent`` ones and, of each
        layer's key / value head, those that received most attention.  They move into free pages; the old ones are free
        afterwards.  Returns, for each layer, the places kept (``evict_cached_tokens``), or nothing where none was too long."""
        self.check_budget(budget, recent)
        long = [b for b, n in enumerate(self.lengths) if n > budget]
        if not long:
            return []
        per = -(-budget // self.page_size)
        if per * len(long) > len(self._free):
            raise RuntimeError(f"{per * len(long)} pages are needed and {len(self._free)} of {self.pages} are free")
        # (taken and given back once all layers have moved: a call that raises leaves the cache as it was)
        free, owned = list(self._free), [list(o) for o in self._owned]
        for b in long:
            owned[b] = [free.pop() for _ in range(per)]
        new = torch.full((self.batch, per), -1, dtype=torch.int32)
        for b, o in enumerate(owned):
            new[b, :min(per, len(o))] = torch.tensor(o[:per], dtype=torch.int32)
        new = send(new, self.table)
        kept = [ops.evict_cached_tokens(self.k[i], self.v[i], self.weights[i], self.table, self.cached, new, budget, recent)
                for i in range(self.k.size(0))]
        for b in long:
            free += reversed(self._owned[b])
            self.lengths[b] = budget
        self._free, self._owned = free, owned
        self._write_table()
        self.cached.copy_(kept[0][1])
        return [k for k, _ in kept]
