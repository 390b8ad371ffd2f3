"""A paged cache of keys, values and newest queries, for generating one token at a time.

The attention modules compute whole sequences; ``decode(cache)`` of either module
(``MTAAttentionTriton``, ``TritonConvAttention``) computes the row of the newest token of
every sequence in a cache.  A sequence lives in a *slot*.  Its keys and values lie in pages of
``page_size`` positions that a table per slot lists, so that sequences grow without moving
and share what they have in common; its newest ``query_rows`` queries lie in a ring, because
the convs of these modules reach back over query rows (``module.decode_query_rows`` of them).

A step::

    cache.extend(1)                    # every slot gets one more position (host: pages, table)
    cache.append(xq, xk, xv)           # (slots, heads, 1, D): into the pages
    out = module.decode(cache)

``extend`` takes a count per slot: prompts of any length, 0 for slots that sit the step out
(their rows of ``out`` are zeros).  Bookkeeping is on the host, in plain Python; what kernels
read of it - the table and two numbers per slot - is copied to the device on the current stream.
The kernels never wait for the host, and a step may be captured into a graph (``append`` and
``decode``; not ``extend``, which is called between replays: the graph reads the table anew every time
and has to be captured with as many new tokens as a slot gets at most; ``mark_appended`` tells the host of a replay).  All calls on one cache
belong on one stream, or are ordered by the caller.
"""
from __future__ import annotations

import heapq
from typing import List, Optional, Sequence, Union

import torch

from . import _lib, ops


class PagedCache:
    """``n_slots`` sequences over ``n_pages`` pages.  ``k``, ``v``: (n_pages, kv_heads, page_size, head_dim); ``q``:
    (n_slots, n_heads, query_rows, head_dim), the query of position i in row i % query_rows; ``table``: int32
    (n_slots, max_pages) and ``state``: int32 (2, n_slots) - tokens before the last ``extend``, tokens it added - on the
    device.  Query head h reads key head h // (n_heads // kv_heads)."""

    def __init__(self, n_slots: int, n_pages: int, n_heads: int, head_dim: int, kv_heads: Optional[int] = None, page_size: int = 64,
                 max_pages: Optional[int] = None, query_rows: int = 1, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        kv_heads = n_heads if kv_heads is None else kv_heads
        max_pages = n_pages if max_pages is None else max_pages
        self._check_sizes(n_slots, n_pages, n_heads, head_dim, kv_heads, page_size, max_pages, query_rows, dtype)
        pool = (n_pages, kv_heads, page_size, head_dim)
        self._take(torch.empty(pool, dtype=dtype, device=device), torch.empty(pool, dtype=dtype, device=device),
                   torch.empty((n_slots, n_heads, query_rows, head_dim), dtype=dtype, device=device), max_pages)

    @staticmethod
    def _check_sizes(n_slots, n_pages, n_heads, head_dim, kv_heads, page_size, max_pages, query_rows, dtype):
        for name, value in (("n_slots", n_slots), ("n_pages", n_pages), ("n_heads", n_heads), ("kv_heads", kv_heads), ("max_pages", max_pages),
                            ("query_rows", query_rows)):
            if not isinstance(value, int) or value <= 0:
                raise ValueError(f"{name} must be a positive number, got {value!r}")
        if n_heads % kv_heads:
            raise ValueError(f"kv_heads={kv_heads} does not divide n_heads={n_heads}")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if n_slots > 65535 or n_heads > 4096 or query_rows > 65535 or n_pages >= 2 ** 31 or max_pages * page_size > 2 ** 30:
            raise ValueError("a cache has at most 65535 slots, 4096 heads, 65535 query rows and 2**30 positions per slot")
        if dtype not in ops._DTYPE_CODE:
            raise TypeError(f"cache: dtype {dtype} is not supported (float32, bfloat16, float16)")

    def _take(self, k, v, q, max_pages: int) -> None:
        self.k, self.v, self.q = k, v, q
        n = q.size(0)
        # what the kernels read of the bookkeeping, in one buffer: state, then table
        self._plan = torch.full((n * (2 + max_pages),), -1, dtype=torch.int32, device=k.device)
        self._plan[:2 * n] = 0
        self.state, self.table = self._plan[:2 * n].view(2, n), self._plan[2 * n:].view(n, max_pages)
        self._host = self._plan.cpu()
        self._host_state, self._host_table = self._host[:2 * n].view(2, n), self._host[2 * n:].view(n, max_pages)
        self._lengths, self._added = [0] * n, [0] * n
        self._due = False          # the tokens of the last extend are in no page yet, as far as the host knows
        self._shared = False       # ... are in pages that a fork has shared since
        self._pages: List[List[int]] = [[] for _ in range(n)]
        self._uses = [0] * k.size(0)
        self._free = list(range(k.size(0)))    # a heap: the lowest page first

    @classmethod
    def adopt(cls, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor, table, lengths: Sequence[int], added: Optional[Sequence[int]] = None) -> "PagedCache":
        """A cache over pools and a ring that are filled already (a restored checkpoint, another process's pages); the tensors
        are used, not copied.  ``table``: (slots, max_pages) page numbers; ``lengths``: tokens per slot, ``added`` of
        them new (default: the newest one), as after ``extend``.  Slots may share pages that lie wholly ahead of
        their new tokens."""
        if k.dim() != 4 or q.dim() != 4 or k.shape != v.shape or k.size(3) != q.size(3) or not k.dtype == v.dtype == q.dtype or not k.device == v.device == q.device:
            raise ValueError("k and v are (pages, key heads, rows, D), q (slots, heads, rows, D), of one dtype and device")
        if not (k.is_contiguous() and v.is_contiguous() and q.is_contiguous()):
            raise ValueError("the tensors of a cache are contiguous")
        table = torch.as_tensor(table).cpu()
        lengths = [int(n) for n in lengths]
        added = [min(n, 1) for n in lengths] if added is None else [int(n) for n in added]
        if table.dim() != 2 or table.size(0) != q.size(0) or len(lengths) != q.size(0) or len(added) != q.size(0):
            raise ValueError(f"table, lengths and added have a row for each of {q.size(0)} slots")
        cls._check_sizes(q.size(0), k.size(0), q.size(1), k.size(3), k.size(1), k.size(2), table.size(1), q.size(2), k.dtype)
        cache, page = cls.__new__(cls), k.size(2)
        cache._take(k, v, q, table.size(1))
        own = [0] * k.size(0)      # slots that write into a page
        for slot, (n, new) in enumerate(zip(lengths, added)):
            need = -(-n // page)
            if not 0 <= new <= n or need > table.size(1):
                raise ValueError(f"slot {slot}: {n} tokens, {new} of them new, do not fit {table.size(1)} pages of {page}")
            pages = table[slot, :need].tolist()
            if any(not 0 <= p < k.size(0) for p in pages) or len(set(pages)) < need:
                raise ValueError(f"slot {slot}: its pages are not {need} different ones of 0 .. {k.size(0) - 1}")
            for i, p in enumerate(pages):
                cache._uses[p] += 1
                own[p] += (i + 1) * page > n - new
            cache._lengths[slot], cache._added[slot], cache._pages[slot] = n, new, pages
        if any(o and u > 1 for o, u in zip(own, cache._uses)):
            raise ValueError("a page with new tokens, or with room for more, belongs to several slots")
        cache._free = [p for p, u in enumerate(cache._uses) if u == 0]
        need = torch.tensor([len(pages) for pages in cache._pages])
        cache._host_table.copy_(torch.where(torch.arange(table.size(1)) < need[:, None], table, -1))
        cache._upload(everything=True)
        return cache

    # ------------------------------------------------------------------ bookkeeping
    @property
    def n_slots(self) -> int:
        return self.q.size(0)

    @property
    def page_size(self) -> int:
        return self.k.size(2)

    @property
    def lengths(self) -> List[int]:
        """Tokens per slot, the new ones included."""
        return list(self._lengths)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages_of(self, slot: int) -> List[int]:
        return list(self._pages[self._slot(slot)])

    @property
    def longest(self) -> int:
        """What sizes a decode: the longest slot; while a graph is captured, what the table has room for (``max_pages`` pages, which also
        size the workspace of ``MTAAttentionTriton.decode``; beyond 2**23 positions that is refused)."""
        if self._capturing():
            return self.table.size(1) * self.page_size
        return max(1, max(self._lengths))

    def _slot(self, slot: int) -> int:
        if not isinstance(slot, int) or not 0 <= slot < self.n_slots:
            raise ValueError(f"a slot is a number from 0 to {self.n_slots - 1}, got {slot!r}")
        return slot

    def _capturing(self) -> bool:
        """Whether the calls go into a graph: on the cache's device, where the work is queued, whatever the current one is."""
        if not self.k.is_cuda:
            return False
        if torch.cuda.current_device() == self.k.device.index:   # (as nearly always, and a switch costs microseconds)
            return torch.cuda.is_current_stream_capturing()
        with torch.cuda.device(self.k.device):
            return torch.cuda.is_current_stream_capturing()

    def _eager(self, what: str) -> None:
        if self._capturing():
            raise RuntimeError(f"{what} is host bookkeeping and cannot be captured into a graph: call it between replays")

    def _upload(self, slots=(), everything: bool = False) -> None:
        """State, and the rows of the table of ``slots`` (``everything``: the table as it is), to the device."""
        n = self.n_slots
        self._host_state[0] = torch.tensor([have - new for have, new in zip(self._lengths, self._added)], dtype=torch.int32)
        self._host_state[1] = torch.tensor(self._added, dtype=torch.int32)
        for slot in slots:
            row = self._host_table[slot]
            row.fill_(-1)
            row[:len(self._pages[slot])] = torch.tensor(self._pages[slot], dtype=torch.int32)
        count = self._host.numel() if everything or len(slots) else 2 * n
        if self.k.is_cuda:
            # (a pinned copy of its own: the mirror may change before the stream gets there)
            with torch.cuda.device(self.k.device):
                self._plan[:count].copy_(self._host[:count].pin_memory(), non_blocking=True)
        else:
            self._plan[:count] = self._host[:count]

    def _release(self, slot: int) -> None:
        for page in self._pages[slot]:
            self._uses[page] -= 1
            if self._uses[page] == 0:
                heapq.heappush(self._free, page)
        self._pages[slot], self._lengths[slot], self._added[slot] = [], 0, 0

    def extend(self, counts: Union[int, Sequence[int]]) -> None:
        """``counts`` more positions for every slot (a number, or one per slot; 0: the slot sits the next steps out).  ``append`` fills
        those of the last call only, so it comes before the next one.  Raises, and changes nothing, where pages or the table run out."""
        self._eager("extend")
        counts = [counts] * self.n_slots if isinstance(counts, int) else [int(c) for c in counts]
        if len(counts) != self.n_slots or any(c < 0 for c in counts):
            raise ValueError(f"extend takes a number of tokens, or one for each of {self.n_slots} slots, got {counts}")
        page, want = self.page_size, []
        for slot, c in enumerate(counts):
            need = -(-(self._lengths[slot] + c) // page)
            if need > self.table.size(1):
                raise RuntimeError(f"slot {slot}: {self._lengths[slot] + c} tokens do not fit {self.table.size(1)} pages of {page}")
            want.append(need - len(self._pages[slot]))
        if sum(want) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {sum(want)} are needed")
        for slot, c in enumerate(counts):
            for _ in range(want[slot]):
                p = heapq.heappop(self._free)
                self._uses[p] = 1
                self._pages[slot].append(p)
            self._lengths[slot] += c
            self._added[slot] = c
        self._due, self._shared = True, False
        self._upload([slot for slot, w in enumerate(want) if w])

    def free(self, slot: int) -> None:
        """Empties a slot; pages that no other slot shares are free again."""
        self._eager("free")
        self._release(self._slot(slot))
        self._upload([slot])

    # ------------------------------------------------------------------ device
    def append(self, xq: torch.Tensor, xk: torch.Tensor, xv: torch.Tensor) -> None:
        """The tokens of the last ``extend``: (slots, n_heads, n, D) queries, (slots, kv_heads, n, D) keys and values, any strides
        with contiguous rows; slot b takes its first ``added[b]`` tokens, n is at least the most of them.  One kernel
        (``mta_cache_append``)."""
        if self._shared and not self._capturing():
            raise RuntimeError("the tokens of the last extend lie in pages that are shared since a fork: extend before the next append")
        if xk.dim() == 4 and xk.size(2) < max(self._added):
            raise ValueError(f"extend made room for up to {max(self._added)} tokens, append got {xk.size(2)}")
        _lib.host().cache_append(self.k, self.v, self.q, self.table, self.state, xq, xk, xv)
        if self._due and not self._capturing():
            self._due = False

    def mark_appended(self) -> None:
        """Says that the tokens of the last ``extend`` are in their pages: after the replay of a graph that appends them, which the
        host does not see, or where something else wrote them.  ``append`` says so by itself."""
        self._due = False

    def fork(self, source: int, targets: Union[int, Sequence[int]]) -> None:
        """Makes ``targets`` copies of slot ``source`` (a beam that splits, samples of one prompt): whole pages are shared, the page
        that is being filled and the ring of queries are copied.  What the targets held is released.  They sit steps out
        until they are extended.  The source's tokens have to be in their pages: between ``extend`` and ``append`` a fork is
        refused (``mark_appended``, where a replayed graph appended them), and what is appended behind it, by a call or by a
        replay, is the tokens of a later ``extend``."""
        self._eager("fork")
        targets = [targets] if isinstance(targets, int) else list(targets)
        for slot in [source] + targets:
            self._slot(slot)
        if source in targets or len(set(targets)) < len(targets):
            raise ValueError(f"fork takes different targets, and none that is the source: {source} to {targets}")
        if targets and self._due and self._added[source]:
            # (their copies would be taken now, and the append to come writes the source's pages alone)
            raise RuntimeError(f"slot {source} holds {self._added[source]} tokens that have not been appended yet: append them before a fork"
                               + ("" if self.k.is_cuda else f" (the cache lives on {self.k.device}: append has no CPU path)"))
        n, page = self._lengths[source], self.page_size
        whole = n // page
        shared, partial = self._pages[source][:whole], self._pages[source][whole:]
        going = {}
        for slot in targets:
            for p in self._pages[slot]:
                going[p] = going.get(p, 0) + 1
        freed = sum(1 for p, times in going.items() if times == self._uses[p])
        if len(partial) * len(targets) > len(self._free) + freed:
            raise RuntimeError(f"the cache has {len(self._free) + freed} free pages, {len(partial) * len(targets)} are needed")
        if partial and targets and not self.k.is_cuda:
            raise RuntimeError(f"the cache lives on {self.k.device}: pages are copied on an AMD GPU only (there is no CPU path)")
        for slot in targets:
            self._release(slot)
        pairs = []
        for slot in targets:
            copies = [heapq.heappop(self._free) for _ in partial]
            for p in shared + copies:
                self._uses[p] += 1
            pairs += list(zip(partial, copies))
            self._pages[slot], self._lengths[slot], self._added[slot] = shared + copies, n, 0
        if targets and whole * page > n - self._added[source]:
            self._shared = True
        self._upload(targets)
        if pairs:
            ops.cache_copy_pages(self.k, self.v, pairs)
        for slot in targets if n else ():
            self.q[slot].copy_(self.q[source])

    def compact(self) -> int:
        """Moves pages so that those in use are the lowest ones; returns how many they are (``k[:n]`` and ``v[:n]`` then hold
        everything there is to save)."""
        self._eager("compact")
        used = sum(1 for u in self._uses if u)
        holes = [p for p in range(used) if not self._uses[p]]
        high = [p for p in range(used, len(self._uses)) if self._uses[p]]
        moves = dict(zip(high, holes))
        if moves:
            ops.cache_copy_pages(self.k, self.v, list(moves.items()))
            for old, new in moves.items():
                self._uses[new], self._uses[old] = self._uses[old], 0
            changed = [slot for slot, pages in enumerate(self._pages) if any(p in moves for p in pages)]
            for slot in changed:
                self._pages[slot] = [moves.get(p, p) for p in self._pages[slot]]
            self._free = list(range(used, len(self._uses)))
            self._upload(changed)
        return used


__all__ = ["PagedCache"]
