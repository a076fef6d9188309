"""Host-side bookkeeping of the cache: who holds which slot and which pages.

Pure Python, no tensors: the tests of "no slot lost, held twice or freed twice"
run on these classes alone. The reference has nothing of the kind: its batch
row is the slot, fixed for a plan, and "reset" is ``pos.zero_()``
(engine/model.py:231-234,290 of willzeng274/kernel-rush-kawk).
"""

from __future__ import annotations


class CacheError(RuntimeError):
    """No free slot or page, a slot used that is not held, or a sequence longer
    than the cache was built for."""


class FreeList:
    """Integers 0..n-1, handed out and taken back. Last freed, first reused, so that
    reuse is exercised at once rather than after a full cycle."""

    def __init__(self, n: int, what: str):
        self.n = n
        self.what = what
        self._free = list(range(n - 1, -1, -1))
        self._held = [False] * n

    def __len__(self) -> int:
        return len(self._free)

    @property
    def held(self) -> int:
        return self.n - len(self._free)

    def take(self) -> int:
        if not self._free:
            raise CacheError(f"no free {self.what}: all {self.n} are held")
        i = self._free.pop()
        self._held[i] = True
        return i

    def give(self, i: int) -> None:
        if not 0 <= i < self.n:
            raise CacheError(f"{self.what} {i} does not exist (there are {self.n})")
        if not self._held[i]:
            raise CacheError(f"{self.what} {i} is freed twice, or was never handed out")
        self._held[i] = False
        self._free.append(i)

    def is_held(self, i: int) -> bool:
        return 0 <= i < self.n and self._held[i]

    def check(self) -> None:
        """Every index is either free exactly once or held; raises otherwise."""
        seen = set(self._free)
        if len(seen) != len(self._free):
            raise CacheError(f"a {self.what} sits in the free list twice")
        for i in range(self.n):
            if self._held[i] == (i in seen):
                raise CacheError(f"{self.what} {i} is {'both held and free' if self._held[i] else 'lost'}")


class PageLedger:
    """Pages of one storage group: a pool and, per slot, the pages it holds in
    logical order. ``ring`` is None for a group that keeps every position, or the
    number of logical pages a slot holds at most for a group that keeps a window (the
    pages of positions that are kept for good come first and count among them).
    A page may be held by several slots (``share``); it goes back to the pool with the last of them."""

    def __init__(self, n_pages: int, n_slots: int, width: int, page_size: int, ring: int | None):
        self.pool = FreeList(n_pages, "cache page")
        self.pages: list[list[int]] = [[] for _ in range(n_slots)]
        self.width = width
        self.page_size = page_size
        self.ring = ring
        self.holders: dict[int, int] = {}  # page -> slots that hold it, where these are more than one

    def pages_for(self, length: int) -> int:
        need = -(-length // self.page_size)
        return min(need, self.ring) if self.ring is not None else need

    def can_grow(self, slot: int, length: int) -> bool:
        return self.pages_for(length) - len(self.pages[slot]) <= len(self.pool)

    def grow(self, slot: int, length: int) -> list[tuple[int, int]]:
        """Make ``slot`` hold pages for ``length`` tokens; returns the new (logical
        index, page) pairs."""
        need = self.pages_for(length)
        if need > self.width:
            raise CacheError(f"a sequence of {length} tokens needs {need} pages; the cache was built for {self.width} "
                             f"({self.width * self.page_size} tokens a sequence)")
        have = self.pages[slot]
        if need - len(have) > len(self.pool):
            raise CacheError(f"the cache is full: {need - len(have)} more pages of {self.page_size} tokens are needed, "
                             f"{len(self.pool)} of {self.pool.n} are free")
        new = []
        while len(have) < need:
            page = self.pool.take()
            new.append((len(have), page))
            have.append(page)
        return new

    def share(self, source: int, slot: int, n_pages: int) -> list[tuple[int, int]]:
        """``slot``, which holds none yet, takes the first ``n_pages`` pages of ``source`` as its own first ones;
        returns the (logical index, page) pairs."""
        if self.ring is not None:
            raise CacheError("pages that a window cycles through cannot be shared")
        if self.pages[slot] or n_pages > len(self.pages[source]):
            raise CacheError(f"a slot with {len(self.pages[slot])} pages cannot share {n_pages} of the {len(self.pages[source])} that another holds")
        self.pages[slot] = self.pages[source][:n_pages]
        for page in self.pages[slot]:
            self.holders[page] = self.holders.get(page, 1) + 1
        return list(enumerate(self.pages[slot]))

    def _give(self, page: int) -> None:
        n = self.holders.pop(page, 1) - 1
        if n == 0:
            self.pool.give(page)
        elif n > 1:
            self.holders[page] = n

    def shrink(self, slot: int, length: int) -> None:
        """Give back the pages behind those that ``length`` positions need."""
        need = self.pages_for(length)
        for page in self.pages[slot][need:]:
            self._give(page)
        del self.pages[slot][need:]

    def release(self, slot: int) -> None:
        for page in self.pages[slot]:
            self._give(page)
        self.pages[slot] = []

    def check(self) -> None:
        self.pool.check()
        count: dict[int, int] = {}
        for pages in self.pages:
            for p in pages:
                count[p] = count.get(p, 0) + 1
        for page, n in count.items():
            if n != self.holders.get(page, 1):
                raise CacheError(f"a cache page is held by two slots or more: by {n}, where {self.holders.get(page, 1)} share it")
        if any(page not in count for page in self.holders):
            raise CacheError("a shared cache page is held by no slot")
        if len(count) != self.pool.held:
            raise CacheError(f"{self.pool.held} pages are handed out but slots hold {len(count)}")
