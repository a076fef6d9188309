"""The cache: a slot for each live sequence, storage for each run of a layer.

Storage is paged: a page holds 64 consecutive positions of one run's keys (or
values) for all kv heads, ``[kv_heads, 64, head_dim]``, and a sequence's slot
owns a row of a page table that maps position // 64 to a page. Kernels read the
table on the device, so a sequence's positions need not be contiguous and the
cache is sized by tokens in flight, not by slots x longest sequence. (The
reference keeps ``[layers, batch, kv_heads, capacity, head_dim]`` with the batch
row as the slot and a capacity fixed per plan: engine/model.py:223,231-234 of
willzeng274/kernel-rush-kawk.)

Runs whose needs differ get storage groups of their own: runs that keep every
key share one group, runs that keep a window of W keys another, whose slots cycle
through a ring of pages, position p living in ring entry (p // 64) % ring. Each
kind of fixed-size per-sequence state is a group too: ``[runs, slots, *shape]``,
zeroed when the slot is handed out.

Pages are not cleared when a slot is given back: every read is bounded by the
sequence's length, as in the reference, whose reset is ``pos.zero_()`` (:290).

Sequences that begin alike may share the pages of their first positions (``fork``): full pages
only, which nobody writes again. A step's attention reads them once for all neighbours in it.

With a ``KeyEviction`` the cache counts, for every key, the attention weight that it has received, and ``evict`` gives
up the keys that received least; a row's place in the cache and its position in the sequence then differ by what
the sequence has given up (``evicted``).
"""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from ..parts.base import KVNeed, StateNeed
from .allocator import CacheError, FreeList, PageLedger
from .eviction import KeyEviction

PAGE = 64  # positions per page; the attention kernels' key block


@dataclass
class KVView:
    """What a mixer's kernels get: this run's pages and its group's page table."""

    k: torch.Tensor  # [pages, kv_heads, PAGE, head_dim]
    v: torch.Tensor  # [pages, kv_heads, PAGE, v_dim]; v_dim is head_dim unless the need says otherwise
    table: torch.Tensor  # int32 [slots, width] on the device
    width: int  # logical pages per slot; position p is in table[slot, (p // PAGE) % width] (but see keep_pages)
    window: int | None
    kv_heads: int
    head_dim: int
    v_dim: int = 0
    #: the first ``keep_pages`` logical pages hold the sequence's first positions for good; later positions
    #: cycle through the others: page index b = p // PAGE sits in entry b if b < keep_pages, else in entry
    #: keep_pages + (b - keep_pages) % (width - keep_pages)
    keep_pages: int = 0
    #: where keys are evicted: the weight that each row has received (float32 [slots, kv_heads, width * PAGE]), its position in the
    #: sequence (int32, the same shape), and how many of a step's last queries count (None: all)
    scores: torch.Tensor | None = None
    positions: torch.Tensor | None = None
    observe: int | None = None

    def __post_init__(self):
        self.v_dim = self.v_dim or self.head_dim


@dataclass
class StateView:
    state: torch.Tensor  # [slots, *shape]


class _KVGroup:
    def __init__(self, need: KVNeed, runs: list[int], n_pages: int, n_slots: int, width: int, ring: int | None,
                 device, dtype, keep_pages: int = 0, eviction: KeyEviction | None = None):
        self.need = need
        self.runs = runs
        self.width = ring if ring is not None else width
        self.keep_pages = keep_pages if ring is not None else 0
        self.ledger = PageLedger(n_pages, n_slots, self.width, PAGE, ring)
        shape = (len(runs), n_pages, need.kv_heads, PAGE, need.head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        # a group without values of its own hands its keys out as values (one row per position serves as both)
        self.v = self.k if not need.values else torch.zeros(shape[:-1] + (need.v_dim or need.head_dim,), dtype=dtype,
                                                           device=device)
        self.table_host = np.zeros((n_slots, self.width), dtype=np.int32)
        self.table = torch.zeros((n_slots, self.width), dtype=torch.int32, device=device)
        self.scores = self.positions = None
        if eviction is not None:
            if need.window is not None or not need.values:
                raise CacheError("keys can be evicted where a run keeps every key and a value for each")
            counts = (len(runs), n_slots, need.kv_heads, self.width * PAGE)
            self.scores = torch.zeros(counts, dtype=torch.float32, device=device)
            self.positions = torch.zeros(counts, dtype=torch.int32, device=device)
        self.dirty: set[int] = set()

    def bytes(self) -> int:
        counts = 0 if self.scores is None else 8 * self.scores.numel()
        return (self.k.numel() + (self.v.numel() if self.need.values else 0)) * self.k.element_size() + counts


class _StateGroup:
    def __init__(self, need: StateNeed, runs: list[int], n_slots: int, device, dtype):
        self.need = need
        self.runs = runs
        dt = {"float32": torch.float32, "int32": torch.int32}.get(need.dtype, dtype)
        self.state = torch.zeros((len(runs), n_slots) + tuple(need.shape), dtype=dt, device=device)


class SequenceCache:
    """needs: one entry per schedule run: KVNeed, StateNeed, None, ("from", j) for
    a run that reads run j's storage, or a tuple of KVNeed / StateNeed for a run that
    keeps several kinds of storage (its view is then a tuple of views in that order).

    max_tokens: positions all live sequences may hold together, each sequence's
    count rounded up to whole pages. max_slots: live sequences. max_context: the
    longest sequence. step_tokens: the most tokens one sequence brings in one step;
    it sizes the rings of window groups. eviction: count the weight that keys receive, for ``evict``; a slot then has room for
    what it may hold when a pass of ``pass_tokens`` new tokens has come (None: for the longest sequence), within the pool. Sums and positions
    take eight bytes for each row of that room, slot and kv head: a smaller pass makes them smaller."""

    def __init__(self, needs: list, max_tokens: int, max_slots: int, max_context: int, device, dtype,
                 step_tokens: int = 2048, eviction: KeyEviction | None = None, pass_tokens: int | None = None):
        self.eviction = eviction
        self.device = torch.device(device)
        self.dtype = dtype
        self.max_slots = int(max_slots)
        self.max_context = int(max_context)
        self.step_tokens = int(step_tokens)
        self.n_pages = max(1, -(-int(max_tokens) // PAGE))
        rows = self.max_context
        if eviction is not None:  # every row of a slot has a sum and a position beside it: no more rows than the pool has
            rows = min(rows, self.n_pages * PAGE)
            if pass_tokens is not None:
                rows = min(rows, eviction.keep + eviction.every - 1 + int(pass_tokens))
        self.width = max(1, -(-rows // PAGE))
        self.slots = FreeList(self.max_slots, "cache slot")
        self.length = [0] * self.max_slots  # rows held
        self.evicted = [0] * self.max_slots  # rows given up: the next row's position is length + evicted
        self._family: list = [None] * self.max_slots  # (number, shared positions) of slots that share pages with others
        self._families = 0
        self.h2d_bytes = 0  # page-table rows (and their indices) copied to the device so far
        self._kv_groups: list[_KVGroup] = []
        self._state_groups: list[_StateGroup] = []
        self._where: list = [None] * len(needs)  # run -> (group, line), a list of them, or None

        by_need: dict = {}
        several: dict = {}  # run -> its needs, for runs that keep more than one kind of storage
        for run, need in enumerate(needs):
            if isinstance(need, (KVNeed, StateNeed)):
                by_need.setdefault(need, []).append((run, None))
            elif isinstance(need, (tuple, list)) and need and all(isinstance(n, (KVNeed, StateNeed)) for n in need):
                several[run] = list(need)
                self._where[run] = [None] * len(need)
                for k, n in enumerate(need):
                    by_need.setdefault(n, []).append((run, k))
        for need, users in by_need.items():
            runs = [run for run, _ in users]
            if isinstance(need, KVNeed):
                ring = None
                pages = self.n_pages
                keep_pages = 0
                if need.window is not None:
                    keep_pages = -(-max(0, int(need.keep_first)) // PAGE)
                    ring = min(self.width, keep_pages + -(-(need.window + self.step_tokens - 1) // PAGE) + 1)
                    keep_pages = min(keep_pages, ring - 1)  # a context this short never reaches the ring's turn
                    pages = min(self.n_pages, self.max_slots * ring)
                group = _KVGroup(need, runs, pages, self.max_slots, self.width, ring, self.device, dtype, keep_pages,
                                 eviction)
                self._kv_groups.append(group)
            else:
                group = _StateGroup(need, runs, self.max_slots, self.device, dtype)
                self._state_groups.append(group)
            for line, (run, k) in enumerate(users):
                if k is None:
                    self._where[run] = (group, line)
                else:
                    self._where[run][k] = (group, line)
        for run, need in enumerate(needs):
            if isinstance(need, tuple) and need and need[0] == "from":
                src = self._where[need[1]]
                if src is None or isinstance(src, list) or not isinstance(src[0], _KVGroup):
                    raise CacheError(f"run {run} reads the cache of run {need[1]}, which keeps no keys and values")
                self._where[run] = src

    # -- slots --------------------------------------------------------------
    def alloc(self) -> int:
        slot = self.slots.take()
        self.length[slot] = self.evicted[slot] = 0
        self._family[slot] = None
        for g in self._state_groups:
            g.state[:, slot].zero_()
        return slot

    def free(self, slot: int) -> None:
        self.slots.give(slot)  # raises on a slot that is not held
        for g in self._kv_groups:
            g.ledger.release(slot)
        self.length[slot] = self.evicted[slot] = 0
        self._family[slot] = None

    def can_share(self) -> bool:
        """Whether sequences can share pages: no run keeps a window of keys, whose pages are written again, and no keys are evicted."""
        return self.eviction is None and all(g.need.window is None for g in self._kv_groups)

    def fork(self, slot: int, length: int) -> int:
        """A new slot whose sequence begins with the first ``length`` positions of ``slot``'s: it holds the same pages, and copies of the
        fixed-size state. ``length`` is a whole number of pages; where there is state, all that ``slot`` holds (the state of an earlier
        position is gone). Single-token and longer steps read shared pages once for the sequences that stand side by side in them."""
        if not self.slots.is_held(slot):
            raise CacheError(f"cache slot {slot} is not held")
        if not self.can_share():
            raise CacheError("sequences share pages where every run keeps all keys and none are evicted")
        if length < 0 or length % PAGE or length > self.length[slot]:
            raise CacheError(f"a fork shares whole pages of {PAGE} positions that its source holds; got {length} of {self.length[slot]}")
        if self._state_groups and length != self.length[slot]:
            raise CacheError(f"the state behind position {length} is gone: the sequence is at {self.length[slot]}")
        new = self.alloc()
        for g in self._kv_groups:
            for logical, page in g.ledger.share(slot, new, length // PAGE):
                g.table_host[new, logical] = page
            g.dirty.add(new)
        for g in self._state_groups:
            g.state[:, new].copy_(g.state[:, slot])
        self.length[new] = length
        if length:
            if self._family[slot] is None:
                self._families += 1
                self._family[slot] = (self._families, length)
            if length >= self._family[slot][1]:  # a fork of less than the family shares has none
                self._family[new] = self._family[slot]
        return new

    @property
    def has_forks(self) -> bool:
        return self._families > 0

    def shared_groups(self, slots) -> tuple[list, list]:
        """(sizes, shared positions) of the neighbours among ``slots`` that share pages, in order; a slot alone shares 0."""
        sizes, lengths, last = [], [], None
        for s in slots:
            family = self._family[s]
            if family is not None and family == last:
                sizes[-1] += 1
                lengths[-1] = family[1]
            else:
                sizes.append(1)
                lengths.append(0)
            last = family
        return sizes, lengths

    # -- eviction -------------------------------------------------------------
    def evict_due(self, slot: int) -> bool:
        """Whether the slot holds so many rows that some go before its next step."""
        return self.eviction is not None and self.length[slot] >= self.eviction.keep + self.eviction.every

    def evict(self, ops, slots, batch=None) -> None:
        """Give up all but ``eviction.keep`` rows of those of ``slots`` that are due. ``batch``: a single-token step of exactly these slots,
        whose description follows on the device."""
        keep = self.eviction.keep
        due = [self.evict_due(s) for s in slots]
        if not any(due):
            return
        if batch is None:
            slots, due = [s for s, d in zip(slots, due) if d], [True] * sum(due)
        lengths = [self.length[s] if d else min(self.length[s], keep) for s, d in zip(slots, due)]
        for i, g in enumerate(self._kv_groups):
            ops.evict_keys(g.k, g.v, g.table, slots, lengths, g.scores, g.positions, keep, self.eviction.recent, batch=None if i else batch)
        for s, d in zip(slots, due):
            if d:
                self.evicted[s] += self.length[s] - keep
                self.length[s] = keep
                for g in self._kv_groups:
                    g.ledger.shrink(s, keep)

    def reserve(self, slot: int, length: int) -> None:
        """Make room for ``slot`` to hold ``length`` positions."""
        if not self.slots.is_held(slot):
            raise CacheError(f"cache slot {slot} is not held")
        if length + self.evicted[slot] > self.max_context:
            length += self.evicted[slot]
            raise CacheError(f"a sequence of {length} tokens exceeds the longest the cache was built for ({self.max_context})")
        for g in self._kv_groups:
            if not g.ledger.can_grow(slot, length):
                g.ledger.grow(slot, length)  # raises with the numbers
        for g in self._kv_groups:
            for logical, page in g.ledger.grow(slot, length):
                g.table_host[slot, logical] = page
                g.dirty.add(slot)

    def advance(self, slot: int, n: int) -> None:
        self.length[slot] += n

    def sync(self) -> None:
        """Bring the device's page tables up to date (rows that changed)."""
        for g in self._kv_groups:
            if not g.dirty:
                continue
            rows = sorted(g.dirty)
            idx = torch.as_tensor(rows, dtype=torch.int64, device=self.device)
            g.table.index_copy_(0, idx, torch.from_numpy(g.table_host[rows]).to(self.device))
            self.h2d_bytes += len(rows) * (8 + 4 * g.width)
            g.dirty.clear()

    def _per_slot(self) -> list:
        """What a second run of the same step would change: fixed-size state, and the weights that keys have received."""
        return [g.state for g in self._state_groups] + [g.scores for g in self._kv_groups if g.scores is not None]

    def save_state(self, slots) -> list:
        """Copies of the fixed-size state that these slots hold, one tensor per state group (then of their keys' received weights)."""
        idx = torch.as_tensor(list(slots), dtype=torch.int64, device=self.device)
        return [t.index_select(1, idx) for t in self._per_slot()]

    def restore_state(self, slots, saved: list) -> None:
        idx = torch.as_tensor(list(slots), dtype=torch.int64, device=self.device)
        for t, s in zip(self._per_slot(), saved):
            t.index_copy_(1, idx, s)

    def per_sequence_step_limit(self) -> int | None:
        """The most tokens one sequence may bring in one pass, or None if any number will do. A group that
        keeps a window of keys cycles through a ring of pages sized for ``step_tokens`` new positions;
        a longer pass would overwrite keys that its own first rows still have to read."""
        if any(g.need.window is not None for g in self._kv_groups):
            return self.step_tokens
        return None

    # -- views --------------------------------------------------------------
    def view(self, run: int):
        where = self._where[run]
        if where is None:
            return None
        if isinstance(where, list):
            return tuple(self._view_of(group, line) for group, line in where)
        return self._view_of(*where)

    def _view_of(self, group, line):
        if isinstance(group, _KVGroup):
            view = KVView(group.k[line], group.v[line], group.table, group.width, group.need.window,
                          group.need.kv_heads, group.need.head_dim, group.need.v_dim or group.need.head_dim,
                          group.keep_pages)
            if group.scores is not None:
                view.scores, view.positions, view.observe = group.scores[line], group.positions[line], self.eviction.observe
            return view
        return StateView(group.state[line])

    # -- accounting ---------------------------------------------------------
    @property
    def live(self) -> int:
        return self.slots.held

    def free_pages(self) -> int:
        return min((len(g.ledger.pool) for g in self._kv_groups), default=0)

    def row_bytes(self) -> int:
        """Bytes of one position's keys and values in one layer (the largest)."""
        return max((g.need.kv_heads * (g.need.head_dim + (g.need.v_dim or g.need.head_dim)) * g.k.element_size() for g in self._kv_groups), default=0)

    def bytes(self) -> int:
        return sum(g.bytes() for g in self._kv_groups) + sum(
            g.state.numel() * g.state.element_size() for g in self._state_groups)

    def check(self) -> None:
        """Raise if a slot or page is lost or held twice."""
        self.slots.check()
        for g in self._kv_groups:
            g.ledger.check()
            for slot in range(self.max_slots):
                if not self.slots.is_held(slot) and g.ledger.pages[slot]:
                    raise CacheError(f"slot {slot} is free but still holds pages")
