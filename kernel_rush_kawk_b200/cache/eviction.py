"""How much of a sequence's cache is kept when keys are evicted by the attention weight that they have received."""

from __future__ import annotations

from dataclasses import dataclass

from .allocator import CacheError


@dataclass(frozen=True)
class KeyEviction:
    """Every kv head of every layer holds at most ``keep + every`` keys of a sequence between its steps: a sequence that holds so many
    falls back to ``keep`` before its next step, to its ``recent`` newest keys and those that received most weight. A step may bring any
    number of tokens, and its queries see all keys that were held before it (one that is cut into passes falls back between them, too).
    ``observe``: of a step's queries of a sequence, the last so many count (None: all)."""

    keep: int
    recent: int = 0
    every: int = 64
    observe: int | None = None

    def __post_init__(self):
        if self.keep < 1 or not 0 <= self.recent <= self.keep:
            raise CacheError(f"at least one key stays, and at most as many by position as stay in all; got keep {self.keep}, recent {self.recent}")
        if self.every < 1 or (self.observe is not None and self.observe < 1):
            raise CacheError(f"an eviction comes after one new key or more, and counts one query or more; got every {self.every}, observe {self.observe}")
