"""Slots, pages and per-sequence state."""

from .allocator import CacheError, FreeList, PageLedger
from .eviction import KeyEviction
from .prefix import PrefixGroups
from .store import PAGE, KVView, SequenceCache, StateView

__all__ = ["CacheError", "FreeList", "KeyEviction", "PageLedger", "PAGE", "PrefixGroups", "KVView", "SequenceCache", "StateView"]
