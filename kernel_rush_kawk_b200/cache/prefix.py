"""Which sequences of a step hold the same first positions in the same pages.

``SequenceCache.fork`` makes such sequences: the fork's page table begins with the pages of the sequence it comes from.
``Kernels.shared_prefix_attention`` takes a step's groups and reads what a group shares once for all of its rows.
"""

from __future__ import annotations

import torch

from .allocator import CacheError
from .store import PAGE


class PrefixGroups:
    """``sizes``: how many neighbouring sequences of the step form each group, in the step's order (one: a sequence alone).
    ``lengths``: the first positions that a group's sequences share, whole pages, 0 for none.

    On the device: cu[g], the first sequence of group g (cu[groups]: their number); length[g]; group[s], the group of
    sequence s. Views of one buffer, filled by a single copy."""

    def __init__(self, sizes, lengths, device):
        sizes, lengths = [int(n) for n in sizes], [int(n) for n in lengths]
        if len(sizes) != len(lengths) or not sizes:
            raise CacheError(f"{len(sizes)} groups of sequences with {len(lengths)} shared lengths")
        for size, length in zip(sizes, lengths):
            if size < 1:
                raise CacheError(f"a group has at least one sequence, got {size}")
            if length < 0 or length % PAGE:
                raise CacheError(f"sequences share whole pages of {PAGE} positions, got {length}")
        self.sizes, self.lengths = tuple(sizes), tuple(lengths)
        self.n_groups, self.n_seqs = len(sizes), sum(sizes)
        self.max_seqs, self.max_length = max(sizes), max(lengths)
        cu = [0]
        for size in sizes:
            cu.append(cu[-1] + size)
        host = cu + lengths + [g for g, size in enumerate(sizes) for _ in range(size)]
        self.buffer = torch.tensor(host, dtype=torch.int32).to(device)
        n = self.n_groups
        self.cu, self.length, self.group = self.buffer[:n + 1], self.buffer[n + 1:2 * n + 1], self.buffer[2 * n + 1:]

    @staticmethod
    def shape_of(sizes, lengths) -> tuple:
        """What a captured step of such groups depends on, beside their number of sequences."""
        return (len(sizes), max(sizes), max(lengths) > 0)

    @property
    def shape(self) -> tuple:
        return self.shape_of(self.sizes, self.lengths)

    def update(self, other: "PrefixGroups") -> None:
        """Take another object's sizes and lengths, in the same device buffer (a captured step goes on reading it)."""
        if (other.shape, other.n_seqs) != (self.shape, self.n_seqs):
            raise CacheError(f"groups of shape {other.shape} over {other.n_seqs} sequences do not fit a step captured for {self.shape} over {self.n_seqs}")
        self.buffer.copy_(other.buffer)
        self.sizes, self.lengths, self.max_length = other.sizes, other.lengths, other.max_length

    def max_rows(self, batch) -> int:
        """The most rows of a step that one group has."""
        if batch.max_q_len == 1:
            return self.max_seqs
        at, most = 0, 0
        for size in self.sizes:
            most = max(most, sum(batch.q_lens[at:at + size]))
            at += size
        return most

    def check(self, batch, cache) -> None:
        """Raise unless the step's sequences are these and lie behind their prefixes."""
        if batch.n_seqs != self.n_seqs:
            raise CacheError(f"groups of {self.n_seqs} sequences for a step of {batch.n_seqs}")
        if self.max_length > cache.width * PAGE:
            raise CacheError(f"a shared prefix of {self.max_length} positions exceeds a slot's {cache.width * PAGE}")
        if min(batch.starts) < self.max_length:
            at = 0
            for size, length in zip(self.sizes, self.lengths):
                first = min(batch.starts[at:at + size])
                if first < length:
                    raise CacheError(f"a sequence that holds {first} positions shares none of a prefix of {length}")
                at += size
