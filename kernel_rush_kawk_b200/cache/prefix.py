"""Which sequences of a step hold the same first positions in the same pages.

``SequenceCache.fork`` makes such sequences: the fork's page table begins with the pages of the sequence it comes from.
``Kernels.shared_prefix_attention`` takes a step's groups and reads what a group shares once for all of its rows.
"""

from __future__ import annotations

import torch

from .allocator import CacheError
from .store import PAGE


# Where reading a prefix once pays. It takes a launch more, and parts of the softmax that have to join, so that what a step does not read again
# has to be worth these.
#
# Single tokens, by the bytes of keys and values of one layer that are not read again: 9 MB a sequence, up to eight of them. A layer's attention with
# rotation and cache write in replayed steps, us, each sequence by itself and shared, 32 heads over 8 of 128 with 100 keys of their own: 2 sequences behind 4,096
# positions (17 MB) 14.3 and 17.4, 8,192 23.0 and 20.1; 4 behind 2,048 (25 MB) 15.8 and 15.5, 4,096 21.7 and 17.4; 8 behind 2,048 (59 MB) 15.5 and 16.7,
# 4,096 24.3 and 19.8; 16 behind 1,024 (63 MB) 16.4 and 19.2, 2,048 24.8 and 19.8; 64 behind 256 (66 MB) 23.3 and 23.4, 1,024 48.0 and 26.4, 8,192
# 279 and 33. 16 heads over 4 of 64, a quarter of the bytes: 32 behind 2,048 (65 MB) 19.0 and 18.2; 64 behind 1,024 (66 MB) 19.0 and 19.8.
SHARE_BYTES = 9 << 20
# Several tokens a sequence: where the products bound the step, sharing saves whole rounds of the device alone (row tiles of short or ragged
# sequences that share theirs, keys split over blocks that would stand idle), and costs the join. Counted in steps of 128 keys (about 2 us, of a pair of
# row tiles; 1.75 times that in the kernel of steps of less than a tile): rounds * steps by themselves against rounds * steps and, for the join, 7 steps
# (half of them where a group's few rows go without tcgen05), 0.3 for each part of a row's prefix that is not empty (twice where a block has more than
# eight rows, which a thread joins one after the other), and (rows * heads) / 4,096.
# Behind 512, 1,024, 2,048 and 4,096 positions, us, by themselves and shared, 32 heads over 8 of 128: 2 sequences of 4 tokens 18.5 and 18.4, 31.5 and 19.1, 57 and
# 21, 109 and 26; 4 of 4 18.6 and 29.8, 31.8 and 36.9, 58 and 37, 110 and 51; 4 of 16 19.5 and 32.0, 32.5 and 43.5, 59 and 44, 111 and 46; 8 of 2 18.0 and 18.7, 31.1
# and 23.8, 57 and 24, 109 and 32; 8 of 30 19.6 and 26.6, 32.8 and 28.5, 59 and 32, 111 and 40; 32 of 8 32.6 and 24.1, 57 and 26, 104 and 30, 200 and 37. Behind
# 1,024 and 4,096: 4 of 60 24.6 and 28.9, 66 and 40; 16 of 60 26.9 and 41.1, 69 and 83; 2 of 250 26.8 and 38.3, 68 and 60; 4 of 250 28.4 and 49.0, 70 and
# 91; 16 of 45 to 90 behind 4,096 126 and 87. 16 heads over 4 of 64: 16 of 60 23.5 and 21.8, 66 and 41, 32 of 60 24.4 and 30.5, 67 and 70.
JOIN_STEPS = 7
PART_STEPS = 0.3


def single_tokens_share(sizes, lengths, row_bytes: int) -> bool:
    """Whether a step of one token a sequence reads these groups' prefixes once. ``row_bytes``: of one position's keys and values in one layer."""
    saved = 0
    for size, length in zip(sizes, lengths):
        saved += (size - 1) * length
    return saved * row_bytes >= SHARE_BYTES * min(sum(sizes), 8)


def longer_steps_share(sizes, lengths, q_lens, per: int, kv_heads: int) -> bool:
    """Whether a step of several tokens a sequence reads these groups' prefixes once. ``per``: query heads of a kv head."""
    steps, pages = max(lengths) / 128, max(lengths) // PAGE
    if 1.75 * steps < JOIN_STEPS:
        return False
    most = max(q_lens) * per  # rows of a sequence, for each kv head
    tile, factor = (256, 1.0) if most >= 128 else (64, 1.75)
    alone = sum(-(-n * per // tile) for n in q_lens) * kv_heads
    group_rows, at = [], 0
    for size in sizes:
        group_rows.append(sum(q_lens[at:at + size]) * per)
        at += size
    few = max(group_rows) <= 32
    shared = max(1, sum(-(-rows // (16 if few else 256)) for rows in group_rows) * kv_heads)
    splits = max(1, min(32, -(-148 // shared) if few else 148 // shared))
    parts = -(-pages // max(1, -(-pages // splits)))  # that are not empty
    rounds = -(-shared // 148) if shared >= 148 else shared / 148
    join = JOIN_STEPS * (0.5 if few else 1) + PART_STEPS * parts * (2 if most > 8 else 1) + sum(q_lens) * per * kv_heads / 4096
    return -(-alone // 148) * factor * steps >= rounds * steps + join


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
        self.max_length = max(lengths)
        cu = [0]
        for size in sizes:
            cu.append(cu[-1] + size)
        host = cu + lengths + [g for g, size in enumerate(sizes) for _ in range(size)]
        self.buffer = torch.tensor(host, dtype=torch.int32).to(device)
        n = self.n_groups
        self.cu, self.length, self.group = self.buffer[:n + 1], self.buffer[n + 1:2 * n + 1], self.buffer[2 * n + 1:]

    @staticmethod
    def shape_of(sizes, lengths) -> tuple:
        """What a captured step of such groups depends on, beside their number of sequences: how many there are, the power of two
        that none has more sequences than, and whether any shares."""
        return (len(sizes), 1 << (max(sizes) - 1).bit_length(), max(lengths) > 0)

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
        """No fewer rows of a step than one group has; where it is captured, for as long as ``update`` takes other groups."""
        if batch.max_q_len == 1:
            return self.shape[1]
        if self.buffer.is_cuda and torch.cuda.is_current_stream_capturing():
            return min(batch.n_rows, self.shape[1] * batch.max_q_len)
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
