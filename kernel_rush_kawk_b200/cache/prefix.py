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
# Single tokens, by the bytes of keys and values of one layer that are not read again: 8 MB a sequence, up to eight of them. A layer's attention with
# rotation and cache write, us, each sequence by itself and shared, 32 heads over 8 of 128 with 100 keys of their own: 2 sequences behind 4,096 positions
# (17 MB) 13.9 and 15.0, 8,192 22.8 and 16.9; 4 behind 2,048 (25 MB) 15.6 and 17.0, 4,096 22.1 and 18.7; 8 behind 2,048 (59 MB) 15.4 and 18.1,
# 4,096 24.4 and 21.3; 16 behind 1,024 (63 MB) 16.2 and 18.9, 2,048 24.5 and 19.0; 64 behind 256 (66 MB) 22.9 and 21.6, 1,024 47.9 and 23.4, 8,192
# 278.8 and 30.9. 16 heads over 4 of 64, a quarter of the bytes: 32 behind 1,024 (33 MB) 12.3 and 17.2, 2,048 18.9 and 18.0; 64 behind 1,024 (66 MB) 18.8 and
# 17.5.
SHARE_BYTES = 8 << 20
# Several tokens a sequence: where the products bound the step, sharing saves whole rounds of the device alone (row tiles of short or ragged
# sequences that share theirs, keys split over blocks that would stand idle), and costs the join. Counted in steps of 128 keys (about 2 us, of a pair of
# row tiles; 1.75 times that in the kernel of steps of less than a tile): rounds * steps by themselves against rounds * steps + 8 + (rows * heads) / 4,096.
# Measured behind 1,024 and 4,096 positions, us, by themselves and shared, 32 heads over 8 of 128: 2 sequences of 4 tokens 32.7 and 18.5, 116 and 25;
# 4 of 16 31.8 and 36.4, 110 and 38.6; 32 of 4 45 and 26.2, 157 and 31.8; 4 of 60 24.7 and 25.3, 66 and 36.4; 16 of 60 26.4 and 40.9, 70 and 82; 16 of 45 to
# 90 behind 4,096 129 and 94; 2 of 250 26.8 and 33.3, 69 and 55; 4 of 250 28 and 51, 71 and 92; 16 heads over 4 of 64, 16 of 60 23.6 and 22.1, 65
# and 42, 32 of 60 24.2 and 30.7, 66 and 70.
JOIN_STEPS = 8


def single_tokens_share(sizes, lengths, row_bytes: int) -> bool:
    """Whether a step of one token a sequence reads these groups' prefixes once. ``row_bytes``: of one position's keys and values in one layer."""
    saved = 0
    for size, length in zip(sizes, lengths):
        saved += (size - 1) * length
    return saved * row_bytes >= SHARE_BYTES * min(sum(sizes), 8)


def longer_steps_share(sizes, lengths, q_lens, per: int, kv_heads: int) -> bool:
    """Whether a step of several tokens a sequence reads these groups' prefixes once. ``per``: query heads of a kv head."""
    steps = max(lengths) / 128
    if 1.75 * steps < JOIN_STEPS:
        return False
    tile, factor = (256, 1.0) if max(q_lens) * per >= 128 else (64, 1.75)
    alone = sum(-(-n * per // tile) for n in q_lens) * kv_heads
    shared, at = 0, 0
    for size in sizes:
        shared += -(-sum(q_lens[at:at + size]) * per // 256) * kv_heads
        at += size
    rounds = -(-shared // 148) if shared >= 148 else shared / 148
    return -(-alone // 148) * factor * steps >= rounds * steps + JOIN_STEPS + sum(q_lens) * per * kv_heads / 4096


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
