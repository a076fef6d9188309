"""Low-rank adapters of one projection, many side by side.

A projection y = x W^T may be a part of several variants of a model, each of which adds a product of low rank of its own,
s (x A^T) B^T with A [r, inputs] and B [outputs, r]. An ``AdapterBank`` holds these for one projection (or several that are one product:
queries, keys and values) in fixed storage, so that variants come and go while captured steps that read it stay valid.
``Kernels.adapted_linear`` and ``Kernels.adapted_gate_up_swiglu`` take a bank and, for each row of a step, the adapter that it has.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

MAX_PARTS = 4  # projections side by side in one product
MAX_RANK = 256


class AdapterError(ValueError):
    pass


@dataclass(frozen=True)
class AdapterRoom:
    """How many low-rank adapters an engine holds at a time, and of which rank at most."""

    count: int
    rank: int

    def __post_init__(self):
        if self.count < 1 or not 1 <= self.rank <= MAX_RANK:
            raise AdapterError(f"an engine has room for one adapter at least, of ranks from 1 to {MAX_RANK}; got {self.count} of rank {self.rank}")


class AdapterBank:
    """Room for ``capacity`` adapters of rank ``rank`` at most, beside a product from ``inputs`` to the outputs ``outs`` (a number, or the
    numbers of several projections side by side, called parts).

    ``a`` [capacity, parts * rank, inputs], ``b`` [capacity, outputs, rank] (the rank rounded up to a multiple of eight), ``scale`` (float32)
    and ``ranks`` (int32) [capacity, parts]; a part whose rank is 0 is left as it is by the adapter. What lies behind an adapter's rank is never read as
    a number. The tensors stay the bank's own: they are filled by ``put``."""

    a = property(lambda self: self._a)
    b = property(lambda self: self._b)
    scale = property(lambda self: self._scale)
    ranks = property(lambda self: self._ranks)

    def __init__(self, inputs: int, outs, capacity: int, rank: int, dtype: torch.dtype, device):
        outs = (int(outs),) if isinstance(outs, int) else tuple(int(n) for n in outs)
        if not 1 <= len(outs) <= MAX_PARTS or min(outs) < 1 or inputs < 1 or capacity < 1:
            raise AdapterError(f"a bank has one to {MAX_PARTS} parts and room for one adapter at least, got {inputs} inputs, outputs {list(outs)}, {capacity} adapters")
        if not 1 <= rank <= MAX_RANK:
            raise AdapterError(f"adapters have ranks from 1 to {MAX_RANK}, got {rank}")
        if dtype not in (torch.float32, torch.bfloat16):
            raise AdapterError(f"adapters are float32 or bfloat16 like the projection beside them, got {dtype}")
        self.inputs, self.outs, self.capacity = int(inputs), outs, int(capacity)
        self.outputs = sum(outs)
        self.most = int(rank)
        self.rank = -(-int(rank) // 8) * 8
        self.dtype = dtype
        self.begin = [sum(outs[:i]) for i in range(len(outs) + 1)]
        parts = len(outs)
        self._a = torch.zeros((capacity, parts * self.rank, self.inputs), dtype=dtype, device=device)
        self._b = torch.zeros((capacity, self.outputs, self.rank), dtype=dtype, device=device)
        self._scale = torch.zeros((capacity, parts), dtype=torch.float32, device=device)
        self._ranks = torch.zeros((capacity, parts), dtype=torch.int32, device=device)
        self._described = None  # how the kernels are told (Kernels keeps it here)

    @property
    def parts(self) -> int:
        return len(self.outs)

    def bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.a, self.b, self.scale, self.ranks))

    def _index(self, index: int) -> int:
        if not 0 <= index < self.capacity:
            raise AdapterError(f"adapter {index} of a bank of {self.capacity}")
        return index

    def check(self, part: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Raise unless ``put`` takes them."""
        if not 0 <= part < self.parts:
            raise AdapterError(f"part {part} of a bank of {self.parts}")
        n = self.outs[part]
        if a.dim() != 2 or b.dim() != 2 or a.shape[1] != self.inputs or b.shape != (n, a.shape[0]):
            raise AdapterError(f"an adapter from {self.inputs} to {n} is [rank, {self.inputs}] and [{n}, rank], got {list(a.shape)} and {list(b.shape)}")
        if not 1 <= a.shape[0] <= self.most:
            raise AdapterError(f"an adapter of rank {a.shape[0]} in a bank of rank {self.most}")
        # rows of other adapters are multiplied by these factors as well, as zeros, and are to stay numbers
        # (the scale is held in 32 bits)
        if not abs(scale) <= torch.finfo(torch.float32).max or not all(torch.isfinite(t.detach().to(self.dtype)).all() for t in (a, b)):
            raise AdapterError(f"an adapter's factors and scale are finite numbers ({self.dtype})")

    @torch.no_grad()
    def put(self, index: int, part: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0) -> None:
        """Adapter ``index`` of ``part``: a [r, inputs], b [the part's outputs, r], of finite numbers (which the host waits to know). The copies are queued
        on the current stream, behind the steps that were queued on it before."""
        self._index(index)
        self.check(part, a, b, scale)
        n, r = self.outs[part], a.shape[0]
        self.a[index, part * self.rank:part * self.rank + r].copy_(a)
        self.b[index, self.begin[part]:self.begin[part] + n, :r].copy_(b)
        if r < self.rank:
            self.b[index, self.begin[part]:self.begin[part] + n, r:].zero_()  # the kernels take whole steps of sixteen
        self.scale[index, part] = float(scale)
        self.ranks[index, part] = r

    def clear(self, index: int) -> None:
        """The adapter adds nothing any more."""
        self.ranks[self._index(index)].zero_()
