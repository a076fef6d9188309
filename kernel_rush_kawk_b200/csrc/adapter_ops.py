"""Python bindings of the maps of a step and of the products with many requests' low-rank adapters. ``Kernels`` (bindings.py)
takes them in.

Scratch is drawn from torch's allocator for each call, so that calls on several streams, and captured steps beside
others, never share any.
"""

from __future__ import annotations

import ctypes
import os
from ctypes import POINTER, Structure, byref, c_float, c_int, c_longlong, c_void_p

import torch

from .build import build_library
from .cache_ops import PAGE, KernelError, _code, _current_device, _load, _ptr

_P = c_void_p
_I32 = torch.int32


class _Bank(Structure):
    _fields_ = [("a", _P), ("b", _P), ("scale", _P), ("ranks", _P), ("capacity", c_int), ("parts", c_int), ("rank", c_int), ("begin", c_int * 5),
                ("wide", c_int)]


_BANK = POINTER(_Bank)
_ADAPT_SIGNATURES = {
    "krk_step_maps": [_P, _P, _P, _P, c_int, c_int, _P, c_int, c_int, _P, c_int, _P, _P, _P, _P, _P, POINTER(_P), POINTER(_P), POINTER(c_int), c_int, _P, _P],
    "krk_adapter_first": [_P, _P, c_longlong, c_int, c_int, _BANK, _P, _P, c_int, _P],
    "krk_adapted_gemm": [_P, _P, c_longlong, _P, c_longlong, c_int, c_int, c_int, _BANK, _P, _P, _P, c_int, c_int, _P, _P, c_int, c_int, _P, _P],
    "krk_adapted_skinny": [_P, _P, _P, c_int, c_int, c_int, _BANK, _P, _P, _P, c_int, c_int, _P, c_int, _P, _P],
    "krk_adapter_second": [_P, _P, _P, c_int, c_int, _BANK, _P, c_int, c_int, _P],
}


class AdapterRows:
    """Which adapter each row of a step has (``row_adapter``, int32 on the device, -1 for none), and for tiles of rows of
    one height or three the adapters that occur in them. Made by ``Kernels.step_maps``."""

    HEIGHTS = (128, 192, 256)

    def __init__(self, n_rows: int, n_seqs: int, device):
        self.n_rows, self.n_seqs = n_rows, n_seqs
        self.heights = self.HEIGHTS if n_rows > 256 else (max(32, -(-n_rows // 32) * 32),)
        tiles = [-(-n_rows // h) for h in self.heights]
        self.n_slots = [t + n_seqs for t in tiles]
        at = n_rows + n_rows % 2  # pairs of words lie on boundaries of theirs
        self.buffer = torch.empty(at + sum(2 * t + 2 * s for t, s in zip(tiles, self.n_slots)), dtype=_I32, device=device)
        self.row_adapter = self.buffer[:n_rows]
        address = self.buffer.data_ptr()
        self.info, self.slots = [], []  # addresses
        for t, s in zip(tiles, self.n_slots):
            self.info.append(address + 4 * at)
            self.slots.append(address + 4 * (at + 2 * t))
            at += 2 * t + 2 * s


class StepMaps:
    """What ``Kernels.step_maps`` makes: ``cu_q`` [sequences + 1], the first row of every sequence; ``row_seq``, ``row_pos`` [rows], a row's sequence and
    position; with a page table ``row_place`` [rows] (int64), its place in the cache, page * 64 + position in the page; ``adapters`` (AdapterRows or None)."""

    def __init__(self, n_rows: int, n_seqs: int, device, with_places: bool = True, with_adapters: bool = True):
        self.n_rows, self.n_seqs = n_rows, n_seqs
        self.buffer = torch.empty(n_seqs + 1 + 2 * n_rows, dtype=_I32, device=device)
        self.cu_q, self.row_seq, self.row_pos = self.buffer[:n_seqs + 1], self.buffer[n_seqs + 1:n_seqs + 1 + n_rows], self.buffer[n_seqs + 1 + n_rows:]
        self.row_place = torch.empty(n_rows, dtype=torch.int64, device=device) if with_places else None
        self.adapters = AdapterRows(n_rows, n_seqs, device) if with_adapters else None


class AdapterOps:
    """Mixed into ``Kernels``."""

    MOST_SEQUENCES = 25000  # of one call of step_maps: every block holds their first rows and pages in shared memory

    @property
    def adapt(self) -> ctypes.CDLL:
        if self._adapt is None:
            self._adapt = _load(build_library("adapt"), _ADAPT_SIGNATURES)
        return self._adapt

    # -- maps of a step ----------------------------------------------------------------------
    def step_maps(self, slots, starts, lengths, n_rows, table=None, pages=None, adapters=None, out=None):
        """The maps of a step from its requests' lengths, on the device and in one launch.

        ``slots``, ``starts``, ``lengths`` (int32, one a sequence): its cache slot, the positions it holds and the tokens it
        brings; ``n_rows``: these together. ``table`` (int32 [slots, pages of a slot]): what the sequences hold in pages of 64; the pages that their new
        tokens need beyond are taken from ``pages`` (int32), in the order of the sequences, and entered. ``adapters`` (int32, one a
        sequence, -1 for none): its low-rank adapter. ``out``: a StepMaps to fill again (a captured step goes on reading it). No two sequences may have one slot.

        Lengths that do not add up to ``n_rows``, slots that the table does not have, and sequences that outgrow it or the given pages are
        found on the device: the error word is set (``check`` raises), and the rows concerned have position or place -1."""
        what, n, n_rows = "maps of a step", lengths.shape[0], int(n_rows)
        if n_rows < 0 or n > self.MOST_SEQUENCES:
            raise KernelError(f"{what}: {n} sequences with {n_rows} rows (up to {self.MOST_SEQUENCES} sequences are taken)")
        for name, t in (("slots", slots), ("starts", starts), ("lengths", lengths), ("adapters", adapters)):
            if t is not None and (t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous()):
                raise KernelError(f"{what}: {name} are contiguous int32, one for each of {n} sequences, got {t.dtype} {list(t.shape)}")
        width = n_slots = n_pages = 0
        if table is not None:
            if table.dtype is not _I32 or table.dim() != 2 or not table.is_contiguous():
                raise KernelError(f"{what}: the page table is contiguous int32 [slots, pages of a slot], got {table.dtype} {list(table.shape)}")
            n_slots, width = table.shape
            if pages is not None:
                if pages.dtype is not _I32 or pages.dim() != 1 or not pages.is_contiguous():
                    raise KernelError(f"{what}: pages are a contiguous int32 list, got {pages.dtype} {list(pages.shape)}")
                n_pages = pages.shape[0]
        elif pages is not None:
            raise KernelError(f"{what}: pages are entered in a page table, and there is none")
        self._check_device(what, slots, starts, lengths, *(t for t in (table, pages, adapters) if t is not None))
        if out is None:
            out = StepMaps(n_rows, n, lengths.device, table is not None, adapters is not None)
        elif (out.n_rows, out.n_seqs) != (n_rows, n) or (table is not None and out.row_place is None) or (out.adapters is None) != (adapters is None):
            raise KernelError(f"{what}: maps made for {out.n_seqs} sequences with {out.n_rows} rows do not fit {n} with {n_rows}, or lack places or adapters")
        rows = out.adapters
        if rows is None:
            info = lists = heights = None
            count = 0
        else:
            count = len(rows.heights)
            info, lists, heights = (_P * count)(*rows.info), (_P * count)(*rows.slots), (c_int * count)(*rows.heights)
        self._ok(self.adapt.krk_step_maps(
            slots.data_ptr(), starts.data_ptr(), lengths.data_ptr(), _ptr(adapters), n, n_rows, _ptr(table), width, n_slots, _ptr(pages), n_pages,
            out.cu_q.data_ptr(), out.row_seq.data_ptr(), out.row_pos.data_ptr(), None if rows is None else rows.row_adapter.data_ptr(),
            None if table is None else out.row_place.data_ptr(), info, lists, heights, count, self.error.data_ptr(), self._stream()), what)
        return out

    # -- products ------------------------------------------------------------------------------
    def _check_adapted(self, what, x, w, bank, rows):
        (M, K), (N, k) = x.shape, w.shape
        if k != K or bank.inputs != K or bank.outputs != N:
            raise KernelError(f"{what}: rows of {K} and weights {list(w.shape)} do not fit a bank from {bank.inputs} to {list(bank.outs)}")
        if x.dtype is not w.dtype or bank.dtype is not w.dtype:
            raise KernelError(f"{what}: rows, weights and adapters have one dtype, got {x.dtype}, {w.dtype} and {bank.dtype}")
        if rows.n_rows != M:
            raise KernelError(f"{what}: {M} rows, and adapters for {rows.n_rows}")
        if x.stride(1) != 1 or w.stride(1) != 1 or (M > 1 and x.stride(0) < K) or (N > 1 and w.stride(0) < K):
            raise KernelError(f"{what}: rows of elements side by side are asked for, got strides {x.stride()} and {w.stride()}")
        here = self.error.get_device()
        if not here == x.get_device() == w.get_device() == bank.a.get_device() == rows.buffer.get_device() == _current_device():
            self._check_device(what, x, w, bank.a, rows.buffer)

    @staticmethod
    def _bank(bank):
        described = bank._described
        if described is None:
            described = bank._described = byref(_Bank(bank.a.data_ptr(), bank.b.data_ptr(), bank.scale.data_ptr(), bank.ranks.data_ptr(), bank.capacity,
                                                      bank.parts, bank.rank, (c_int * 5)(*bank.begin, *[bank.outputs] * (5 - len(bank.begin))),
                                                      -(-bank.rank // 16) * 16))
        return described

    def adapted_linear(self, x, w, bank, rows):
        """y = x W^T + s (x A^T) B^T, A, B and s those of each row's adapter: x [rows, inputs], w [outputs, inputs], ``bank`` (parts.adapters.AdapterBank)
        the adapters, ``rows`` (AdapterRows) which row has which. Any number of rows, float32 or bfloat16; sums are held in
        32 bits and rounded once. A float32 row gives the same bits whatever stands beside it. Rows without an adapter give x W^T."""
        return self._adapted("adapted product", self._resolve(x), w, bank, rows, 0)

    def adapted_gate_up_swiglu(self, x, w_gate_up, intermediate, bank, rows):
        """silu(g) * u with g and u the two halves of ``adapted_linear``: w_gate_up [2 * intermediate, inputs], a bank of two parts of ``intermediate``
        outputs each. Gate and up are not rounded on the way."""
        if tuple(bank.outs) != (intermediate, intermediate):
            raise KernelError(f"adapted gate and up: a bank of two parts of {intermediate} outputs is asked for, got {list(bank.outs)}")
        return self._adapted("adapted gate and up", self._resolve(x), w_gate_up, bank, rows, intermediate)

    PAIRS = 74  # of SMs

    def _tiling(self, rows, M: int, K: int, N: int) -> tuple[int, int]:
        """(which of the rows' tile heights, the first tile that the pairs share): by the time of whole rounds of the pairs, or of whole rounds
        and shares of what is left, in clocks."""
        if len(rows.heights) == 1:
            return 0, 0
        if os.environ.get('TR'):
            h = int(os.environ['TR']); i = rows.heights.index(h); tiles = -(-M // h) * -(-N // 256)
            return i, (tiles if os.environ.get('NOSH') else tiles // 74 * 74)
        best = None
        for i, h in enumerate(rows.heights):
            tiles = -(-M // h) * -(-N // 256)
            tile = -(-K // 64) * (176 + 1.3125 * h)
            whole, rest = divmod(tiles, self.PAIRS)
            for cost, shared in (((whole + (rest > 0)) * tile, tiles), (whole * tile + rest / self.PAIRS * tile + 6000 + (self.PAIRS + rest) * h / 2, tiles - rest)):
                if best is None or cost < best[0]:
                    best = cost, i, shared
        return best[1], best[2]

    def _adapted(self, what, x, w, bank, rows, gated):
        self._check_adapted(what, x, w, bank, rows)
        (M, K), N = x.shape, w.shape[0]
        out = x.new_empty(M, gated or N)
        if M == 0:
            return out
        described, dtype, error = self._bank(bank), _code(w.dtype), self.error.data_ptr()
        ldx, ldw, x_at, w_at = x.stride(0) if M > 1 else K, w.stride(0) if N > 1 else K, x.data_ptr(), w.data_ptr()
        if w.dtype is torch.bfloat16 and K >= 64 and not (K | ldx | ldw | (gated or N)) & 7 and not (x_at | w_at) & 15:
            if M <= self.SKINNY_MAX_ROWS and K % 32 == 0 and ldx == K and ldw == K and not os.environ.get("NOSK"):
                t = self.error.new_empty(M * bank.parts * (-(-bank.rank // 16) * 8))
                self.launches += 1
                self._ok(self.adapt.krk_adapted_skinny(
                    out.data_ptr(), x_at, w_at, M, N, K, described, rows.row_adapter.data_ptr(), rows.info[0], rows.slots[0], rows.n_slots[0], rows.heights[0],
                    t.data_ptr(), int(gated > 0), error, self._stream()), what)
                return out
            which, shared = self._tiling(rows, M, K, N)
            height = rows.heights[which]
            n_slots, tiles = rows.n_slots[which], -(-M // height) * -(-N // 256)
            t_words = n_slots * height * bank.parts * (-(-bank.rank // 16) * 8)
            rest = tiles - shared
            t = self.error.new_empty(t_words + (rest * ((-(-self.PAIRS // rest) + 1) * height * 256 + 2) if rest else 0))
            t_at = t.data_ptr()
            self.launches += 1
            self._ok(self.adapt.krk_adapted_gemm(
                out.data_ptr(), x_at, ldx, w_at, ldw, M, N, K, described, rows.row_adapter.data_ptr(), rows.info[which], rows.slots[which], n_slots, height,
                t_at, t_at + 4 * t_words if rest else None, shared, int(gated > 0), error, self._stream()), what)
            return out
        t = self.error.new_empty(M * bank.parts * (-(-bank.rank // 16) * 16))
        if not x.is_contiguous():
            x = x.contiguous()
        y = self.linear(x, w, out_float32=True)
        stream, row_adapter = self._stream(), rows.row_adapter.data_ptr()
        self._ok(self.adapt.krk_adapter_first(t.data_ptr(), x.data_ptr(), K, M, K, described, row_adapter, error, dtype, stream), what)
        self._ok(self.adapt.krk_adapter_second(out.data_ptr(), y.data_ptr(), t.data_ptr(), M, N, described, row_adapter, int(gated > 0), dtype, stream), what)
        return out
