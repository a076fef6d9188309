"""Python bindings of the maps of a step and of the products with many requests' low-rank adapters. ``Kernels`` (bindings.py)
takes them in.

Scratch is drawn from torch's allocator for each call, so that calls on several streams, and captured steps beside
others, never share any.
"""

from __future__ import annotations

import ctypes
from ctypes import POINTER, Structure, byref, c_int, c_longlong, c_void_p
from functools import lru_cache

import torch

from .build import build_library
from .cache_ops import KernelError, _code, _current_device, _load, _ptr

_P = c_void_p
_I32 = torch.int32


class _Bank(Structure):
    _fields_ = [("a", _P), ("b", _P), ("scale", _P), ("ranks", _P), ("capacity", c_int), ("parts", c_int), ("rank", c_int), ("begin", c_int * 5),
                ("wide", c_int)]


_BANK = POINTER(_Bank)
_ADAPT_SIGNATURES = {
    "krk_step_maps": [_P, _P, _P, _P, c_int, c_int, _P, c_int, c_int, _P, c_int, _P, c_int, _P, _P],
    "krk_adapter_first": [_P, _P, c_longlong, c_int, c_int, _BANK, _P, _P, c_int, _P],
    "krk_adapted_gemm": [_P, _P, c_longlong, _P, c_longlong, c_int, c_int, c_int, _BANK, _P, _P, _P, c_int, c_int, _P, _P, c_int, c_int, _P, _P],
    "krk_adapted_skinny": [_P, _P, _P, c_int, c_int, c_int, _BANK, _P, _P, _P, c_int, c_int, _P, c_int, _P, _P],
    "krk_adapted_few_f32": [_P, _P, c_longlong, _P, c_longlong, c_int, c_int, c_int, _BANK, _P, _P, _P, _P],
    "krk_adapter_second": [_P, _P, _P, c_int, c_int, _BANK, _P, c_int, c_int, _P],
}


class AdapterRows:
    """Which adapter each row of a step has (``row_adapter``, int32 on the device, -1 for none), and for tiles of rows of
    one height or three the adapters that occur in them. A part of ``StepMaps``."""

    HEIGHTS = (128, 192, 256)

    def __init__(self, maps: "StepMaps", at: int):
        self.n_rows, self.n_seqs = maps.n_rows, maps.n_seqs
        self.heights = self.HEIGHTS if self.n_rows > 256 else (max(32, -(-self.n_rows // 32) * 32),)
        self.buffer, self._at = maps.buffer, at
        self.row_adapter_at = maps.address + 4 * at

    @property
    def row_adapter(self):
        return self.buffer[self._at:self._at + self.n_rows]

    def tiles(self, which: int) -> tuple:
        """(height, address of the tiles' first slots and counts, address of the slots, slots) for one of the heights."""
        at = self.row_adapter_at + 4 * (self.n_rows + self.n_rows % 2)
        for i, height in enumerate(self.heights):
            tiles = -(-self.n_rows // height)
            if i == which:
                return height, at, at + 8 * tiles, tiles + self.n_seqs
            at += 8 * (2 * tiles + self.n_seqs)
        raise IndexError(which)

    def words(self) -> int:
        """Of the buffer: a row's adapter, then on a boundary of eight bytes the heights' tiles and slots, two words each."""
        return self.n_rows + self.n_rows % 2 + sum(2 * (2 * -(-self.n_rows // h) + self.n_seqs) for h in self.heights)


class StepMaps:
    """What ``Kernels.step_maps`` makes: ``cu_q`` [sequences + 1], the first row of every sequence; ``row_seq``, ``row_pos`` [rows], a row's sequence and
    position; with a page table ``row_place`` [rows] (int64), its place in the cache, page * 64 + position in the page (-1 where maps with room for places are filled without a table); ``adapters`` (AdapterRows or None).
    All are views of one buffer."""

    def __init__(self, n_rows: int, n_seqs: int, device, with_places: bool = True, with_adapters: bool = True):
        self.n_rows, self.n_seqs, self.with_places = n_rows, n_seqs, with_places
        # places first; adapters on a boundary of eight bytes
        self._first = 2 * n_rows if with_places else 0
        at = self._first + n_seqs + 1 + 2 * n_rows
        at += at % 2
        extra = 0
        if with_adapters:
            tiles = sum(2 * (2 * -(-n_rows // h) + n_seqs) for h in AdapterRows.HEIGHTS) if n_rows > 256 else 2 * (2 * (n_rows > 0) + n_seqs)
            extra = n_rows + n_rows % 2 + tiles
        self.buffer = torch.empty(at + extra, dtype=_I32, device=device)
        self.address = self.buffer.data_ptr()
        self.adapters = AdapterRows(self, at) if with_adapters else None
        self._views = None

    def _split(self):
        if self._views is None:
            n, rows, words = self.n_seqs + 1, self.n_rows, self.buffer
            parts = words.split_with_sizes((self._first, n, rows, rows, words.shape[0] - self._first - n - 2 * rows))
            self._views = (parts[0].view(torch.int64) if self.with_places else None, parts[1], parts[2], parts[3])
        return self._views

    row_place = property(lambda self: self._split()[0])
    cu_q = property(lambda self: self._split()[1])
    row_seq = property(lambda self: self._split()[2])
    row_pos = property(lambda self: self._split()[3])


class AdapterOps:
    """Mixed into ``Kernels``."""

    MOST_SEQUENCES = 25000  # of one call of step_maps: every block holds their first rows and pages in shared memory
    MOST_ROWS = 1 << 28

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

        Lengths that do not add up to ``n_rows``, slots that the table does not have, sequences that outgrow it or the given pages, and pages that a sequence
        holds and the table lacks (entries below 0) are found on the device: the error word is set (``check`` raises), and the rows concerned have position or place -1."""
        what, n, n_rows = "maps of a step", lengths.shape[0], int(n_rows)
        if not 0 <= n_rows <= self.MOST_ROWS or n > self.MOST_SEQUENCES:
            raise KernelError(f"{what}: {n} sequences with {n_rows} rows (up to {self.MOST_SEQUENCES} sequences and {self.MOST_ROWS} rows are taken)")
        tensors = (slots, starts, lengths) if adapters is None else (slots, starts, lengths, adapters)
        for t in tensors:
            if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous():
                raise KernelError(f"{what}: slots, starts, lengths and adapters are contiguous int32, one for each of {n} sequences, got "
                                  f"{', '.join(f'{t.dtype} {list(t.shape)}' for t in tensors)}")
        width = n_slots = n_pages = 0
        if table is not None:
            if table.dtype is not _I32 or table.dim() != 2 or not table.is_contiguous():
                raise KernelError(f"{what}: the page table is contiguous int32 [slots, pages of a slot], got {table.dtype} {list(table.shape)}")
            n_slots, width = table.shape
            tensors += (table,)
            if pages is not None:
                if pages.dtype is not _I32 or pages.dim() != 1 or not pages.is_contiguous():
                    raise KernelError(f"{what}: pages are a contiguous int32 list, got {pages.dtype} {list(pages.shape)}")
                n_pages = pages.shape[0]
                tensors += (pages,)
        elif pages is not None:
            raise KernelError(f"{what}: pages are entered in a page table, and there is none")
        self._check_device(what, *tensors)
        if out is None:
            out = StepMaps(n_rows, n, lengths.device, table is not None, adapters is not None)
        elif (out.n_rows, out.n_seqs) != (n_rows, n) or (table is not None and not out.with_places) or (out.adapters is None) != (adapters is None):
            raise KernelError(f"{what}: maps made for {out.n_seqs} sequences with {out.n_rows} rows do not fit {n} with {n_rows}, or lack places or adapters")
        elif out.buffer.get_device() != lengths.get_device():
            raise KernelError(f"{what}: maps on {out.buffer.device} for lengths on {lengths.device}")
        self._ok(self.adapt.krk_step_maps(
            slots.data_ptr(), starts.data_ptr(), lengths.data_ptr(), _ptr(adapters), n, n_rows, _ptr(table), width, n_slots, _ptr(pages), n_pages,
            out.address, int(out.with_places), self.error.data_ptr(), self._stream()), what)
        return out

    # -- products ------------------------------------------------------------------------------
    def _check_adapted(self, what, x, w, bank, rows):
        """Raise unless the product can be taken; (rows, inputs, outputs, elements between rows of x and of w, their addresses)."""
        (M, K), (N, k), (ldx, step_x), (ldw, step_w), dtype = x.shape, w.shape, x.stride(), w.stride(), w.dtype
        if k != K or bank.inputs != K or bank.outputs != N:
            raise KernelError(f"{what}: rows of {K} and weights {list(w.shape)} do not fit a bank from {bank.inputs} to {list(bank.outs)}")
        if x.dtype is not dtype or bank.dtype is not dtype:
            raise KernelError(f"{what}: rows, weights and adapters have one dtype, got {x.dtype}, {w.dtype} and {bank.dtype}")
        if rows.n_rows != M:
            raise KernelError(f"{what}: {M} rows, and adapters for {rows.n_rows}")
        if M <= 1:
            ldx = K  # (a single row has no stride that means anything)
        if N <= 1:
            ldw = K
        if step_x != 1 or step_w != 1 or ldx < K or ldw < K:
            raise KernelError(f"{what}: rows of elements side by side are asked for, got strides {x.stride()} and {w.stride()}")
        if not self.error.get_device() == x.get_device() == w.get_device() == bank.a.get_device() == rows.buffer.get_device() == _current_device():
            self._check_device(what, x, w, bank.a, rows.buffer)
        return M, K, N, ldx, ldw, x.data_ptr(), w.data_ptr()

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
        32 bits and rounded once. Scratch of more than 16 bfloat16 rows: their tiles' height times tiles and sequences times parts times the rank, 16 bits each
        (a thousand sequences of one token, rank 64, three parts: 99 MB; 25,000, rank 16: 0.6 GB). A float32 row gives the same bits whatever stands beside it. Rows without an adapter give x W^T."""
        return self._adapted("adapted product", self._resolve(x), w, bank, rows, 0)

    def adapted_gate_up_swiglu(self, x, w_gate_up, intermediate, bank, rows):
        """silu(g) * u with g and u the two halves of ``adapted_linear``: w_gate_up [2 * intermediate, inputs], a bank of two parts of ``intermediate``
        outputs each. Gate and up are not rounded on the way."""
        if tuple(bank.outs) != (intermediate, intermediate):
            raise KernelError(f"adapted gate and up: a bank of two parts of {intermediate} outputs is asked for, got {list(bank.outs)}")
        return self._adapted("adapted gate and up", self._resolve(x), w_gate_up, bank, rows, intermediate)

    PAIRS = 74  # of SMs

    @staticmethod
    @lru_cache(maxsize=4096)
    def _tiling(heights, M: int, K: int, N: int) -> tuple[int, int]:
        """(which of the rows' tile heights, the first tile that the pairs share): whole rounds of the pairs, or whole rounds and shares of what is left, by
        their time in clocks. Up to 128 rows W's bytes are the cost, and all pairs share all tiles: 64 rows of 2,560 x 6,144 22.5 us, as whole tiles
        24.6, of 9,728 x 2,560 26.6 and 53.2; 128 rows 25.9 and 27.3, 32.8 and 61.4.

        Above, a round takes what a block of k takes of a pair, 380 clocks and half a clock a row, and shares take the way to memory and back, as many times as
        a tile has pairs; a row tile takes its first factor. The constants come from six shapes (K and N of 2,560 to 9,728 and 19,456), 160 to 4,096 rows, every
        height with shares and without: what this picks is 0.4 % behind the fastest on average, 8 % at worst. Cold, us, whole and shares: 256 rows of 2,560 x
        6,144 27.3 and 32.8, of 9,728 x 2,560 57.3 and 45.1; 2,268 rows of that, tiles of 256, 124.9 and 110.6; 400 rows of 2,560 x 6,144 in tiles of 256 26.6 and
        38.9, of 192 30.7, of 128 38.9; 512 rows of 2,560 x 19,456 61.4 and 86."""
        if len(heights) == 1 and heights[0] <= 128:
            return 0, 0
        best = None
        for i, h in enumerate(heights):
            row_tiles = -(-M // h)
            tiles = row_tiles * -(-N // 256)
            tile = -(-K // 64) * (380 + 0.516 * h)
            shared = tiles // AdapterOps.PAIRS * AdapterOps.PAIRS if len(heights) > 1 else 0
            rest = tiles - shared
            options = [(-(-tiles // AdapterOps.PAIRS) * tile, tiles)]
            if rest:
                options.append(((shared + rest) / AdapterOps.PAIRS * tile + 8000 + 24 * h * (2 + AdapterOps.PAIRS / rest), shared))
            for cost, first in options:
                cost += 4000 * row_tiles
                if best is None or cost < best[0]:
                    best = cost, i, first
        return best[1], best[2]

    def _adapted(self, what, x, w, bank, rows, gated):
        M, K, N, ldx, ldw, x_at, w_at = self._check_adapted(what, x, w, bank, rows)
        out = x.new_empty(M, gated or N)
        if M == 0:
            return out
        described, error, stream, row_adapter = self._bank(bank), self.error.data_ptr(), self._stream(), rows.row_adapter_at
        if bank.dtype is torch.bfloat16 and K >= 64 and not (K | ldx | ldw | (gated or N)) & 7 and not (x_at | w_at) & 15:
            self.launches += 1
            half_width = bank.parts * (-(-bank.rank // 16) * 8)
            if M <= self.SKINNY_MAX_ROWS and not K & 31 and ldx == K and ldw == K:
                height, info, slots, n_slots = rows.tiles(0)
                t = self.error.new_empty(M * half_width)
                self._ok(self.adapt.krk_adapted_skinny(out.data_ptr(), x_at, w_at, M, N, K, described, row_adapter, info, slots, n_slots, height, t.data_ptr(),
                                                       int(gated > 0), error, stream), what)
                return out
            which, shared = self._tiling(rows.heights, M, K, N)
            height, info, slots, n_slots = rows.tiles(which)
            rest = -(-M // height) * -(-N // 256) - shared
            t_words = n_slots * height * half_width
            t = self.error.new_empty(t_words + (rest * ((-(-self.PAIRS // rest) + 1) * height * 256 + 2) if rest else 0))
            t_at = t.data_ptr()
            self._ok(self.adapt.krk_adapted_gemm(out.data_ptr(), x_at, ldx, w_at, ldw, M, N, K, described, row_adapter, info, slots, n_slots, height, t_at,
                                                 t_at + 4 * t_words if rest else None, shared, int(gated > 0), error, stream), what)
            return out
        # The second factor behind each sum, by the thread that holds it, up to 256 ranks times rows; more of them go over all SMs in a launch of their own. us,
        # 2,560 x 6,144, 9,728 x 2,560 and gate and up of 2,560 x 19,456: one row of rank 16 18.5, 36.9 and 45.1 (a launch of its own 24.5, 43.0 and 47.1), eight rows
        # with eight of rank 32 32.8, 55 and 68 (34.8, 61 and 64), sixteen with nine of rank 32 49, 98 and 121 (45, 98 and 109), of rank 64 64, 104 and 147 (51, 102 and 123).
        if w.dtype is torch.float32 and M <= self.SKINNY_MAX_ROWS and M * bank.rank <= 256 and not (K | ldx | ldw) & 3 and not (x_at | w_at) & 15:
            self.launches += 1
            t, y = self.error.new_empty(M * bank.parts * (-(-bank.rank // 16) * 16)), x.new_empty(M, N) if gated else out
            self._ok(self.adapt.krk_adapted_few_f32(y.data_ptr(), x_at, ldx, w_at, ldw, M, N, K, described, row_adapter, t.data_ptr(), error, stream), what)
            return self.swiglu(y, gated) if gated else out
        # more rows of float32, and sizes, strides and addresses that the tensor cores' copies do not take
        if not x.is_contiguous():
            x = x.contiguous()
        t = self.error.new_empty(M * bank.parts * (-(-bank.rank // 16) * 16))
        y, dtype = self.linear(x, w, out_float32=True), _code(w.dtype)
        self._ok(self.adapt.krk_adapter_first(t.data_ptr(), x.data_ptr(), K, M, K, described, row_adapter, error, dtype, stream), what)
        self._ok(self.adapt.krk_adapter_second(out.data_ptr(), y.data_ptr(), t.data_ptr(), M, N, described, row_adapter, int(gated > 0), dtype, stream), what)
        return out
