"""Python bindings of the kernels that share and thin out the cache: attention behind a prefix that several sequences hold
in the same pages, attention that adds up the weight which each cached key receives, and the eviction of the keys that
received least. ``Kernels`` (bindings.py) takes them in.

Scratch is drawn from torch's allocator for each call, so that calls on several streams, and captured steps beside
others, never share any.
"""

from __future__ import annotations

import ctypes
from ctypes import c_float, c_int, c_longlong, c_void_p

import torch

from ..cache.prefix import longer_steps_share, single_tokens_share
from .build import build_library

F32, BF16 = 0, 1
_F32, _I32 = torch.float32, torch.int32
_P = c_void_p
PAGE = 64
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)  # (the function around it costs as much again)


def _code(dtype: torch.dtype) -> int:
    if dtype == torch.float32:
        return F32
    if dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"kernels take float32 or bfloat16 tensors, got {dtype}")


class KernelError(RuntimeError):
    pass


def _load(path, signatures) -> ctypes.CDLL:
    lib = ctypes.CDLL(str(path))
    for name, args in signatures.items():
        try:
            fn = getattr(lib, name)
        except AttributeError:
            continue
        fn.argtypes = args
        fn.restype = c_int
    return lib


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


_SEGMENTS = [_P] * 7 + [c_int, c_int, _P, c_int]
_PARTS_SIGNATURES = {
    "krk_attention_in_parts": [_P, _P, _P, _P, c_int, c_int, c_int, _P, _P, _P, _P, c_int, c_int, c_int, c_int, _P, c_int, c_int, c_int, *_SEGMENTS, _P, _P, c_int,
                               c_int, c_float, c_int, _P],
    "krk_key_weights": [_P, _P, _P, _P, c_int, _P, c_int, _P, c_int, c_int, c_int, *_SEGMENTS, _P, c_int, c_int, c_float, c_int, _P],
}
_PARTS_SIGNATURES.update({
    "krk_prefix_few_rows": [_P, _P, c_int, c_int, c_int, _P, c_int, c_int, c_int, *_SEGMENTS, _P, _P, c_int, c_int, c_float, _P, _P],
    "krk_prefix_tcgen05": [_P, _P, c_int, c_int, c_int, _P, c_int, c_int, c_int, *_SEGMENTS, _P, _P, c_int, c_int, c_int, c_float, _P, _P],
    "krk_shared_single": [_P, _P, _P, c_int, c_int, c_int, _P, c_int, c_int, c_int, *_SEGMENTS, _P, _P, c_int, c_int, c_float, _P, _P],
    "krk_scored_single": [_P, _P, _P, _P, _P, _P, c_int, c_int, _P, c_int, c_int, c_int, *_SEGMENTS, _P, _P, c_int, c_float, _P, _P],
})
_PARTS_SIGNATURES.update({
    "krk_own_rows": [_P, _P, _P, _P, c_int, c_int, _P, c_int, c_int, c_int, *_SEGMENTS, _P, _P, c_int, c_float, _P],
    "krk_key_weights_tcgen05": [_P, _P, _P, _P, c_int, _P, c_int, _P, c_int, c_int, c_int, *_SEGMENTS, _P, c_int, c_int, c_int, c_int, c_float, _P, _P],
})
_CACHE_SIGNATURES = {
    "krk_evict_max_seqs": [],
    "krk_evict_keys": [_P, _P, c_longlong, c_longlong, c_int, c_int, c_int, c_int, _P, c_int, _P, _P, _P, _P, c_longlong, c_int, _P, _P, c_int,
                       c_int, c_int, _P, _P, c_int, _P, _P, _P, _P],
}


class CacheOps:
    """Mixed into ``Kernels``."""

    PREFIX_TENSOR_ROWS = 33  # rows of a group from which on its prefix goes to the tcgen05 kernel
    EVICT_SCRATCH_BYTES = 64 << 20  # the lists of moves of one pair of launches; more sequences take several pairs

    def _parts_lib(self, head_dim: int) -> ctypes.CDLL:
        lib = self.parts.get(head_dim)
        if lib is None:
            if head_dim % 2 or head_dim > 256:
                raise KernelError(f"attention kernels take an even head size up to 256, got {head_dim}")
            lib = self.parts[head_dim] = _load(build_library("parts", head_dim), _PARTS_SIGNATURES)
        return lib

    @property
    def cache_lib(self) -> ctypes.CDLL:
        if self._cache_lib is None:
            self._cache_lib = _load(build_library("cache"), _CACHE_SIGNATURES)
        return self._cache_lib

    # -- what both attentions ask of their arguments ---------------------------------
    def _check_step(self, what, qkv, heads, kv_in_row, head_dim, batch, cache, also=None):
        """Raise unless the step can be taken; (address of the rows, elements between them, addresses of the pages of keys and of values).
        ``also``: one more tensor (or None) that the call reads on the device."""
        shape, dtype, k, v, table, kv, width = qkv.shape, qkv.dtype, cache.k, cache.v, cache.table, cache.kv_heads, cache.width
        strides, pages, slots, held = qkv.stride(), k.shape, batch.slots, table.shape
        if len(shape) != 2 or strides[1] != 1 or shape[1] != (heads + 2 * kv_in_row) * head_dim:
            raise KernelError(f"{what}: rows of {(heads + 2 * kv_in_row) * head_dim} elements side by side are asked for, got {tuple(shape)}")
        if heads % kv or cache.head_dim != head_dim or cache.v_dim != head_dim:
            raise KernelError(f"{what}: {heads} heads of {head_dim} do not fit a cache of {kv} heads of {cache.head_dim} (values: {cache.v_dim})")
        if cache.window is not None or cache.keep_pages:
            raise KernelError(f"{what}: the cache keeps a window of keys; every key is asked for")
        if (k.dtype is not dtype or v.dtype is not dtype or not k.is_contiguous() or not v.is_contiguous() or v.shape != pages
                or pages != (pages[0], kv, PAGE, head_dim)):
            raise KernelError(f"{what}: the cache's pages are contiguous [pages, kv heads, {PAGE}, head size] of the rows' dtype ({dtype}), "
                              f"got {k.dtype} {list(pages)} and {v.dtype} {list(v.shape)}")
        if held != (held[0], width) or table.dtype is not _I32 or not table.is_contiguous():
            raise KernelError(f"{what}: the page table is contiguous int32 [slots, {width}], got {table.dtype} {list(held)}")
        rows = shape[0]
        if rows != batch.n_rows or batch.max_kv_len > width * PAGE:
            raise KernelError(f"{what}: {rows} rows for a step of {batch.n_rows} with up to {batch.max_kv_len} keys, in slots of {width * PAGE}")
        if slots and (min(slots) < 0 or max(slots) >= held[0]):
            raise KernelError(f"{what}: slots {list(slots)} of {held[0]}")
        if rows > 1 and strides[0] < shape[1]:
            raise KernelError(f"{what}: rows that overlap (a stride of {strides[0]})")
        here, cu = self.error.get_device(), batch.cu_q
        if not (here == qkv.get_device() == k.get_device() == v.get_device() == table.get_device() == cu.get_device() == _current_device()
                and (also is None or also.get_device() == here)):
            self._check_device(what, qkv, k, v, table, cu, *(() if also is None else (also,)))
        # (a single row has no stride that means anything)
        return qkv.data_ptr(), strides[0] if rows > 1 else shape[1], k.data_ptr(), v.data_ptr()

    @staticmethod
    def _one_each(batch) -> bool:
        """Whether every sequence brings one token: what the single-token kernels, which take a sequence's number for its row, need. (Steps in which some
        bring none are longer ones to them.)"""
        return batch.is_decode and batch.n_rows == batch.n_seqs

    def _check_device(self, what, *tensors):
        mine = self.error.get_device()
        for t in tensors:
            if t.get_device() != mine:
                break
        else:
            if _current_device() == mine:
                return
        raise KernelError(f"{what}: tensors on {', '.join(str(t.device) for t in tensors)}, device {torch.cuda.current_device()} current, "
                          f"kernels on {self.error.device}")

    @staticmethod
    def _segments(batch, cache, prefix):
        groups = (None, None, None, batch.n_seqs, 0) if prefix is None else (
            prefix.cu.data_ptr(), prefix.length.data_ptr(), prefix.group.data_ptr(), batch.n_seqs, prefix.n_groups)
        return (batch.cu_q.data_ptr(), batch.seq_slot.data_ptr(), batch.seq_start.data_ptr(), batch.seq_qlen.data_ptr(), *groups,
                cache.table.data_ptr(), cache.width)

    @staticmethod
    def _splits(blocks: int, wanted: int) -> int:
        """Parts that the keys of a unit of work are split into, so that there are blocks enough for the device. By the numbers of rows
        and heads, never by lengths: a captured step stays valid."""
        return max(1, min(32, -(-wanted // max(blocks, 1))))

    @staticmethod
    def _places(blocks: int, head_dim: int) -> int:
        """Parts of a prefix, whose blocks have equal work, for the kernel of every type: of its blocks an SM has two, or one of large heads, and as many
        come as run at once (four sequences of 30 tokens behind 1,024 positions, 32 heads over 8 of 128 in float32: 103 us, 128 with half a round more). Own
        keys are unequally many, and come in more: a prompt of 600 tokens, 16 heads over 4 of 64, 115 us in three parts a tile and 150 in one."""
        return max(1, min(32, 148 * (2 if head_dim <= 128 else 1) // max(blocks, 1)))

    @staticmethod
    def _cluster_splits(items: int, all_keys: bool) -> int:
        """Blocks of a cluster that share the keys of a sequence's token, by the number of (sequence, kv head, row tile) items. ``all_keys``: all
        that the sequence holds, unequally many; else those behind a shared prefix, which are few.

        As many as run at once, four blocks an SM: 60 clusters of eight, 132 of four, 296 of two. Counted tokens of 32 heads over 8 of 128 or of 4 over one, us
        after 300, 1,500 and 8,000 keys, from keys in memory: 48 items in eight 9.6, 14.1 and 39, in four 9.2, 14.0 and 44; 66 in eight 12.5, 18.4 and
        52, in four 9.7, 15.9 and 56; 128 in four 11.2, 23.5 and 92, in two 11.1, 24.5 and 104; 144 in four 17.9, 35.9 and 137, in two
        11.3, 26.4 and 111; 296 in two 15.2, 45.2 and 208, in one 13.6, 46.4 and 228; 297 in two 22.4, 59 and 264, in one 14.3, 48 and 234. One sequence, eight
        items, after 1,500 keys in 1, 2, 4 and 8: 23.5, 15.5, 11.3 and 9.4.

        Behind a prefix of 4,096, with 100, 500 and 2,000 keys of their own (the prefix's kernel among it): 16 items in two 14.1, 12.7 and 20.9, in one 11.6,
        13.9 and 30.6; 24 in two 15.7, 17.6 and 21.4, in one 13.5, 14.0 and 31.0; 64 in two 20.1, 22.2 and 30.5, in one 16.2, 16.4 and 30.4."""
        if all_keys:
            return 8 if items <= 60 else 4 if items <= 132 else 2 if items <= 296 else 1
        return 2 if items <= 16 else 1

    @staticmethod
    def _by_mma(dtype, head_dim, q, stride, k, v) -> bool:
        """Whether the tensor-core kernels take these rows and pages: bfloat16, head sizes in steps of 16, rows from 4-byte, pages from 16-byte
        boundaries on."""
        return dtype == torch.bfloat16 and head_dim % 16 == 0 and stride % 2 == 0 and q % 4 == 0 and (k | v) % 16 == 0

    @staticmethod
    def _by_tcgen05(head_dim, q, stride) -> bool:
        """Whether the tcgen05 kernels take rows that ``_by_mma`` takes: heads of 64 or 128, rows from 16-byte boundaries on."""
        return head_dim in (64, 128) and stride % 8 == 0 and q % 16 == 0

    # -- a shared prefix -----------------------------------------------------------------
    def shared_prefix_attention(self, qkv, heads, kv_in_row, head_dim, batch, cache, scale, prefix):
        """``attention`` for a step whose sequences share prefixes: [rows, heads * head_dim], every row over all keys up to its own
        position. ``prefix`` (cache.prefix.PrefixGroups) says which neighbouring sequences of the step hold the same first positions in the
        same pages (``SequenceCache.fork`` makes such sequences); a group's keys and values are read once for all of its rows where that pays
        (cache.prefix says when; elsewhere each sequence reads its own table's). The step's
        own keys and values must be in the cache already, and its rows lie behind their group's prefix. Any number of tokens a
        sequence, float32 or bfloat16; a captured step stays valid while the groups' number and sizes last, whatever the lengths become."""
        q, stride, k, v = self._check_step("shared prefix attention", qkv, heads, kv_in_row, head_dim, batch, cache, prefix.buffer)
        prefix.check(batch, cache)
        lib, rows, kv, per, D = self._parts_lib(head_dim), batch.n_rows, cache.kv_heads, heads // cache.kv_heads, head_dim
        out = qkv.new_empty(rows, heads * D)
        if rows == 0:
            return out
        scale, stream, error = float(scale), self._stream(), self.error.data_ptr()
        by_mma, one_each = self._by_mma(qkv.dtype, D, q, stride, k, v), self._one_each(batch)
        if by_mma and not (single_tokens_share(prefix.sizes, prefix.lengths, 4 * kv * D) if one_each else
                           longer_steps_share(prefix.sizes, prefix.lengths, batch.q_lens, per, kv)):
            self._whole_attention(out, None, (q, stride, heads, kv), D, batch, cache, (k, v), scale)  # each sequence by itself, through its own page table
            return out
        step = (q, stride, heads, kv, *self._segments(batch, cache, prefix), k, v)
        group_rows = prefix.max_rows(batch) if prefix.max_length else 0
        tiles = -(-group_rows * per // 16) * kv
        by_mma = by_mma and tiles <= 65535
        # the prefixes' parts, then the own keys, which join them
        own_splits, tensor = 0, 0
        if not by_mma:
            splits = self._places(-(-group_rows * per // 64) * kv * prefix.n_groups, D) if group_rows else 0
            own_splits = self._splits(-(-batch.max_q_len * per // 64) * kv * batch.n_seqs, 444)
        elif group_rows * per >= self.PREFIX_TENSOR_ROWS and self._by_tcgen05(D, q, stride):
            tensor = 2 if group_rows * per <= 112 else 1  # one tile: its halves take the keys in turn
            splits = max(1, min(32, 148 // (-(-group_rows * per // 256) * kv * prefix.n_groups)))
        else:
            # eight sequences of four heads behind 1,024 positions: 10.6 us with one block an SM, 15.3 with two, 17.9 with three (the
            # parts that the own keys' kernel has to join grow with them)
            splits = self._splits(tiles * prefix.n_groups, 148) if group_rows else 0
        parts = splits * max(tensor, 1) + own_splits
        scratch = self._scratch(parts * rows * heads * (D + 2))
        o = scratch.data_ptr()
        ml = o + 4 * parts * rows * heads * D
        if not by_mma:
            self.launches += 1
            self._ok(lib.krk_attention_in_parts(out.data_ptr(), None, o, ml, rows, splits, own_splits, None, None, None, None, 0, 0, 1, 1, *step, group_rows,
                                                batch.max_q_len, scale, _code(qkv.dtype), stream), "shared prefix attention")
        elif one_each:
            self.launches += splits > 0
            self._ok(lib.krk_shared_single(out.data_ptr(), o, ml, splits, self._cluster_splits(-(-per // 16) * kv * batch.n_seqs, False), tensor, *step,
                                           cache.k.shape[0], group_rows, scale, error, stream), "shared prefix attention")
        else:
            if tensor:
                self._ok(lib.krk_prefix_tcgen05(o, ml, rows, 0, splits, *step, cache.k.shape[0], group_rows, tensor == 2, scale, error, stream),
                         "prefix attention")
            elif splits:
                self._ok(lib.krk_prefix_few_rows(o, ml, rows, 0, splits, *step, cache.k.shape[0], group_rows, scale, error, stream), "prefix attention")
            self._ok(lib.krk_own_rows(out.data_ptr(), None, o, ml, rows, parts, *step, batch.max_q_len, scale, stream), "attention over own keys")
        return out

    def _scratch(self, n: int):
        """n places of 32 bits, of this call alone; the caller holds them until its launches are queued."""
        return self.error.new_empty(n)

    def _whole_attention(self, out, lse, q, D, batch, cache, pages, scale):
        """Every row over all of its sequence's keys, for what ``_by_mma`` takes; ``lse`` (float32 [rows, heads] or None) takes the base-two
        logarithm of each row's sum. Unlike ``attention``, whatever lies in pages and rows that no query sees."""
        address, stride, heads, kv = q
        rows, per = batch.n_rows, heads // kv
        lib, error, stream = self._parts_lib(D), self.error.data_ptr(), self._stream()
        if lse is None and self._one_each(batch):
            self._ok(lib.krk_shared_single(out.data_ptr(), None, None, 0, self._cluster_splits(-(-per // 16) * kv * batch.n_seqs, True), 0, *q,
                                           *self._segments(batch, cache, None), *pages, cache.k.shape[0], 0, scale, error, stream), "single-token attention")
        elif self._by_tcgen05(D, address, stride) and batch.max_q_len * per >= 128 and self.use_tcgen05_attention:
            if lse is None:
                lse = self._scratch(rows * heads)
            self._ok(self._attn_lib(D).krk_attention_prefill_lse(
                out.data_ptr(), lse.data_ptr(), *q, batch.seq_slot.data_ptr(), batch.seq_start.data_ptr(), batch.seq_qlen.data_ptr(), batch.cu_q.data_ptr(),
                cache.table.data_ptr(), cache.width, *pages, cache.k.shape[0], batch.n_seqs, batch.max_q_len, rows, scale, error, stream), "prompt attention")
        else:
            self._ok(lib.krk_own_rows(out.data_ptr(), _ptr(lse), None, None, rows, 0, *q, *self._segments(batch, cache, None), *pages, batch.max_q_len,
                                      scale, stream), "prompt attention")

    # -- weights per key -------------------------------------------------------------------
    @staticmethod
    def _check_scores(what, cache, scores, positions, out_scores):
        shape, device = (cache.table.shape[0], cache.kv_heads, cache.width * PAGE), cache.k.get_device()
        for t, dtype in ((scores, _F32), (positions, _I32), (None if out_scores is scores else out_scores, _F32)):
            if t is not None and (t.shape != shape or t.dtype is not dtype or not t.is_contiguous() or t.get_device() != device):
                name = "scores" if t is scores else "positions" if t is positions else "out_scores"
                raise KernelError(f"{what}: {name} are contiguous {dtype} [slots, kv heads, rows of a slot] = {list(shape)} beside the cache, "
                                  f"got {t.dtype} {list(t.shape)}")

    def scored_attention(self, qkv, heads, kv_in_row, head_dim, batch, cache, scale, scores, positions=None, observe=None, out_scores=None):
        """``attention`` that also adds up, for every cached row, the weight it receives: ``scores`` [slots, kv heads, rows] float32 grow by
        the softmax weights of the step's queries, summed over the heads of a kv head and over the last ``observe`` queries of each sequence
        (None: all). Rows that the step itself brings start from its own weights; rows behind a sequence's last stay as they are.
        ``positions`` (int32, the same shape) take the step's rows' positions in the sequence, which lie ``batch.seq_shift`` behind their
        rows where keys were evicted. ``out_scores`` takes the sums in place of ``scores``."""
        shift = getattr(batch, "seq_shift", None)
        address, stride, k, v = self._check_step("scored attention", qkv, heads, kv_in_row, head_dim, batch, cache, shift)
        out_scores = scores if out_scores is None else out_scores
        self._check_scores("scored attention", cache, scores, positions, out_scores)
        if observe is not None and observe < 1:
            raise KernelError(f"scored attention: at least one query a sequence is observed, got {observe}")
        if len(set(batch.slots)) != len(batch.slots):
            raise KernelError(f"scored attention: every slot comes once, its sums are one call's; got {list(batch.slots)}")
        lib, rows, kv, per, D = self._parts_lib(head_dim), batch.n_rows, cache.kv_heads, heads // cache.kv_heads, head_dim
        out = qkv.new_empty(rows, heads * D)
        if rows == 0:
            return out
        scale, stream, error, capacity = float(scale), self._stream(), self.error.data_ptr(), cache.width * PAGE
        counts = (scores.data_ptr(), out_scores.data_ptr(), _ptr(positions), _ptr(shift), capacity)
        segments = self._segments(batch, cache, None)
        q, pages = (address, stride, heads, kv), (k, v)
        by_mma = self._by_mma(qkv.dtype, D, address, stride, k, v)
        if by_mma and per <= 16 and self._one_each(batch):
            raw = self._scratch(rows * heads * capacity)
            self._ok(lib.krk_scored_single(out.data_ptr(), raw.data_ptr(), *counts, self._cluster_splits(kv * rows, True), *q, *segments, *pages,
                                           cache.k.shape[0], scale, error, stream), "scored attention")
            return out
        # the output with every row's log sum, then the weights by these
        lse = self._scratch(rows * heads)
        page_blocks = max(1, min(cache.width, -(-888 // (kv * batch.n_seqs))))
        seen = min(batch.max_q_len, observe or batch.max_q_len)
        last = seen if observe else 0  # (0: all; no sequence of the step has more than seen either way)
        if not by_mma:
            parts = self._splits(-(-batch.max_q_len * per // 64) * kv * batch.n_seqs, 444)
            scratch = self._scratch(parts * rows * heads * (D + 2))
            o = scratch.data_ptr()
            self.launches += 2
            self._ok(lib.krk_attention_in_parts(out.data_ptr(), lse.data_ptr(), o, o + 4 * parts * rows * heads * D, rows, 0, parts, *counts, last,
                                                page_blocks, seen, *q, *segments, *pages, 0, batch.max_q_len, scale, _code(qkv.dtype), stream), "scored attention")
            return out
        self._whole_attention(out, lse, q, D, batch, cache, pages, scale)
        if self._by_tcgen05(D, address, stride) and not batch.is_decode and per <= 64:
            longest = cache.width * PAGE if torch.cuda.is_current_stream_capturing() else batch.max_kv_len  # a captured step's sequences grow
            self._ok(lib.krk_key_weights_tcgen05(*counts, lse.data_ptr(), last, *q, *segments, pages[0], cache.k.shape[0], rows, seen, longest,
                                                 scale, error, stream), "weights of keys")
        else:
            self._ok(lib.krk_key_weights(*counts, lse.data_ptr(), last, *q, *segments, pages[0], page_blocks, seen, scale, _code(qkv.dtype),
                                         stream), "weights of keys")
        return out

    # -- eviction ----------------------------------------------------------------------------
    def evict_keys(self, k, v, table, slots, lengths, scores, positions, keep, recent, out_scores=None, out_positions=None, batch=None):
        """Give up all but ``keep`` rows of every head of these cache slots (host lists ``slots`` and ``lengths``, the rows that each holds),
        in every layer run at once (no two of the slots share a page): ``k`` and ``v`` [runs, pages, kv heads, 64, head size], ``table``
        [slots, pages of a slot], ``scores`` and ``positions`` [runs, slots, kv heads, rows]. The ``recent`` rows of highest position stay, of the others those of largest score
        (ties: the lowest row; a NaN counts as the largest). What stays from row ``keep`` on moves, in place, into the rows below it that
        are given up, in ascending order of both; scores and positions move along, or go to ``out_scores`` and ``out_positions`` (rows from
        ``keep`` on are not written). A slot that holds no more than ``keep`` rows stays as it is. ``batch``: the description of a
        single-token step of exactly these slots, whose rows and shifts follow on the device. Returns the rows held now, as a list."""
        what, error = "eviction", self.error
        keep, recent = int(keep), int(recent)
        shape = k.shape
        runs, n_pages, heads, page, dim = shape if len(shape) == 5 else (0, 0, 0, 0, 0)
        if page != PAGE or v.dim() != 5 or v.shape[:4] != shape[:4] or k.dtype != v.dtype:
            raise KernelError(f"{what}: pages are [runs, pages, kv heads, {PAGE}, head size], got {list(shape)} and {list(v.shape)}")
        _code(k.dtype)
        if (k.stride()[1:] != (heads * PAGE * dim, PAGE * dim, dim, 1) or v.stride()[1:] != (heads * PAGE * v.shape[4], PAGE * v.shape[4], v.shape[4], 1)
                or (runs > 1 and (k.stride(0) < n_pages * k.stride(1) or v.stride(0) < n_pages * v.stride(1)))
                or not table.is_contiguous() or table.dtype != torch.int32 or table.dim() != 2):
            raise KernelError(f"{what}: every run's pages and the page table (int32 [slots, pages of a slot]) are contiguous, and runs lie apart")
        out_scores = scores if out_scores is None else out_scores
        out_positions = positions if out_positions is None else out_positions
        n_slots, width = table.shape
        capacity = width * PAGE
        counts = (runs, n_slots, heads, capacity)
        for name, t, dtype in (("scores", scores, torch.float32), ("positions", positions, torch.int32),
                               ("out_scores", out_scores, torch.float32), ("out_positions", out_positions, torch.int32)):
            if t.shape != counts or t.dtype != dtype or not t.is_contiguous() or t.device != error.device:
                raise KernelError(f"{what}: {name} are contiguous {dtype} [runs, slots, kv heads, rows of a slot] = {list(counts)} on {error.device}, "
                                  f"got {t.dtype} {list(t.shape)} on {t.device}")
        self._check_device(what, k, v, table)
        if keep < 1 or not 0 <= recent <= keep:
            raise KernelError(f"{what}: at least one row stays, and at most as many by their position as stay in all; got keep {keep}, recent {recent}")
        n = len(slots)
        if n != len(lengths) or len(set(slots)) != n:
            raise KernelError(f"{what}: every slot comes once, with its length")
        if n == 0:
            return []
        longest = max(lengths)
        if min(slots) < 0 or max(slots) >= n_slots or min(lengths) < 0 or longest > capacity:
            raise KernelError(f"{what}: slots {list(slots)} of {n_slots} with {list(lengths)} rows of {capacity}")
        if batch is not None and (batch.n_seqs != n or batch.n_rows != n or getattr(batch, "seq_shift", None) is None):
            raise KernelError(f"{what}: the step that follows has one token of each slot and keeps shifts")
        if batch is not None:
            self._check_device(what, batch.seq_start, batch.seq_shift)
        left = [keep if m > keep else m for m in lengths]
        if k.numel() == 0:
            return left
        lib, stream, size = self.cache_lib, self._stream(), k.element_size()
        same = v.data_ptr() == k.data_ptr()
        # as many sequences at once as the arguments and the scratch take
        moves = max(0, min(keep, longest - keep))
        most = max(1, min(lib.krk_evict_max_seqs(), n, self.EVICT_SCRATCH_BYTES // max(1, runs * heads * moves * 8)))
        lists = self._scratch(runs * most * heads * (2 * moves + 1))
        head = (k.data_ptr(), None if same else v.data_ptr(), k.stride(0) * size, v.stride(0) * size, dim * size, v.shape[4] * size, heads, runs,
                table.data_ptr(), width, scores.data_ptr(), positions.data_ptr(), out_scores.data_ptr(), out_positions.data_ptr(), scores.stride(0), capacity)
        moves_at = lists.data_ptr()
        counts_at = moves_at + 8 * runs * most * heads * moves
        for at in range(0, n, most):
            part = slots[at:at + most]
            ints = c_int * len(part)
            follow = (None, None, None) if batch is None else (batch.seq_start.data_ptr() + 4 * at, batch.row_pos.data_ptr() + 4 * at,
                                                               batch.seq_shift.data_ptr() + 4 * at)
            self._ok(lib.krk_evict_keys(*head, ints(*part), ints(*lengths[at:at + most]), len(part), keep, recent, moves_at, counts_at, moves, *follow,
                                        stream), what)
        return left
