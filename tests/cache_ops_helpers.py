"""Shared by the tests of the operators that share and thin out the cache: a cache and a step made by hand, and the operators'
definitions in 64 bits, with how far an arithmetic of the kernels' kind may be off."""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

PAGE = 64
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def make_step(device, dtype, heads, kv, dim, held, brings, seed, groups=None, width=None, row_extra=0, key_std=1.0, q_std=1.5):
    """A cache whose sequences hold ``held`` rows and bring ``brings`` more (already written), and the step of these rows. ``groups``:
    (sizes, lengths) of neighbouring sequences that share their first pages. Everything that belongs to no sequence is NaN: rows behind
    the ends, pages of nobody. Slots are in no order, and there are more of them than sequences."""
    g = torch.Generator().manual_seed(seed)
    host = random.Random(seed)
    n = len(held)
    need = [-(-(h + t) // PAGE) for h, t in zip(held, brings)]
    width = width or max(need) + 1
    n_slots = n + 2
    slots = host.sample(range(n_slots), n)
    pages = list(range(sum(need) + 3))
    host.shuffle(pages)
    n_pages = len(pages)
    nan = float("nan")
    k = torch.full((n_pages, kv, PAGE, dim), nan)
    v = torch.full((n_pages, kv, PAGE, dim), nan)
    table = torch.full((n_slots, width), n_pages - 1, dtype=torch.int32)
    group_of = [i for i, s in enumerate(groups[0]) for _ in range(s)] if groups else list(range(n))
    shared = {}
    for s in range(n):
        old = shared.get(group_of[s])
        start = len(old) * PAGE if old else 0
        mine = (old or []) + [pages.pop() for _ in range(need[s] - len(old or []))]
        if groups and old is None:
            shared[group_of[s]] = mine[:groups[1][group_of[s]] // PAGE]
        for p in range(start, held[s] + brings[s]):
            k[mine[p // PAGE], :, p % PAGE] = torch.randn((kv, dim), generator=g) * key_std
            v[mine[p // PAGE], :, p % PAGE] = torch.randn((kv, dim), generator=g)
        table[slots[s], :need[s]] = torch.tensor(mine, dtype=torch.int32)
    rows = sum(brings)
    wide = torch.randn((rows, (heads + 2 * kv) * dim + row_extra), generator=g)
    wide[:, :heads * dim] *= q_std
    qkv = wide.to(dtype).to(device)[:, :(heads + 2 * kv) * dim]
    cache = SimpleNamespace(k=k.to(dtype).to(device), v=v.to(dtype).to(device), table=table.to(device), width=width, window=None, kv_heads=kv,
                            head_dim=dim, v_dim=dim, keep_pages=0)
    return qkv, make_batch(device, slots, held, brings), cache


def make_batch(device, slots, starts, brings):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    cu = [0]
    for t in brings:
        cu.append(cu[-1] + t)
    return SimpleNamespace(n_rows=cu[-1], n_seqs=len(slots), slots=list(slots), starts=list(starts), q_lens=list(brings),
                           row_seq=i32([s for s, t in enumerate(brings) for _ in range(t)]),
                           row_pos=i32([p + i for p, t in zip(starts, brings) for i in range(t)]), seq_slot=i32(slots), seq_start=i32(starts),
                           seq_qlen=i32(brings), cu_q=i32(cu), max_q_len=max(brings), max_kv_len=max(a + b for a, b in zip(starts, brings)),
                           is_decode=max(brings) == 1)


def exact_attention(qkv, heads, kv, dim, batch, cache, scale, observe=None):
    """In 64 bits: output [rows, heads * dim], how far it may be off, and per sequence the weights [kv, rows held] that its keys receive
    from the last ``observe`` queries with how far these may be off.

    A score of float32 products and sums, in any order, is off by at most (dim + 2) half steps of the sum of magnitudes (twice that where the
    tensor cores cut off instead of rounding); a weight relatively by twice the scores' error (its own and its denominator's), the
    exponentials' 2^-21 (two of them, in float32 or approximate, and the rounding of their arguments, which are below 2^5 times the spread of the
    scores), and the sum's keys * 2^-24. Weights rounded to the rows' dtype before they meet the values add half a step of the sum of
    weight times value's magnitude, the output's rounding half a step of it."""
    dtype = qkv.dtype
    per = heads // kv
    out, off, weights, weights_off = [], [], [], []
    row = 0
    for slot, start, t in zip(batch.slots, batch.starts, batch.q_lens):
        total = start + t
        where = torch.arange(total, device=qkv.device)
        page = cache.table[slot].long()[where // PAGE]
        k = cache.k[page, :, where % PAGE].double().transpose(0, 1).repeat_interleave(per, 0)  # [heads, keys, dim]
        v = cache.v[page, :, where % PAGE].double().transpose(0, 1).repeat_interleave(per, 0)
        q = qkv[row:row + t, :heads * dim].double().view(t, heads, dim).transpose(0, 1)
        s = q @ k.transpose(1, 2) * scale
        size = q.abs() @ k.abs().transpose(1, 2) * abs(scale)
        seen = where[None, :] <= start + torch.arange(t, device=qkv.device)[:, None]
        s = s.masked_fill(~seen, -math.inf)
        w = torch.softmax(s, dim=-1)
        spread = s.masked_fill(~seen, 0).abs().amax(dim=(1, 2), keepdim=True)
        rel = 2 * (2 * (dim + 2) * 2.0 ** -24 * size.amax(dim=(1, 2), keepdim=True)) + 2.0 ** -21 * (1 + spread) + (total + 16) * 2.0 ** -24
        o = w @ v
        mag = w @ v.abs()
        # the rows' error acts on numerator and denominator alike
        out.append(o.transpose(0, 1).reshape(t, heads * dim))
        off.append((mag * (2 * rel + (HALF[dtype] if dtype != torch.float32 else 0)) + o.abs() * HALF[dtype] * 1.001).transpose(0, 1).reshape(t, heads * dim))
        last = t if observe is None else min(t, observe)
        got = w[:, t - last:].view(kv, per, last, total)
        weights.append(got.sum(dim=(1, 2)))
        weights_off.append((got * (2 * rel).view(kv, per, 1, 1)).sum(dim=(1, 2)) + got.sum(dim=(1, 2)) * per * last * 2.0 ** -24 + 1e-30)
        row += t
    return torch.cat(out), torch.cat(off), weights, weights_off


def exact_evict(k, v, table, slots, lengths, scores, positions, keep, recent):
    """The eviction by its definition, row by row, in place on copies: (k, v, scores, positions)."""
    k, v, scores, positions = k.clone(), v.clone(), scores.clone(), positions.clone()
    for slot, n in zip(slots, lengths):
        if n <= keep:
            continue
        page = [int(p) for p in table[slot]]
        for run in range(k.shape[0]):
            for h in range(k.shape[2]):
                pos = positions[run, slot, h, :n].tolist()
                val = [math.inf if x != x else x for x in scores[run, slot, h, :n].tolist()]
                nan = [x != x for x in scores[run, slot, h, :n].tolist()]
                newest = set(sorted(range(n), key=lambda r: (-pos[r], r))[:recent])
                rest = sorted((r for r in range(n) if r not in newest), key=lambda r: (not nan[r], -val[r], r))
                kept = newest | set(rest[:keep - recent])
                free = [r for r in range(keep) if r not in kept]
                moved = [r for r in range(keep, n) if r in kept]
                assert len(free) == len(moved)
                for d, s in zip(free, moved):
                    for pool in (k, v):
                        pool[run, page[d // PAGE], h, d % PAGE] = pool[run, page[s // PAGE], h, s % PAGE]
                    scores[run, slot, h, d] = scores[run, slot, h, s]
                    positions[run, slot, h, d] = positions[run, slot, h, s]
    return k, v, scores, positions
