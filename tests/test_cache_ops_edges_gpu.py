"""The cache's operators where their paths meet (cache_ops_helpers.py has the definitions in 64 bits): values that are no numbers in the prompt
attention with log sums, head sizes whose splits fill shared memory, shares of more pages than the loading warp reads at once."""

import math

import pytest
import torch

from cache_ops_helpers import PAGE, exact_attention, make_batch, make_step
from test_cache_ops_gpu import BF16, DEVICE, F32, groups, ops, within  # noqa: F401

pytestmark = pytest.mark.gpu


def scores_of(cache, kv):
    return torch.zeros((cache.table.shape[0], kv, cache.width * PAGE), device=DEVICE)


@pytest.mark.parametrize("dtype,shape", [(F32, (6, 2, 64)), (BF16, (6, 2, 48)), (BF16, (6, 2, 64)), (BF16, (6, 2, 128)), (BF16, (2, 2, 128)), (BF16, (40, 2, 64)),
                                         (BF16, (66, 2, 128))])
@pytest.mark.parametrize("held", [0, 70, 191])
@pytest.mark.parametrize("operator", ["alone", "scored"])
def test_rows_before_values_that_are_no_numbers(ops, dtype, shape, held, operator):
    """Prompts whose sequences are read each by itself, and counted ones: a value that is no number reaches the rows that see it, in its column, and
    changes nothing else; a key that is none reaches the rows that see it. At the edges of pages, of blocks of 128 keys and of tiles."""
    heads, kv, dim = shape
    starts, brings = [5, held], [130, 400]
    qkv, batch, cache = make_step(DEVICE, dtype, heads, kv, dim, starts, brings, 3 * held + dim)
    assert brings[0] * (heads // kv) >= 128

    def call():
        if operator == "alone":
            return ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, 0.1, groups([2], [0])), None
        scores = scores_of(cache, kv)
        return ops.scored_attention(qkv, heads, kv, dim, batch, cache, 0.1, scores), scores

    exact, off, _, _ = exact_attention(qkv, heads, kv, dim, batch, cache, 0.1)
    clean, sums = call()
    within(clean, exact, off, "without them")
    inf, nan = float("inf"), float("nan")
    clean_v, clean_k = cache.v.clone(), cache.k.clone()
    column = heads * dim // 2 + 3  # of the second kv head's first query head
    per_half = heads // 2 * dim
    for plant in [((33, inf),), ((0, nan),), ((399, -inf),), ((127, inf), (128, -inf)), ((200, inf), (370, nan)), ((63, -inf), (64, -inf))]:
        for token, bad in plant:
            at = held + token
            cache.v[cache.table[batch.slots[1], at // PAGE], 1, at % PAGE, 3] = bad
        got, got_sums = call()
        want = clean.clone()
        # a finite column that holds what is no number from the token on, for every query head of the second kv head
        columns = torch.arange(column, heads * dim, dim, device=DEVICE)
        for token, bad in plant:
            want[brings[0] + token:, columns] += bad
        where = torch.isfinite(want)
        within(got[where], exact[where], off[where], f"{plant}: what does not see them")
        assert torch.equal(torch.isnan(got[~where]), torch.isnan(want[~where])), f"{plant}: what does"
        infinite = torch.isinf(want)
        assert torch.equal(got[infinite], want[infinite]), f"{plant}: infinities keep their signs"
        if sums is not None:
            assert torch.equal(got_sums, sums), f"{plant}: weights depend on no value"
        cache.v.copy_(clean_v)
    for token, bad in [(33, nan), (128, inf), (399, -inf)]:
        at = held + token
        cache.k[cache.table[batch.slots[1], at // PAGE], 0, at % PAGE] = bad
        got, _ = call()
        first = brings[0] + token
        within(got[:first], exact[:first], off[:first], "rows before the key")
        within(got[first:, per_half:], exact[first:, per_half:], off[first:, per_half:], "the other kv head")
        cache.k.copy_(clean_k)
    ops.check()


@pytest.mark.parametrize("shape", [(16, 1, 224), (16, 1, 240), (24, 1, 240), (28, 2, 240)])
@pytest.mark.parametrize("n_seqs", [1, 5, 70])
def test_single_tokens_of_many_large_heads(ops, shape, n_seqs, monkeypatch):
    """Where a cluster's parts and a block's pages would not fit shared memory together, fewer blocks share a sequence's keys."""
    from kernel_rush_kawk_b200.cache import prefix

    heads, kv, dim = shape
    held = [130 + 7 * i for i in range(n_seqs)]
    qkv, batch, cache = make_step(DEVICE, BF16, heads, kv, dim, held, [1] * n_seqs, n_seqs)
    scale = 1 / math.sqrt(dim)
    want, off, weights, weights_off = exact_attention(qkv, heads, kv, dim, batch, cache, scale)
    scores = scores_of(cache, kv)
    within(ops.scored_attention(qkv, heads, kv, dim, batch, cache, scale, scores), want, off, "counted")
    for i, (slot, n) in enumerate(zip(batch.slots, held)):
        within(scores[slot, :, :n + 1], weights[i], weights_off[i], f"weights of sequence {i}")
    within(ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, scale, groups([n_seqs], [0])), want, off, "no prefix, shared")
    monkeypatch.setattr(prefix, "SHARE_BYTES", 1 << 60)
    within(ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, scale, groups([n_seqs], [0])), want, off, "each sequence by itself")
    ops.check()


@pytest.mark.parametrize("heads,kv,dim", [(16, 8, 128), (32, 8, 64)])
def test_shares_of_more_pages_than_the_loading_warp_reads_at_once(ops, heads, kv, dim, monkeypatch):
    """Page numbers come 32 at a time: single tokens whose blocks have 31 to 36 pages each, of two blocks a sequence."""
    from kernel_rush_kawk_b200.cache import prefix

    lengths = [31 * 128, 32 * 128, 33 * 128, 4500, 63, 4095, 64 * 64 + 1, 70 * 64]
    held = [lengths[i % len(lengths)] - 1 for i in range(24)]
    assert ops._cluster_splits(kv * len(held), True) == 2
    qkv, batch, cache = make_step(DEVICE, BF16, heads, kv, dim, held, [1] * len(held), 12)
    scale = 1 / math.sqrt(dim)
    want, off, weights, weights_off = exact_attention(qkv, heads, kv, dim, batch, cache, scale)
    scores = scores_of(cache, kv)
    within(ops.scored_attention(qkv, heads, kv, dim, batch, cache, scale, scores), want, off, "counted")
    for i, (slot, n) in enumerate(zip(batch.slots, held)):
        within(scores[slot, :, :n + 1], weights[i], weights_off[i], f"weights of sequence {i}")
    monkeypatch.setattr(prefix, "SHARE_BYTES", 1 << 60)
    within(ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, scale, groups([len(held)], [0])), want, off, "each sequence by itself")
    ops.check()


@pytest.mark.parametrize("dtype,shape", [(F32, (8, 2, 64)), (BF16, (8, 2, 48)), (BF16, (8, 2, 128)), (BF16, (40, 2, 64)), (BF16, (5, 1, 20))])
@pytest.mark.parametrize("sizes,lengths,own,brings", [([2, 1], [64, 0], [3, 0, 70], [0, 1, 1]), ([3], [128], [0, 70, 5], [1, 0, 1]), ([2, 2], [64, 192], [1, 90, 0, 200], [0, 70, 0, 5]),
                                                     ([1, 2], [0, 0], [0, 64, 9], [0, 0, 150]), ([1, 1], [64, 0], [0, 5], [0, 1])])
@pytest.mark.parametrize("together", [True, False])
def test_sequences_that_bring_nothing(ops, dtype, shape, sizes, lengths, own, brings, together, monkeypatch):
    """Beside others that bring one token or more: these come out as without them, and of the idle ones nothing changes."""
    from kernel_rush_kawk_b200.cache import prefix

    if not together:
        monkeypatch.setattr(prefix, "SHARE_BYTES", 1 << 60)
        monkeypatch.setattr(prefix, "JOIN_STEPS", 1e9)
    heads, kv, dim = shape
    held = [p + o for p, o in zip([p for s, p in zip(sizes, lengths) for _ in range(s)], own)]
    qkv, batch, cache = make_step(DEVICE, dtype, heads, kv, dim, held, brings, 21, (sizes, lengths))
    busy = [i for i, t in enumerate(brings) if t]
    some = make_batch(DEVICE, [batch.slots[i] for i in busy], [held[i] for i in busy], [brings[i] for i in busy])
    want, off, weights, weights_off = exact_attention(qkv, heads, kv, dim, some, cache, 0.1)
    within(ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, 0.1, groups(sizes, lengths)), want, off, "behind prefixes")
    scores = torch.rand((cache.table.shape[0], kv, cache.width * PAGE), device=DEVICE)
    before = scores.clone()
    within(ops.scored_attention(qkv, heads, kv, dim, batch, cache, 0.1, scores), want, off, "counted")
    for j, i in enumerate(busy):
        slot, n, t = batch.slots[i], held[i], brings[i]
        sums = weights[j].clone()
        sums[:, :n] += before[slot, :, :n].double()
        within(scores[slot, :, :n + t], sums, weights_off[j] + sums * 2.0 ** -24, f"weights of sequence {i}")
        before[slot, :, :n + t] = scores[slot, :, :n + t]
    assert torch.equal(scores, before), "other slots"
    ops.check()


@pytest.mark.parametrize("dtype,dim", [(F32, 64), (BF16, 48), (BF16, 128)])
@pytest.mark.parametrize("observe", [2 ** 32 + 5, 2 ** 31, 10 ** 30])
def test_more_observed_queries_than_there_are(ops, dtype, dim, observe):
    """A number beyond 32 bits is as good as all."""
    qkv, batch, cache = make_step(DEVICE, dtype, 8, 2, dim, [60, 0], [9, 40], 4)
    all_of_them, some = scores_of(cache, 2), scores_of(cache, 2)
    ops.scored_attention(qkv, 8, 2, dim, batch, cache, 0.1, all_of_them)
    ops.scored_attention(qkv, 8, 2, dim, batch, cache, 0.1, some, observe=observe)
    assert torch.equal(all_of_them, some)
