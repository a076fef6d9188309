"""The operators that share and thin out the cache, each alone against its definition in 64 bits (cache_ops_helpers.py, which
also says how far the kernels' arithmetic may be off). Rows and pages that no query sees are NaN throughout."""

import math
import random

import pytest
import torch

from cache_ops_helpers import PAGE, exact_attention, exact_evict, make_batch, make_step

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
DEVICE = "cuda"


@pytest.fixture(scope="module")
def ops():
    from kernel_rush_kawk_b200.csrc import load_kernels

    return load_kernels(())


@pytest.fixture(autouse=True)
def always_shared(monkeypatch):
    """Small cases take the kernels that large ones do."""
    from kernel_rush_kawk_b200.cache import prefix

    monkeypatch.setattr(prefix, "SHARE_BYTES", 0)
    monkeypatch.setattr(prefix, "JOIN_STEPS", -1e9)


def groups(sizes, lengths):
    from kernel_rush_kawk_b200.cache.prefix import PrefixGroups

    return PrefixGroups(sizes, lengths, DEVICE)


def within(got, want, off, what):
    bad = ~((got.double() - want).abs() <= off)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, first at {at}: {got[tuple(at)].item()} for "
                             f"{want[tuple(at)].item()}, allowed {off[tuple(at)].item():.3g}")


SHAPES = [(4, 2, 16), (6, 2, 32), (5, 1, 48), (8, 8, 64), (16, 4, 64), (14, 2, 80), (32, 8, 128), (40, 2, 128), (6, 2, 256)]
# (sizes, shared lengths, rows held behind the prefix, tokens): alone, a group without a prefix, odd numbers of pages, a token
# that opens a page, one that fills one, pieces of unequal lengths, more rows than a tile
GROUPS = [
    ([1], [64], [0], [1]),
    ([3], [128], [0, 63, 64], [1, 1, 1]),
    ([2, 1, 4], [192, 0, 320], [5, 130, 1, 0, 127, 64, 200], [1] * 7),
    ([9], [704], [3, 17, 64, 0, 99, 1, 255, 31, 8], [1] * 9),
    ([2, 3], [64, 192], [0, 0, 0, 0, 0], [5, 70, 1, 33, 64]),
    ([1, 2], [0, 128], [0, 10, 140], [1, 90, 131]),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_shared_prefix_attention(ops, dtype, shape, case):
    heads, kv, dim = shape
    sizes, lengths, own, brings = GROUPS[case]
    held = [p + o for p, o in zip([p for s, p in zip(sizes, lengths) for _ in range(s)], own)]
    qkv, batch, cache = make_step(DEVICE, dtype, heads, kv, dim, held, brings, 7 * case + dim, (sizes, lengths), row_extra=8 * (case % 2))
    scale = 1 / math.sqrt(dim)
    got = ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, scale, groups(sizes, lengths))
    want, off, _, _ = exact_attention(qkv, heads, kv, dim, batch, cache, scale)
    within(got, want, off, "shared prefix attention")
    again = ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, scale, groups(sizes, lengths))
    assert torch.equal(got, again), "the same call gives the same bits"
    ops.check()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
@pytest.mark.parametrize("dim", [48, 128])
def test_shared_prefix_attention_of_other_scales(ops, dtype, scale, dim):
    """A negative scale, none, and one that leaves a single key with weight."""
    qkv, batch, cache = make_step(DEVICE, dtype, 8, 2, dim, [320 + o for o in (0, 5, 70)], [1, 1, 1], 5, ([3], [320]))
    got = ops.shared_prefix_attention(qkv, 8, 2, dim, batch, cache, scale, groups([3], [320]))
    want, off, _, _ = exact_attention(qkv, 8, 2, dim, batch, cache, scale)
    within(got, want, off, f"scale {scale}")


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n_seqs,length", [(10, 320), (40, 192)])
def test_shared_prefix_attention_of_many_rows_and_other_scales(ops, n_seqs, length, dim, scale):
    """Rows that fill a tile in part, or two, and an odd number of pages."""
    qkv, batch, cache = make_step(DEVICE, BF16, 8, 2, dim, [length + i for i in range(n_seqs)], [1] * n_seqs, 5, ([n_seqs], [length]))
    got = ops.shared_prefix_attention(qkv, 8, 2, dim, batch, cache, scale, groups([n_seqs], [length]))
    want, off, _, _ = exact_attention(qkv, 8, 2, dim, batch, cache, scale)
    within(got, want, off, f"scale {scale}")


@pytest.mark.parametrize("dtype,dim", [(F32, 48), (BF16, 48), (BF16, 128)])
def test_shared_prefix_attention_of_captured_pieces(ops, dtype, dim):
    """A captured step of several tokens a sequence, replayed for a group with more sequences than the step was captured for."""
    heads, kv, n, each = 8, 2, 5, 9
    qkv, batch, cache = make_step(DEVICE, dtype, heads, kv, dim, [256 + 3 * i for i in range(n)], [each] * n, 6, ([n], [256]))
    prefix = groups([3, 2], [128, 64])
    call = lambda: ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, 0.2, prefix)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    want, off, _, _ = exact_attention(qkv, heads, kv, dim, batch, cache, 0.2)
    for sizes, lengths in (([3, 2], [128, 64]), ([4, 1], [256, 0]), ([1, 4], [64, 192])):
        prefix.update(groups(sizes, lengths))
        out.fill_(float("nan"))
        graph.replay()
        within(out, want, off, f"replayed for {sizes}")


@pytest.mark.parametrize("n_seqs,length,dim", [(64, 2048, 128), (70, 1088, 64), (33, 4032, 128), (5, 16384, 128)])
def test_shared_prefix_attention_of_many_rows(ops, n_seqs, length, dim):
    """More rows than several tiles, long prefixes, odd numbers of pages: the sizes of a server."""
    host = random.Random(n_seqs)
    held = [length + host.randint(0, 300) for _ in range(n_seqs)]
    qkv, batch, cache = make_step(DEVICE, BF16, 16, 4, dim, held, [1] * n_seqs, 3, ([n_seqs], [length]))
    got = ops.shared_prefix_attention(qkv, 16, 4, dim, batch, cache, 1 / math.sqrt(dim), groups([n_seqs], [length]))
    want, off, _, _ = exact_attention(qkv, 16, 4, dim, batch, cache, 1 / math.sqrt(dim))
    within(got, want, off, "shared prefix attention of many rows")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_prefix_attention_in_a_captured_step(ops, dtype):
    """Captured once, replayed for other lengths, other pages and other groups of the same number and size, beside eager calls on another
    stream: what a call uses is its own."""
    heads, kv, dim = 8, 2, 128
    first = make_step(DEVICE, dtype, heads, kv, dim, [64 + 3, 64 + 9, 128 + 70], [1] * 3, 1, ([2, 1], [64, 128]), width=9)
    then = make_step(DEVICE, dtype, heads, kv, dim, [256 + 90, 256 + 1, 65], [1] * 3, 2, ([2, 1], [256, 64]), width=9)
    scale = 1 / math.sqrt(dim)
    qkv, batch, cache = first
    prefix = groups([2, 1], [64, 128])
    # the second step's pages in the first one's pool
    pool_k, pool_v = torch.zeros_like(torch.cat([first[2].k, then[2].k])), torch.zeros_like(torch.cat([first[2].v, then[2].v]))
    n = first[2].k.shape[0]
    pool_k[:n], pool_v[:n], pool_k[n:], pool_v[n:] = first[2].k, first[2].v, then[2].k, then[2].v
    cache.k, cache.v = pool_k, pool_v
    call = lambda: ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, scale, prefix)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    want, off, _, _ = exact_attention(qkv, heads, kv, dim, batch, cache, scale)
    within(out, want, off, "replayed")
    other_qkv, other, other_cache = then
    qkv.copy_(other_qkv)
    for name in ("seq_slot", "seq_start", "row_pos"):
        getattr(batch, name).copy_(getattr(other, name))
    batch.slots, batch.starts = other.slots, other.starts
    cache.table.copy_(other_cache.table + n)
    prefix.update(groups([2, 1], [256, 64]))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            eager = ops.shared_prefix_attention(other_qkv, heads, kv, dim, other, other_cache, scale, prefix)
    graph.replay()
    torch.cuda.synchronize()
    want, off, _, _ = exact_attention(qkv, heads, kv, dim, batch, cache, scale)
    within(out, want, off, "replayed for another step")
    assert torch.equal(out, eager)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [20, 48, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_shared_prefix_attention_beside_keys_that_are_no_numbers(ops, dtype, dim, bad):
    """A token whose key and value are no numbers spoils the rows that see it, and no row before it nor any other sequence."""
    heads, kv = 6, 2
    held, brings = [128, 128 + 70], [40, 90]
    qkv, batch, cache = make_step(DEVICE, dtype, heads, kv, dim, held, brings, 9, ([2], [128]))
    call = lambda: ops.shared_prefix_attention(qkv, heads, kv, dim, batch, cache, 0.1, groups([2], [128]))
    want = call()
    at = held[1] + 33  # a token in the middle of the second sequence's
    page = cache.table[batch.slots[1], at // PAGE]
    cache.v[page, 1, at % PAGE, 3] = bad
    cache.k[page, 0, at % PAGE] = bad
    got = call()
    first = brings[0] + 33
    assert torch.equal(got[:first], want[:first]), "rows that do not see it"
    assert not torch.isfinite(got[first:, heads * dim // 2 + 3]).any(), "rows that do"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(5, 1, 48), (16, 4, 64), (32, 8, 128), (40, 2, 128)])
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_each_sequence_by_itself(ops, dtype, shape, case, monkeypatch):
    """Groups that do not pay: the same definition through each sequence's own table."""
    from kernel_rush_kawk_b200.cache import prefix

    monkeypatch.setattr(prefix, "SHARE_BYTES", 1 << 60)
    monkeypatch.setattr(prefix, "JOIN_STEPS", 1e9)
    test_shared_prefix_attention(ops, dtype, shape, case)


# -- weights per key -----------------------------------------------------------------------------------------
SCORED = [
    ([0], [1], None), ([63], [1], None), ([64, 700, 5], [1, 1, 1], 4), ([0, 0, 0], [1, 64, 200], None), ([0, 0], [130, 65], 32),
    ([100, 0, 70], [1, 129, 90], 7), ([1500] * 3 + [9] * 9, [1] * 12, None),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("case", range(len(SCORED)))
def test_scored_attention(ops, dtype, shape, case):
    heads, kv, dim = shape
    held, brings, observe = SCORED[case]
    qkv, batch, cache = make_step(DEVICE, dtype, heads, kv, dim, held, brings, case + dim, row_extra=8 * (case % 2))
    scale = 1 / math.sqrt(dim)
    shape = (cache.table.shape[0], kv, cache.width * PAGE)
    g = torch.Generator(DEVICE).manual_seed(case)
    scores = torch.rand(shape, generator=g, device=DEVICE) * 4
    positions = torch.full(shape, -7, dtype=torch.int32, device=DEVICE)
    before, before_pos = scores.clone(), positions.clone()
    want, off, weights, weights_off = exact_attention(qkv, heads, kv, dim, batch, cache, scale, observe)
    apart = torch.full(shape, -3.0, device=DEVICE)
    out = ops.scored_attention(qkv, heads, kv, dim, batch, cache, scale, scores, positions=None, observe=observe, out_scores=apart)
    assert torch.equal(scores, before) and torch.equal(positions, before_pos)
    batch.seq_shift = torch.arange(1, batch.n_seqs + 1, dtype=torch.int32, device=DEVICE) * 1000
    got = ops.scored_attention(qkv, heads, kv, dim, batch, cache, scale, scores, positions=positions, observe=observe)
    assert torch.equal(got, out)
    within(got, want, off, "output")
    for i, (slot, start, t) in enumerate(zip(batch.slots, batch.starts, batch.q_lens)):
        sums = weights[i].clone()
        sums[:, :start] += before[slot, :, :start].double()
        allowed = weights_off[i] + sums * 2.0 ** -24
        within(scores[slot, :, :start + t], sums, allowed, f"weights of sequence {i}")
        assert torch.equal(apart[slot, :, :start + t], scores[slot, :, :start + t])
        assert (positions[slot, :, start:start + t] == torch.arange(start, start + t, device=DEVICE, dtype=torch.int32) + 1000 * (i + 1)).all()
        before[slot, :, :start + t] = scores[slot, :, :start + t]
        before_pos[slot, :, start:start + t] = positions[slot, :, start:start + t]
        apart[slot, :, :start + t] = -3.0
    assert torch.equal(scores, before) and torch.equal(positions, before_pos), "rows behind the sequences' ends, and other slots, stay"
    assert (apart == -3.0).all()
    ops.check()


@pytest.mark.parametrize("held,brings,observe", [([3000, 4090, 2], [1, 1, 1], None), ([0], [2100], None), ([0, 0], [1300, 700], 64), ([900], [1100], 200),
                                               ([0, 0, 0], [1300, 40, 1100], None), ([0, 100], [1900, 130], None)])
@pytest.mark.parametrize("dim", [64, 128])
def test_scored_attention_of_long_sequences(ops, held, brings, observe, dim):
    heads, kv = 12, 4
    qkv, batch, cache = make_step(DEVICE, BF16, heads, kv, dim, held, brings, 11)
    scores = torch.zeros((cache.table.shape[0], kv, cache.width * PAGE), device=DEVICE)
    want, off, weights, weights_off = exact_attention(qkv, heads, kv, dim, batch, cache, 0.1, observe)
    got = ops.scored_attention(qkv, heads, kv, dim, batch, cache, 0.1, scores, observe=observe)
    within(got, want, off, "output")
    for i, (slot, start, t) in enumerate(zip(batch.slots, batch.starts, batch.q_lens)):
        within(scores[slot, :, :start + t], weights[i], weights_off[i], f"weights of sequence {i}")
        assert (scores[slot, :, start + t:] == 0).all()


def test_scored_attention_in_a_captured_step(ops):
    """A captured step replayed while the sequences grow: sums add up over the replays."""
    heads, kv, dim, steps = 8, 2, 128, 5
    held = [61, 300, 0]
    qkv, batch, cache = make_step(DEVICE, BF16, heads, kv, dim, [h + steps for h in held], [1] * 3, 4)
    batch = make_batch(DEVICE, batch.slots, held, [1] * 3)
    shape = (cache.table.shape[0], kv, cache.width * PAGE)
    scores, positions = torch.zeros(shape, device=DEVICE), torch.zeros(shape, dtype=torch.int32, device=DEVICE)
    call = lambda: ops.scored_attention(qkv, heads, kv, dim, batch, cache, 0.1, scores, positions)
    call()
    scores.zero_()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    want, allowed = torch.zeros(shape, dtype=torch.float64, device=DEVICE), torch.zeros(shape, dtype=torch.float64, device=DEVICE)
    for _ in range(steps):
        graph.replay()
        _, _, weights, weights_off = exact_attention(qkv, heads, kv, dim, batch, cache, 0.1)
        for i, (slot, start) in enumerate(zip(batch.slots, batch.starts)):
            want[slot, :, :start + 1] += weights[i]
            allowed[slot, :, :start + 1] += weights_off[i] + want[slot, :, :start + 1] * 2.0 ** -24
        batch.starts = [s + 1 for s in batch.starts]
        batch.seq_start += 1
        batch.row_pos += 1
    within(scores, want, allowed, "sums over replays")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scored_attention_of_captured_pieces(ops, dtype):
    """A captured step of several tokens a sequence, replayed for sequences that have grown over pages that the captured one did not see."""
    heads, kv, dim, each, later = 8, 2, 128, 5, 500
    held = [40, 0]
    qkv, batch, cache = make_step(DEVICE, dtype, heads, kv, dim, [h + later for h in held], [each] * 2, 4)
    batch = make_batch(DEVICE, batch.slots, held, [each] * 2)
    scores = torch.zeros((cache.table.shape[0], kv, cache.width * PAGE), device=DEVICE)
    call = lambda: ops.scored_attention(qkv, heads, kv, dim, batch, cache, 0.1, scores)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    batch.starts = [s + later for s in batch.starts]
    batch.seq_start += later
    batch.row_pos += later
    scores.zero_()
    graph.replay()
    want, off, weights, weights_off = exact_attention(qkv, heads, kv, dim, batch, cache, 0.1)
    within(out, want, off, "output")
    for i, (slot, start) in enumerate(zip(batch.slots, batch.starts)):
        within(scores[slot, :, :start + each], weights[i], weights_off[i], f"weights of sequence {i}")


# -- eviction ---------------------------------------------------------------------------------------------------
def evict_case(dtype, runs, kv, dim, width, seed, n_slots=5, ties=True):
    g = torch.Generator(DEVICE).manual_seed(seed)
    n_pages = n_slots * width + 3
    k = torch.randn((runs, n_pages, kv, PAGE, dim), generator=g, device=DEVICE).to(dtype)
    v = torch.randn((runs, n_pages, kv, PAGE, dim), generator=g, device=DEVICE).to(dtype)
    table = torch.randperm(n_pages, generator=g, device=DEVICE)[:n_slots * width].view(n_slots, width).int().contiguous()
    scores = torch.randn((runs, n_slots, kv, width * PAGE), generator=g, device=DEVICE)
    if ties:
        scores = (scores * 2).round() / 2  # many equal ones, both zeros among them
    positions = torch.argsort(torch.rand(scores.shape, generator=g, device=DEVICE), dim=-1).int()
    return k, v, table, scores, positions


@pytest.mark.parametrize("dtype,dim", [(F32, 48), (BF16, 128), (BF16, 20), (BF16, 6), (F32, 2)])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (64, 10), (100, 100), (77, 0), (130, 33)])
def test_evict_keys(ops, dtype, dim, keep, recent):
    runs, kv, width = 2, 3, 4
    k, v, table, scores, positions = evict_case(dtype, runs, kv, dim, width, keep + dim)
    slots, lengths = [3, 0, 4, 1], [256, 131, keep, max(keep - 1, 0)]
    want = exact_evict(k, v, table, slots, lengths, scores, positions, keep, recent)
    # apart first: what is read stays
    out_scores, out_positions = torch.full_like(scores, 9.5), torch.full_like(positions, -5)
    k2, v2 = k.clone(), v.clone()
    left = ops.evict_keys(k2, v2, table, slots, lengths, scores, positions, keep, recent, out_scores=out_scores, out_positions=out_positions)
    assert left == [min(n, keep) for n in lengths]
    assert torch.equal(k2, want[0]) and torch.equal(v2, want[1])
    for slot, n in zip(slots, left):
        assert torch.equal(out_scores[:, slot, :, :n], want[2][:, slot, :, :n]) and torch.equal(out_positions[:, slot, :, :n], want[3][:, slot, :, :n])
        out_scores[:, slot, :, :n], out_positions[:, slot, :, :n] = 9.5, -5
    assert (out_scores == 9.5).all() and (out_positions == -5).all(), "rows that are not held stay as they were"
    ops.evict_keys(k, v, table, slots, lengths, scores, positions, keep, recent)
    for got, ref in zip((k, v, scores, positions), want):
        assert torch.equal(got, ref)


@pytest.mark.parametrize("fill", ["equal", "nan", "inf", "descending"])
def test_evict_keys_of_odd_scores(ops, fill):
    """All equal (ties go to the lowest rows), NaN and infinities among them, both zeros, and scores in order."""
    k, v, table, scores, positions = evict_case(BF16, 1, 2, 16, 8, 3, ties=False)
    if fill == "equal":
        scores.fill_(0.0)
        scores[..., ::3] = -0.0
    elif fill == "nan":
        scores[..., 100:340:7] = float("nan")
        scores[..., 101:340:11] = -float("nan")
    elif fill == "inf":
        scores[..., ::2] = -float("inf")
        scores[..., 5:500:50] = float("inf")
    else:
        scores = torch.arange(scores.shape[-1], 0, -1, device=DEVICE).float().expand_as(scores).contiguous()
    slots, lengths = [2, 1], [512, 411]
    want = exact_evict(k, v, table, slots, lengths, scores, positions, 200, 40)
    ops.evict_keys(k, v, table, slots, lengths, scores, positions, 200, 40)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1]) and torch.equal(positions, want[3])
    assert torch.equal(scores.view(torch.int32), want[2].view(torch.int32)), "moved to the bit"


def test_evict_keys_of_many_rows_and_sequences(ops):
    """Longer than one pass of a block, more sequences than one launch takes, scratch that only some of them fit, keys that serve
    as values, runs of a larger storage."""
    k, v, table, scores, positions = evict_case(BF16, 2, 1, 16, 90, 8, n_slots=2, ties=True)
    want = exact_evict(k, v, table, [1], [5700], scores, positions, 1100, 500)
    ops.evict_keys(k, v, table, [1], [5700], scores, positions, 1100, 500)
    for got, ref in zip((k, v, scores, positions), want):
        assert torch.equal(got, ref)
    # as long that the keys of a head do not fit shared memory; by torch's own sort
    k, v, table, scores, positions = evict_case(F32, 1, 2, 4, 500, 10, n_slots=1, ties=True)
    L, keep, recent = 31000, 9000, 700
    rank = scores[0, 0, :, :L].clone()
    rank.scatter_(-1, positions[0, 0, :, :L].argsort(dim=-1, descending=True)[:, :recent], float("inf"))
    kept = rank.sort(dim=-1, descending=True, stable=True).indices[:, :keep].sort(dim=-1).values
    before = [k.clone(), positions.clone()]
    ops.evict_keys(k, v, table, [0], [L], scores, positions, keep, recent)
    for h in range(2):
        stay = set(kept[h].tolist())
        src = list(range(keep))
        for d, s in zip([r for r in range(keep) if r not in stay], [r for r in sorted(stay) if r >= keep]):
            src[d] = s
        src = torch.tensor(src, device=DEVICE)
        assert torch.equal(positions[0, 0, h, :keep], before[1][0, 0, h, src])
        page, old = table[0].long()[torch.arange(keep, device=DEVICE) // PAGE], table[0].long()[src // PAGE]
        assert torch.equal(k[0, page, h, torch.arange(keep, device=DEVICE) % PAGE], before[0][0, old, h, src % PAGE])
    n = 150
    k, v, table, scores, positions = evict_case(BF16, 1, 1, 8, 2, 9, n_slots=n)
    slots, lengths = list(range(n - 1, -1, -1)), [70 + i % 59 for i in range(n)]
    want = exact_evict(k, k, table, slots, lengths, scores, positions, 69, 5)
    saved = ops.EVICT_SCRATCH_BYTES
    try:
        type(ops).EVICT_SCRATCH_BYTES = 20000
        ops.evict_keys(k, k, table, slots, lengths, scores, positions, 69, 5)
    finally:
        type(ops).EVICT_SCRATCH_BYTES = saved
    assert torch.equal(k, want[0]) and torch.equal(scores, want[2]) and torch.equal(positions, want[3])


@pytest.mark.parametrize("L,keep,recent", [(6001, 40, 7), (9000, 5000, 1), (23000, 2048, 2048), (23001, 64, 3)])
def test_evict_keys_of_few_long_heads(ops, L, keep, recent):
    """On both sides of the lengths at which the blocks change."""
    k, v, table, scores, positions = evict_case(BF16, 1, 2, 4, -(-L // PAGE), L, n_slots=1, ties=False)
    want = exact_evict(k, v, table, [0], [L], scores, positions, keep, recent)
    assert ops.evict_keys(k, v, table, [0], [L], scores, positions, keep, recent) == [keep]
    for got, ref in zip((k, v, scores, positions), want):
        assert torch.equal(got, ref)


def test_evict_keys_moves_the_step_on(ops):
    """A single-token step of the evicted slots: rows fall back, shifts take what was given up."""
    k, v, table, scores, positions = evict_case(BF16, 1, 2, 16, 4, 3)
    batch = make_batch(DEVICE, [3, 0, 1], [200, 64, 20], [1, 1, 1])
    batch.seq_shift = torch.tensor([5, 0, 7], dtype=torch.int32, device=DEVICE)
    ops.evict_keys(k, v, table, [3, 0, 1], [200, 64, 20], scores, positions, 64, 3, batch=batch)
    assert batch.seq_start.tolist() == [64, 64, 20] and batch.row_pos.tolist() == [64, 64, 20] and batch.seq_shift.tolist() == [141, 0, 7]


# -- one after the other ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_steps_and_evictions_together(ops, dtype):
    """Prompts, single tokens and evictions in turn, as a server runs them: after each step the output is the attention over the rows that the
    definition keeps, and the sums and positions are the definition's."""
    heads, kv, dim, keep, recent, width = 6, 2, 64, 70, 20, 5
    n_slots, n_pages = 3, 15
    g = torch.Generator(DEVICE).manual_seed(1)
    k = torch.zeros((1, n_pages, kv, PAGE, dim), dtype=dtype, device=DEVICE)
    v = torch.zeros_like(k)
    table = torch.randperm(n_pages, generator=g, device=DEVICE).view(n_slots, width).int()
    scores = torch.zeros((1, n_slots, kv, width * PAGE), device=DEVICE)
    positions = torch.zeros(scores.shape, dtype=torch.int32, device=DEVICE)
    from types import SimpleNamespace
    cache = SimpleNamespace(k=k[0], v=v[0], table=table, width=width, window=None, kv_heads=kv, head_dim=dim, v_dim=dim, keep_pages=0)
    slots, held, gone = [2, 0], [0, 0], [0, 0]
    for step in range(14):
        brings = [150, 90] if step == 0 else [1, 1] if step % 5 else [40, 3]
        batch = make_batch(DEVICE, slots, held, brings)
        batch.seq_shift = torch.tensor(gone, dtype=torch.int32, device=DEVICE)
        qkv = torch.randn((batch.n_rows, (heads + 2 * kv) * dim), generator=g, device=DEVICE).to(dtype)
        ops.qk_norm_rope_write(qkv, heads, kv, dim, None, None, 1e-6, None, None, batch, cache)
        want, off, weights, weights_off = exact_attention(qkv, heads, kv, dim, batch, cache, 0.2)
        before = scores.clone()
        out = ops.scored_attention(qkv, heads, kv, dim, batch, cache, 0.2, scores[0], positions[0])
        within(out, want, off, f"step {step}")
        for i, slot in enumerate(slots):
            sums = weights[i].clone()
            sums[:, :held[i]] += before[0, slot, :, :held[i]].double()
            within(scores[0, slot, :, :held[i] + brings[i]], sums, weights_off[i] + sums * 2.0 ** -24, f"sums, step {step}")
        held = [h + t for h, t in zip(held, brings)]
        ref = exact_evict(k, v, table, slots, held, scores, positions, keep, recent)
        left = ops.evict_keys(k, v, table, slots, held, scores, positions, keep, recent)
        for got, r in zip((k, v, scores, positions), ref):
            assert torch.equal(got, r)
        gone = [a + h - n for a, h, n in zip(gone, held, left)]
        held = left
        for i, slot in enumerate(slots):  # the newest positions are among them, each once
            last = held[i] + gone[i]
            for h in range(kv):
                got = positions[0, slot, h, :held[i]].tolist()
                assert len(set(got)) == len(got) and set(range(last - min(recent, held[i]), last)) <= set(got)
    ops.check()


# -- refusals ------------------------------------------------------------------------------------------------------
def test_refusals(ops):
    from kernel_rush_kawk_b200.cache import CacheError
    from kernel_rush_kawk_b200.csrc import KernelError

    qkv, batch, cache = make_step(DEVICE, BF16, 4, 2, 32, [70, 80], [1, 1], 1, ([2], [64]))
    good = dict(qkv=qkv, heads=4, kv=2, dim=32, batch=batch, cache=cache)

    def shared(prefix=None, **change):
        a = {**good, **change}
        return ops.shared_prefix_attention(a["qkv"], a["heads"], a["kv"], a["dim"], a["batch"], a["cache"], 0.1, prefix or groups([2], [64]))

    shared()
    from types import SimpleNamespace
    for error, change in [(KernelError, dict(qkv=qkv[:, :-1])), (KernelError, dict(qkv=qkv.float())), (KernelError, dict(heads=3)),
                          (KernelError, dict(cache=SimpleNamespace(**{**vars(cache), "window": 64}))), (KernelError, dict(qkv=qkv[:1])),
                          (KernelError, dict(qkv=qkv.t().contiguous().t())), (CacheError, dict(prefix=groups([3], [64]))),
                          (KernelError, dict(qkv=qkv.as_strided(qkv.shape, (qkv.shape[1] - 64, 1)))),
                          (KernelError, dict(batch=SimpleNamespace(**{**vars(batch), "max_kv_len": cache.width * PAGE + 1}))),
                          (KernelError, dict(cache=SimpleNamespace(**{**vars(cache), "k": cache.k[:, :1]}))),
                          (CacheError, dict(prefix=groups([2], [128]))), (CacheError, dict(prefix=groups([1, 1], [64, 640])))]:
        with pytest.raises(error):
            shared(**change)
    scores = torch.zeros((cache.table.shape[0], 2, cache.width * PAGE), device=DEVICE)
    score = lambda s=scores, **kw: ops.scored_attention(qkv, 4, 2, 32, batch, cache, 0.1, s, **kw)
    score()
    for s, kw in [(scores[:, :, 1:], {}), (scores.double(), {}), (scores, dict(observe=0)), (scores, dict(positions=scores)), (scores, dict(out_scores=scores[:1]))]:
        with pytest.raises(KernelError):
            score(s, **kw)
    k, v, table, scores, positions = evict_case(BF16, 1, 2, 16, 3, 3)
    evict = lambda slots=(0,), lengths=(100,), keep=10, recent=3, **kw: ops.evict_keys(k, v, table, slots, lengths, scores, positions, keep, recent, **kw)
    for kw in [dict(slots=(0, 0), lengths=(100, 100)), dict(slots=(5,)), dict(slots=(-1,)), dict(lengths=(193,)), dict(lengths=(1, 2)), dict(keep=0, recent=0),
               dict(recent=11), dict(recent=-1), dict(out_scores=scores.half()), dict(out_positions=positions[:, :1]), dict(batch=batch)]:
        before = [t.clone() for t in (k, v, scores, positions)]
        with pytest.raises(KernelError):
            evict(**kw)
        for a, b in zip(before, (k, v, scores, positions)):
            assert torch.equal(a, b)
    assert ops.evict_keys(k, v, table, [], [], scores, positions, 10, 3) == []


@pytest.mark.parametrize("dim", [64, 48])
def test_a_single_row_has_no_stride(ops, dim):
    """A step of one row from a view whose stride is odd: the row alone decides which kernel takes it."""
    qkv, batch, cache = make_step(DEVICE, BF16, 4, 2, dim, [130], [1], 1)
    odd = torch.empty((2, qkv.shape[1] + 1), dtype=BF16, device=DEVICE)[:1, :-1]
    odd.copy_(qkv)
    want = ops.shared_prefix_attention(qkv, 4, 2, dim, batch, cache, 0.1, groups([1], [128]))
    assert torch.equal(ops.shared_prefix_attention(odd, 4, 2, dim, batch, cache, 0.1, groups([1], [128])), want)


def test_steps_without_rows(ops):
    """An empty step comes back empty."""
    qkv, batch, cache = make_step(DEVICE, BF16, 4, 2, 32, [70], [1], 1)
    empty = make_batch(DEVICE, batch.slots, batch.starts, [1])
    empty.n_rows, empty.q_lens = 0, [0]
    assert ops.shared_prefix_attention(qkv[:0], 4, 2, 32, empty, cache, 0.1, groups([1], [64])).shape == (0, 128)
