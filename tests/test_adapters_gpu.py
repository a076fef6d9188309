"""Products with the adapters of many requests, and the maps of a step, against the definition in 64 bits and by hand."""

import pytest
import torch

from adapter_helpers import (assert_within, gated64, make_adapters, make_bank, maps_by_hand, per_row, product64, rows_of_step)
from kernel_rush_kawk_b200.csrc import KernelError, load_kernels
from kernel_rush_kawk_b200.csrc.adapter_ops import StepMaps

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    return load_kernels()


def case(seed, dtype, inputs, outs, lengths, of_sequence, rank, count, skip=(), capacity=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((sum(lengths), inputs), generator=g).to(DEV, dtype)
    w = (torch.randn((sum(outs), inputs), generator=g) / inputs ** 0.5).to(DEV, dtype)
    adapters = make_adapters(g, count, inputs, outs, rank, dtype, DEV, skip)
    return x, w, adapters, make_bank(adapters, inputs, outs, rank, dtype, DEV, capacity)


def spread(lengths, count, none=0):
    return [-1 if none and i % none == 0 else (2 * i + 1) % count for i in range(len(lengths))]


STEPS = {
    "one": [1], "two": [1, 1], "eight": [1] * 8, "sixteen": [1] * 16, "seventeen": [1] * 17, "many_single": [1] * 67, "full": [1] * 300,
    "prompt": [45], "prompts": [33, 1, 0, 90, 7], "long": [150, 131, 1, 1, 260], "empty_first": [0, 0, 5, 0], "pieces": [16] * 20, "tiles": [256, 256, 100],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("step", list(STEPS))
@pytest.mark.parametrize("inputs, outs, rank", [(64, (64, 32, 32), 8), (320, (264,), 16), (256, (192, 40, 40, 8), 20), (96, (77,), 5), (333, (50, 3), 3), (1024, (520,), 128)])
def test_linear(ops, dtype, step, inputs, outs, rank):
    lengths = STEPS[step]
    count = 5
    of = spread(lengths, count, none=4)
    x, w, adapters, bank = case(1, dtype, inputs, outs, lengths, of, rank, count, skip={(1, 0), (3, len(outs) - 1)})
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    ops.check()
    ref, bound = product64(x, w, adapters, outs, per_row(lengths, of), dtype == torch.bfloat16)
    assert got.dtype == dtype and got.shape == (sum(lengths), sum(outs))
    assert_within(got, ref, bound, f"{step} {inputs} {outs}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("step", ["one", "eight", "sixteen", "seventeen", "many_single", "prompts", "long", "tiles"])
@pytest.mark.parametrize("inputs, width, rank", [(64, 96, 8), (256, 200, 16), (90, 33, 4), (640, 512, 72)])
def test_gate_up(ops, dtype, step, inputs, width, rank):
    lengths = STEPS[step]
    count = 4
    of = spread(lengths, count, none=5)
    x, w, adapters, bank = case(2, dtype, inputs, (width, width), lengths, of, rank, count, skip={(0, 1), (2, 0)})
    got = ops.adapted_gate_up_swiglu(x, w, width, bank, rows_of_step(ops, lengths, of, DEV))
    ops.check()
    ref, bound = gated64(*product64(x, w, adapters, (width, width), per_row(lengths, of), dtype == torch.bfloat16))
    assert got.shape == (sum(lengths), width)
    assert_within(got, ref, bound, f"{step} {inputs} {width}")


@pytest.mark.parametrize("rows", [1, 12, 64, 200, 900])
def test_every_row_its_own_adapter(ops, rows):
    """And a bank with room to spare."""
    lengths, of = [1] * rows, [(7 * i) % min(rows, 90) for i in range(rows)]
    x, w, adapters, bank = case(3, torch.bfloat16, 256, (256, 64, 64), lengths, of, 16, min(rows, 90), capacity=100)
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    ref, bound = product64(x, w, adapters, (256, 64, 64), of, True)
    ops.check()
    assert_within(got, ref, bound)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths", [[1] * 9, [1] * 40, [40, 30, 300]])
def test_without_any_adapter(ops, dtype, lengths):
    of = [-1] * len(lengths)
    x, w, adapters, bank = case(4, dtype, 128, (96,), lengths, of, 8, 2)
    bank.a.fill_(float("nan"))
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    assert_within(got, *product64(x, w, adapters, (96,), per_row(lengths, of), True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths", [[1] * 5, [1] * 16, [1] * 30, [50, 40, 20, 1, 200], [200, 300]])
def test_numbers_that_are_none_stay_in_their_rows(ops, dtype, lengths):
    """An infinity in a row, a NaN in an adapter: the rows that have neither are as without them."""
    count = 4
    of = [i % 3 for i in range(len(lengths))]
    x, w, adapters, bank = case(5, dtype, 256, (128, 64), lengths, of, 12, count)
    rows = per_row(lengths, of)
    bad_row = sum(lengths) // 2
    x[bad_row, 3] = float("inf")
    bank.a[1].fill_(float("nan"))
    bank.b[3].fill_(float("nan"))
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    good = [r for r, a in enumerate(rows) if a != 1 and r != bad_row]
    x[bad_row, 3] = 0
    ref, bound = product64(x, w, adapters, (128, 64), rows, True)
    assert_within(got[good], ref[good], bound[good])
    assert not torch.isfinite(got[bad_row]).all()
    for r, a in enumerate(rows):
        if a == 1:
            assert torch.isnan(got[r]).all()


@pytest.mark.parametrize("lengths", [[1] * 3, [1] * 16, [1] * 40, [70, 300, 2]])
def test_what_lies_behind_a_rank_is_no_number(ops, lengths):
    """A place that a larger adapter had before a smaller one: nothing of the larger is left; a part that the adapter leaves alone may hold anything."""
    x, w, adapters, bank = case(6, torch.bfloat16, 128, (64, 64), lengths, None, 24, 2, skip={(0, 1)})
    big = make_adapters(torch.Generator().manual_seed(9), 1, 128, (64, 64), 24, torch.bfloat16, DEV)[0]
    for p in range(2):
        bank.put(0, p, big[p][0], big[p][1], 1.0)
    bank.a[0].fill_(float("inf"))
    bank.b[0].fill_(float("nan"))
    bank.clear(0)
    small = (adapters[0][0][0][:3].contiguous(), adapters[0][0][1][:, :3].contiguous(), 1.5)
    bank.put(0, 0, *small)
    adapters[0][0] = small
    of = [i % 2 for i in range(len(lengths))]
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    assert_within(got, *product64(x, w, adapters, (64, 64), per_row(lengths, of), True))


def test_float32_rows_are_the_same_in_any_company(ops):
    lengths = [1, 5, 30, 1, 11, 300]
    of = [0, 1, 2, -1, 1, 0]
    x, w, _, bank = case(7, torch.float32, 200, (96, 40), lengths, of, 10, 3)
    rows = per_row(lengths, of)
    whole = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    again = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    assert torch.equal(whole, again)
    for r in (0, 3, 7, 35, 36, 37, 200):
        alone = ops.adapted_linear(x[r:r + 1], w, bank, rows_of_step(ops, [1], [rows[r]], DEV))
        assert torch.equal(alone[0], whole[r])


@pytest.mark.parametrize("rows", [1, 2, 5, 9, 16])
@pytest.mark.parametrize("outs,K,rank", [((96, 40, 7), 36, 3), ((300, 20), 516, 17), ((16400, 33), 64, 8), ((65, 64, 63, 2), 128, 128), ((12300,), 1028, 40), ((70, 41), 260, 16)])
def test_few_float32_rows(ops, rows, outs, K, rank):
    """Up to sixteen rows in the product's own launch: every way that it splits rows and columns, borders of parts inside it, and the bits of many rows."""
    lengths, of = [1] * rows, spread([1] * rows, 5)
    x, w, adapters, bank = case(14, torch.float32, K, outs, lengths, of, rank, 5, skip={(1, len(outs) - 1)})
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    assert_within(got, *product64(x, w, adapters, outs, of, True))
    more = torch.cat([x, torch.randn((30, K), device=DEV)])
    many = ops.adapted_linear(more, w, bank, rows_of_step(ops, [1] * (rows + 30), of + [2] * 30, DEV))
    assert torch.equal(got, many[:rows])


@pytest.mark.parametrize("rows", [1, 9, 16, 40, 700])
def test_the_same_call_gives_the_same_bits(ops, rows):
    lengths = [1] * rows if rows < 100 else [rows - 200, 150, 50]
    of = spread(lengths, 6)
    x, w, _, bank = case(8, torch.bfloat16, 512, (256, 128), lengths, of, 16, 6)
    step = rows_of_step(ops, lengths, of, DEV)
    first = ops.adapted_linear(x, w, bank, step)
    for _ in range(3):
        assert torch.equal(first, ops.adapted_linear(x, w, bank, step))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [3, 20, 300])
def test_strided_rows_and_weights(ops, dtype, rows):
    """Rows that are a slice of wider ones, at addresses that no vector load takes."""
    lengths, of = [1] * rows, spread([1] * rows, 3)
    x, w, adapters, bank = case(10, dtype, 128, (96,), lengths, of, 8, 3)
    wide_x, wide_w = torch.randn((rows, 141), device=DEV).to(dtype), torch.randn((96, 133), device=DEV).to(dtype)
    wide_x[:, 5:133], wide_w[:, 3:131] = x, w
    step = rows_of_step(ops, lengths, of, DEV)
    ref, bound = product64(x, w, adapters, (96,), of, True)
    assert_within(ops.adapted_linear(wide_x[:, 5:133], w, bank, step), ref, bound)
    assert_within(ops.adapted_linear(wide_x[:, 5:133], wide_w[:, 3:131], bank, step), ref, bound)


@pytest.mark.parametrize("rows", [1, 12, 30, 290])
def test_captured_with_adapters_that_change(ops, rows):
    """Two graphs over one bank, replayed in turn: other requests, another adapter in an old place."""
    lengths = [1] * rows
    x, w, adapters, bank = case(11, torch.bfloat16, 256, (128, 64), lengths, None, 16, 4)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    n, zeros = ints(lengths), ints([0] * rows)
    graphs = []
    for k in range(2):
        of = ints([k] * rows)
        maps = ops.step_maps(zeros, zeros, n, rows, adapters=of)
        ops.adapted_linear(x, w, bank, maps.adapters)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.step_maps(zeros, zeros, n, rows, adapters=of, out=maps)
            y = ops.adapted_linear(x, w, bank, maps.adapters)
        graphs.append((graph, of, y, maps))  # (whose buffers the graph goes on reading)
    for turn in range(3):
        for k, (graph, of, y, _) in enumerate(graphs):
            now = [(i * (turn + 1) + k) % 5 - 1 for i in range(rows)]
            of.copy_(ints(now))
            if turn == 1:
                fresh = make_adapters(torch.Generator().manual_seed(50 + k), 1, 256, (128, 64), 16, torch.bfloat16, DEV)[0]
                for p in range(2):
                    bank.put(2, p, *fresh[p])
                adapters[2] = fresh
            graph.replay()
            ref, bound = product64(x, w, adapters, (128, 64), now, True)
            assert_within(y, ref, bound, f"graph {k} turn {turn}")
    ops.check()


def test_on_another_stream(ops):
    lengths, of = [40, 1, 25], [0, 2, 1]
    x, w, adapters, bank = case(12, torch.bfloat16, 512, (256,), lengths, of, 16, 3)
    ref, bound = product64(x, w, adapters, (256,), per_row(lengths, of), True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            outs.append(ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV)))
    torch.cuda.synchronize()
    for y in outs:
        assert_within(y, ref, bound)


@pytest.mark.parametrize("rows", [4, 30, 300])
def test_adapters_that_the_bank_lacks(ops, rows):
    x, w, adapters, bank = case(13, torch.bfloat16, 128, (64,), [1] * rows, None, 8, 2)
    of = [0, 1, 7, -1] + [0] * (rows - 4)
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, [1] * rows, of, DEV))
    with pytest.raises(KernelError, match="does not hold"):
        ops.check()
    of[2] = -1
    assert_within(got, *product64(x, w, adapters, (64,), of, True))


# -- maps ---------------------------------------------------------------------------------------------------------------

def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def check_lists(rows, per_sequence, lengths):
    """The slots of every tile hold the adapters of its rows, each once, and nothing else; no two tiles have a slot in common, and all slots are said to be."""
    words = rows.buffer.cpu().tolist()
    of = per_row(lengths, per_sequence)
    base = rows.buffer.data_ptr()
    for which in range(len(rows.heights)):
        height, info, slots, n_slots = rows.tiles(which)
        at = (slots - base) // 4
        pairs = list(zip(words[at:at + 2 * n_slots:2], words[at + 1:at + 2 * n_slots:2]))
        used, last = set(), 0
        for tile in range(-(-rows.n_rows // height)):
            first, count = words[(info - base) // 4 + 2 * tile:(info - base) // 4 + 2 * tile + 2]
            assert first >= last
            last = first + count
            assert all(t == tile for _, t in pairs[first:last])
            assert sorted(a for a, _ in pairs[first:last]) == sorted({a for a in of[tile * height:(tile + 1) * height] if a >= 0})
            used.update(range(first, last))
        assert last <= n_slots and (rows.n_rows == 0 or all(a == -1 for i, (a, _) in enumerate(pairs) if i not in used))


@pytest.mark.parametrize("starts, lengths", [
    ([0], [1]), ([63], [1]), ([64], [1]), ([5, 64, 0, 127, 128], [1, 1, 1, 1, 1]), ([0, 10, 0], [0, 0, 0]), ([], []), ([0, 70, 0, 3], [0, 130, 0, 61]),
    ([0] * 3, [700, 768, 65]), (list(range(0, 900, 3)), [1] * 300), ([i % 130 for i in range(1500)], [i % 7 for i in range(1500)]), ([1000, 0], [5000, 4000])])
def test_maps(ops, starts, lengths):
    n = len(starts)
    slots = [(7 * i + 3) % n if n % 7 else n - 1 - i for i in range(n)]
    width = max([-(-(s + t) // 64) for s, t in zip(starts, lengths)], default=1) + 1
    adapters = [(i * 5) % 9 - 1 for i in range(n)]
    pool = list(range(100, 100 + sum(-(-(s + t) // 64) for s, t in zip(starts, lengths)) + 3))[::-1]
    table = [[-7] * width for _ in range(n + 2)]
    for slot, s in zip(slots, starts):
        for logical in range(-(-s // 64)):
            table[slot][logical] = pool.pop()
    device_table = ints(table).view(n + 2, width)
    rows = sum(lengths)
    maps = ops.step_maps(ints(slots), ints(starts), ints(lengths), rows, table=device_table, pages=ints(pool), adapters=ints(adapters))
    cu, seq, pos, place, of = maps_by_hand(slots, starts, lengths, table, pool, adapters)
    ops.check()
    assert maps.cu_q.tolist() == cu and maps.row_seq.tolist() == seq and maps.row_pos.tolist() == pos
    assert maps.row_place.tolist() == place and maps.adapters.row_adapter.tolist() == of
    assert device_table.tolist() == table
    check_lists(maps.adapters, adapters, lengths)
    again = ops.step_maps(ints(slots), ints(starts), ints(lengths), rows, table=device_table, pages=ints(pool), adapters=ints(adapters), out=maps)
    assert again is maps and maps.row_place.tolist() == place and device_table.tolist() == table
    bare = ops.step_maps(ints(slots), ints(starts), ints(lengths), rows)
    assert bare.row_place is None and bare.adapters is None and bare.row_pos.tolist() == pos and bare.cu_q.tolist() == cu


def test_maps_of_many_sequences(ops):
    """More than shared memory takes without asking, in and out of step with the threads."""
    for n in (4097, 24999):
        lengths = [i % 3 for i in range(n)]
        maps = ops.step_maps(ints(list(range(n))), ints([i % 64 for i in range(n)]), ints(lengths), sum(lengths))
        cu, seq, pos, _, _ = maps_by_hand(list(range(n)), [i % 64 for i in range(n)], lengths, None, None, None)
        assert maps.cu_q.tolist() == cu and maps.row_seq.tolist() == seq and maps.row_pos.tolist() == pos


@pytest.mark.parametrize("change", ["short", "long", "negative", "slot", "width", "pages", "start"])
def test_maps_that_do_not_fit(ops, change):
    """Nothing out of range is written; the error word says so."""
    starts, lengths, slots, rows, pages = [10, 64, 0], [3, 70, 1], [2, 0, 1], 74, [9, 8, 7]
    if change == "short":
        rows = 80
    elif change == "long":
        rows = 60
    elif change == "negative":
        lengths[0] = -4
    elif change == "slot":
        slots[1] = 5
    elif change == "width":
        starts[1] = 64 * 3 - 2
    elif change == "pages":
        pages = [9]
    elif change == "start":
        starts[1] = -70
    table = torch.full((5, 3), 77, dtype=torch.int32, device=DEV)
    guard = table.clone()
    maps = ops.step_maps(ints(slots), ints(starts), ints(lengths), rows, table=table[1:4], pages=ints(pages), adapters=ints([0, 1, 2]))
    with pytest.raises(KernelError, match="do not fit a step"):
        ops.check()
    assert torch.equal(table[0], guard[0]) and torch.equal(table[4], guard[4])
    if change == "short":
        assert maps.row_pos[74:].eq(-1).all() and maps.adapters.row_adapter[74:].eq(-1).all() and maps.row_place[74:].eq(-1).all()
    ops.check()


def test_maps_in_a_captured_step(ops):
    """Lengths that change between replays."""
    maps = StepMaps(6, 4, DEV)
    slots, starts, lengths, of = ints([3, 1, 0, 2]), ints([0, 0, 0, 0]), ints([6, 0, 0, 0]), ints([0, 1, 2, 3])
    table, pages = torch.zeros((4, 4), dtype=torch.int32, device=DEV), ints([5, 6, 7, 8])
    ops.step_maps(slots, starts, lengths, 6, table=table, pages=pages, adapters=of, out=maps)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.step_maps(slots, starts, lengths, 6, table=table, pages=pages, adapters=of, out=maps)
    for s, n in (([0, 63, 1, 2], [2, 2, 1, 1]), ([64, 0, 0, 0], [0, 0, 0, 6]), ([0, 0, 0, 62], [0, 0, 0, 6])):
        starts.copy_(ints(s))
        lengths.copy_(ints(n))
        host = table.tolist()
        graph.replay()
        cu, seq, pos, place, at = maps_by_hand([3, 1, 0, 2], s, n, host, [5, 6, 7, 8], [0, 1, 2, 3])
        assert maps.cu_q.tolist() == cu and maps.row_seq.tolist() == seq and maps.row_pos.tolist() == pos and maps.row_place.tolist() == place
        assert maps.adapters.row_adapter.tolist() == at and table.tolist() == host
        check_lists(maps.adapters, [0, 1, 2, 3], n)
    ops.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths", [[1], [1] * 16, [1] * 33, [100, 1, 180]])
@pytest.mark.parametrize("outs,rank", [((64, 40, 24, 8), 130), ((128, 64), 256), ((264,), 200), ((16, 16, 16, 16), 72)])
def test_large_ranks_and_many_parts(ops, dtype, lengths, outs, rank):
    of = spread(lengths, 3)
    x, w, adapters, bank = case(15, dtype, 192, outs, lengths, of, rank, 3, skip={(0, len(outs) - 1)})
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    assert_within(got, *product64(x, w, adapters, outs, per_row(lengths, of), True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("length", [1, 3])
def test_a_thousand_sequences(ops, dtype, length):
    lengths, of = [length] * 1000, spread([1] * 1000, 150, 7)
    x, w, adapters, bank = case(16, dtype, 96, (72, 24), lengths, of, 8, 150)
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    assert_within(got, *product64(x, w, adapters, (72, 24), per_row(lengths, of), True))


def test_two_streams_at_once(ops):
    """Products of every kind on two streams, side by side: the bits of one after the other."""
    calls = []
    for seed, dtype, lengths, K, outs in [(17, torch.bfloat16, [700, 300], 2048, (1024, 512)), (18, torch.bfloat16, [1] * 64, 2048, (2048,)),
                                          (19, torch.bfloat16, [1] * 8, 2048, (2048,)), (20, torch.float32, [1] * 6, 1024, (1024,)),
                                          (21, torch.bfloat16, [513], 1024, (256,)), (22, torch.bfloat16, [1] * 200, 1024, (4096,))]:
        of = spread(lengths, 4)
        x, w, _, bank = case(seed, dtype, K, outs, lengths, of, 16, 4)
        rows = rows_of_step(ops, lengths, of, DEV)
        calls.append(lambda x=x, w=w, bank=bank, rows=rows: ops.adapted_linear(x, w, bank, rows))
    expected = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for turn in range(12):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for j in range(len(calls)):
                    which = (j + 3 * i + turn) % len(calls)
                    got[i].append((which, calls[which]()))
    torch.cuda.synchronize()
    for results in got:
        for which, y in results:
            assert torch.equal(y, expected[which])
    ops.check()


@pytest.mark.parametrize("lengths", [[1] * 200, [9] * 28, [100] + [1] * 60, [1] * 129])
@pytest.mark.parametrize("K,outs,rank", [(72, (64, 40), 24), (5000, (96,), 8), (640, (128, 128), 64)])
def test_large_tiles_with_many_adapters(ops, lengths, K, outs, rank):
    """One tile of 129 to 256 rows whose slots are many: adapters of one row and of a hundred, unequal parts of k."""
    of = spread(lengths, 29, 5)
    x, w, adapters, bank = case(23, torch.bfloat16, K, outs, lengths, of, rank, 29, skip={(2, 0)})
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    assert_within(got, *product64(x, w, adapters, outs, per_row(lengths, of), True))


@pytest.mark.parametrize("rows", [1, 7, 16])
@pytest.mark.parametrize("K,outs,rank", [(64, (48,), 8), (9728, (40, 24), 40), (2592, (64, 64, 64), 16)])
def test_few_rows_and_every_length_of_k(ops, rows, K, outs, rank):
    lengths, of = [1] * rows, spread([1] * rows, 4, 6)
    x, w, adapters, bank = case(24, torch.bfloat16, K, outs, lengths, of, rank, 4, skip={(1, 0)})
    step = rows_of_step(ops, lengths, of, DEV)
    assert_within(ops.adapted_linear(x, w, bank, step), *product64(x, w, adapters, outs, of, True))


def test_two_graphs_side_by_side(ops):
    """Captured products of many and of few rows over one bank, replayed on two streams at once: neither's scratch is the other's."""
    graphs = []
    for seed, lengths in ((25, [400, 330]), (26, [1] * 70), (27, [1] * 12), (28, [1] * 230)):
        of = spread(lengths, 4)
        x, w, _, bank = case(29, torch.bfloat16, 1024, (1024, 256), lengths, of, 16, 4)
        rows = rows_of_step(ops, lengths, of, DEV)
        expected = ops.adapted_linear(x, w, bank, rows)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.adapted_linear(x, w, bank, rows)
        graphs.append((graph, y, expected, x, w, bank, rows))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for stream, (graph, y, *_) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                y.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, y, expected, *_ in graphs:
        assert torch.equal(y, expected)
    ops.check()


@pytest.mark.parametrize("rows", [1, 5, 16])
@pytest.mark.parametrize("half,K,rank", [(100, 68, 5), (8200, 96, 16), (33, 1000, 64)])
def test_few_float32_rows_with_gate_and_up(ops, rows, half, K, rank):
    """And the bits that many rows give."""
    lengths, of = [1] * rows, spread([1] * rows, 5, 4)
    x, w, adapters, bank = case(30, torch.float32, K, (half, half), lengths, of, rank, 5, skip={(1, 1)})
    got = ops.adapted_gate_up_swiglu(x, w, half, bank, rows_of_step(ops, lengths, of, DEV))
    assert_within(got, *gated64(*product64(x, w, adapters, (half, half), of, True)))
    more = torch.cat([x, torch.randn((20, K), device=DEV)])
    many = ops.adapted_gate_up_swiglu(more, w, half, bank, rows_of_step(ops, [1] * (rows + 20), of + [2] * 20, DEV))
    assert torch.equal(got, many[:rows])
