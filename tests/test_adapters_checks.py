"""What adapters and the maps of a step ask of their arguments before anything is launched (no GPU)."""

import pytest
import torch

from adapter_helpers import gated64, make_adapters, make_bank, maps_by_hand, product64
from kernel_rush_kawk_b200.csrc import adapter_ops, cache_ops
from kernel_rush_kawk_b200.csrc.adapter_ops import AdapterOps, StepMaps
from kernel_rush_kawk_b200.csrc.cache_ops import CacheOps, KernelError
from kernel_rush_kawk_b200.parts.adapters import AdapterBank, AdapterError


class Checks(CacheOps, AdapterOps):
    error = torch.zeros(1, dtype=torch.int32)

    def _resolve(self, x):
        return x


@pytest.fixture(autouse=True)
def a_device(monkeypatch):
    for module in (cache_ops, adapter_ops):
        monkeypatch.setattr(module, "_current_device", lambda: -1)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


def elsewhere(t):
    """A tensor like this one on another device."""
    return type("Elsewhere", (), dict(get_device=lambda self: 1, device="cuda:1", __getattr__=lambda self, name: getattr(t, name)))()


@pytest.mark.parametrize("make", [
    lambda: AdapterBank(8, (), 1, 4, torch.float32, "cpu"), lambda: AdapterBank(8, (4,) * 5, 1, 4, torch.float32, "cpu"),
    lambda: AdapterBank(8, (4, 0), 1, 4, torch.float32, "cpu"), lambda: AdapterBank(0, 4, 1, 4, torch.float32, "cpu"),
    lambda: AdapterBank(8, 4, 0, 4, torch.float32, "cpu"), lambda: AdapterBank(8, 4, 1, 0, torch.float32, "cpu"),
    lambda: AdapterBank(8, 4, 1, 257, torch.float32, "cpu"), lambda: AdapterBank(8, 4, 1, 4, torch.float16, "cpu")])
def test_banks_that_make_no_sense(make):
    with pytest.raises(AdapterError):
        make()


def test_what_a_bank_takes():
    bank = AdapterBank(8, (4, 6), 2, 5, torch.float32, "cpu")
    assert bank.rank == 8 and bank.begin == [0, 4, 10] and bank.parts == 2
    a, b = torch.randn(5, 8), torch.randn(6, 5)
    bank.b.fill_(9)
    bank.put(1, 1, a, b, 0.5)
    assert torch.equal(bank.a[1, 8:13], a) and torch.equal(bank.b[1, 4:, :5], b) and not bank.b[1, 4:, 5:].any()
    assert bank.ranks.tolist() == [[0, 0], [0, 5]] and bank.scale[1, 1] == 0.5
    bank.clear(1)
    assert not bank.ranks.any()
    for args in ((2, 0, a, b), (-1, 0, a, b), (0, 2, a, b), (0, 0, a, b), (0, 1, a[:, :7], b), (0, 1, a[:4], b), (0, 1, a[:0], b[:, :0]),
                 (0, 1, torch.randn(9, 8), torch.randn(6, 9)), (0, 1, a[0], b)):
        with pytest.raises(AdapterError):
            bank.put(*args)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bank_holds_numbers(dtype):
    """Rows of other adapters are multiplied by an adapter's factors too, as zeros: an infinity would make them none."""
    bank = AdapterBank(8, (4, 6), 2, 5, dtype, "cpu")
    a, b = torch.randn(5, 8), torch.randn(6, 5)
    bank.put(0, 1, a, b, 0.5)
    held = [t.clone() for t in (bank.a, bank.b, bank.scale, bank.ranks)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        for which in range(3):
            args = [a.clone(), b.clone(), 1.0]
            if which == 2:
                args[2] = bad
            else:
                args[which][2, 3] = bad
            with pytest.raises(AdapterError, match="finite"):
                bank.put(0, 1, *args)
    if dtype is torch.bfloat16:  # finite in 32 bits, and not in 16
        with pytest.raises(AdapterError, match="finite"):
            bank.put(0, 1, a, torch.full((6, 5), torch.finfo(torch.float32).max))
    assert all(torch.equal(t, was) for t, was in zip((bank.a, bank.b, bank.scale, bank.ranks), held))


def test_a_bank_keeps_its_tensors():
    bank = AdapterBank(8, 4, 1, 4, torch.float32, "cpu")
    for name in ("a", "b", "scale", "ranks"):
        with pytest.raises(AttributeError):
            setattr(bank, name, getattr(bank, name).clone())
    a = torch.randn(4, 8, requires_grad=True)
    bank.put(0, 0, a, torch.randn(4, 4))
    assert torch.equal(bank.a[0, :4], a) and not bank.a.requires_grad


def product(x=None, w=None, bank=None, rows=None, gated=0):
    x = torch.randn(3, 16) if x is None else x
    w = torch.randn(12, 16) if w is None else w
    bank = AdapterBank(16, (8, 4), 2, 4, torch.float32, "cpu") if bank is None else bank
    rows = StepMaps(3, 3, "cpu").adapters if rows is None else rows
    if gated:
        return Checks().adapted_gate_up_swiglu(x, w, gated, bank, rows)
    return Checks()._check_adapted("adapted product", x, w, bank, rows)


def test_a_product_that_fits_is_taken():
    product()


@pytest.mark.parametrize("change", [
    dict(x=torch.randn(3, 15)), dict(w=torch.randn(12, 15)), dict(w=torch.randn(11, 16)), dict(x=torch.randn(3, 16).bfloat16()),
    dict(x=torch.randn(3, 16).bfloat16(), w=torch.randn(12, 16).bfloat16()), dict(x=torch.randn(4, 16)), dict(rows=StepMaps(2, 2, "cpu").adapters),
    dict(x=torch.randn(16, 3).t()), dict(w=torch.randn(16, 12).t()), dict(x=torch.randn(1, 16).expand(3, 16)), dict(x=elsewhere(torch.randn(3, 16))),
    dict(w=elsewhere(torch.randn(12, 16))), dict(bank=AdapterBank(16, (8, 5), 2, 4, torch.float32, "cpu")),
    dict(bank=AdapterBank(15, (8, 4), 2, 4, torch.float32, "cpu")), dict(gated=8), dict(gated=6)])
def test_products_that_do_not_fit(change):
    with pytest.raises(KernelError):
        product(**change)


@pytest.mark.parametrize("change", [
    dict(lengths=ints(1, 2).long()), dict(starts=ints(0)), dict(slots=ints(0, 1, 2)), dict(adapters=ints(0)), dict(n_rows=-1), dict(slots=ints(0, 9, 1, 9)[::2]),
    dict(table=torch.zeros(2, 3)), dict(table=ints(1, 2, 3)), dict(table=torch.zeros((3, 2), dtype=torch.int32).t()), dict(pages=ints(1, 2)),
    dict(table=torch.zeros((2, 3), dtype=torch.int32), pages=ints(1, 2).long()), dict(table=torch.zeros((2, 3), dtype=torch.int32), pages=ints(1, 2)[None]),
    dict(lengths=elsewhere(ints(1, 2))), dict(starts=elsewhere(ints(0, 0))), dict(table=elsewhere(torch.zeros((2, 3), dtype=torch.int32))),
    dict(out=StepMaps(4, 2, "cpu")), dict(out=StepMaps(3, 3, "cpu")), dict(out=StepMaps(3, 2, "cpu")),
    dict(adapters=ints(0, 1), out=StepMaps(3, 2, "cpu", with_adapters=False)),
    dict(table=torch.zeros((2, 3), dtype=torch.int32), out=StepMaps(3, 2, "cpu", with_places=False, with_adapters=False))])
def test_maps_that_do_not_fit(change):
    args = dict(slots=ints(0, 1), starts=ints(0, 0), lengths=ints(1, 2), n_rows=3)
    args.update(change)
    with pytest.raises(KernelError):
        Checks().step_maps(**args)


def test_too_many_sequences():
    many = torch.zeros(AdapterOps.MOST_SEQUENCES + 1, dtype=torch.int32)
    with pytest.raises(KernelError):
        Checks().step_maps(many, many, many, 0)
    with pytest.raises(KernelError):
        Checks().step_maps(many[:1], many[:1], many[:1], AdapterOps.MOST_ROWS + 1)


def test_lists_have_room_for_every_tile():
    for places in (False, True):
        for n_rows, n_seqs in ((0, 3), (1, 1), (255, 8), (256, 256), (257, 3), (5000, 40), (777, 0)):
            maps = StepMaps(n_rows, n_seqs, "cpu", with_places=places)
            rows = maps.adapters
            end = maps.address + 4 * maps.buffer.numel()
            assert rows.row_adapter_at % 8 == 0 and rows.row_adapter_at >= maps.address + 4 * (2 * n_rows * places + n_seqs + 1 + 2 * n_rows)
            at = rows.row_adapter_at + 4 * (n_rows + n_rows % 2)
            for i, h in enumerate(rows.heights):
                height, info, slots, n_slots = rows.tiles(i)
                tiles = -(-n_rows // h)
                assert height == h and info == at and slots == at + 8 * tiles and n_slots == tiles + n_seqs and info % 8 == 0
                at = slots + 8 * n_slots
            assert at == end == rows.row_adapter_at + 4 * rows.words()
            assert n_rows > 256 or rows.heights[0] >= n_rows
            assert (maps.row_place is None) != places and maps.row_pos.shape == (n_rows,) and maps.cu_q.shape == (n_seqs + 1,)


def test_the_definition_itself():
    """In 64 bits: the merged weights give the same; a gradient step along a factor changes the product by its derivative."""
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn((5, 12), generator=g).double(), torch.randn((7, 12), generator=g).double()
    adapters = make_adapters(g, 2, 12, (4, 3), 3, torch.float64, "cpu", skip={(1, 0)})
    of = [0, 1, -1, 1, 0]
    y, _ = product64(x, w, adapters, (4, 3), of, False)
    for r, a in enumerate(of):
        merged = w.clone()
        for p, (lo, hi) in enumerate(((0, 4), (4, 7))):
            if a >= 0 and adapters[a][p] is not None:
                A, B, s = adapters[a][p]
                merged[lo:hi] += s * B @ A
        assert torch.allclose(y[r], merged @ x[r], rtol=1e-12, atol=1e-12)
    z, _ = gated64(torch.cat([y[:, :3], y[:, 4:]], 1), torch.zeros(5, 6).double())
    assert torch.allclose(z, torch.nn.functional.silu(y[:, :3]) * y[:, 4:])


def test_maps_by_hand_of_a_small_step():
    table = [[4, 0], [0, 0], [8, 0]]
    cu, seq, pos, place, of = maps_by_hand([2, 0, 1], [63, 5, 0], [2, 0, 1], table, [9, 3], [1, 0, -1])
    assert cu == [0, 2, 2, 3] and seq == [0, 0, 2] and pos == [63, 64, 0] and place == [8 * 64 + 63, 9 * 64, 3 * 64] and of == [1, 1, -1]
    assert table == [[4, 0], [3, 0], [8, 9]]


def test_banks_of_adapters():
    g = torch.Generator().manual_seed(1)
    adapters = make_adapters(g, 3, 16, (8, 4), 6, torch.float32, "cpu", skip={(2, 1)})
    bank = make_bank(adapters, 16, (8, 4), 6, torch.float32, "cpu")
    assert bank.ranks[2, 1] == 0 and (bank.ranks[:2] > 0).all()
