"""The maps of a step where a table or maps to fill again hold something else than they should."""

import pytest
import torch

from kernel_rush_kawk_b200.csrc import KernelError, load_kernels
from kernel_rush_kawk_b200.csrc.adapter_ops import StepMaps

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    return load_kernels()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("lengths", [[1, 1], [70, 1], [3, 900]])
def test_a_held_page_that_the_table_lacks(ops, lengths):
    """The rows on it have no place, and the error word says so."""
    table = ints([[4, -1, -1], [-1, -1, -1], [9, 8, -1]])
    starts = [70, 5]
    n_pages = sum(-(-(s + n) // 64) - -(-s // 64) for s, n in zip(starts, lengths))
    table = torch.cat([table, torch.full((3, 17), -1, dtype=torch.int32, device=DEV)], 1)
    maps = ops.step_maps(ints([0, 2]), ints(starts), ints(lengths), sum(lengths), table=table, pages=ints(list(range(20, 20 + n_pages))))
    with pytest.raises(KernelError, match="do not fit a step"):
        ops.check()
    on_it = [p < 128 for p in range(70, 70 + lengths[0])]
    place = maps.row_place.tolist()
    assert all((place[r] == -1) == lost for r, lost in enumerate(on_it)) and all(v >= 0 for v in place[lengths[0]:])
    ops.check()


@pytest.mark.parametrize("n", [1, 900])
def test_places_without_a_table(ops, n):
    """Maps that are filled again without a table keep no places of the step before."""
    maps = StepMaps(n + 2, 2, DEV, with_adapters=False)
    maps.buffer.fill_(77)
    args = ints([0, 1]), ints([64, 3]), ints([n, 2]), n + 2
    table = torch.arange(40, dtype=torch.int32, device=DEV).view(2, 20).contiguous()
    ops.step_maps(*args, table=table, pages=ints(list(range(50, 70))), out=maps)
    assert maps.row_place.ge(0).all()
    ops.step_maps(*args, out=maps)
    assert maps.row_place.eq(-1).all() and maps.row_pos.tolist() == list(range(64, 64 + n)) + [3, 4]
    ops.check()
