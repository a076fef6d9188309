"""Rows whose adapters the bank lacks, wherever they stand: the error word is set, and every other row is as it would be without them."""

import pytest
import torch

from adapter_helpers import assert_within, gated64, make_adapters, make_bank, product64, rows_of_step
from kernel_rush_kawk_b200.csrc import KernelError, load_kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    return load_kernels()


@pytest.fixture
def full_scratch():
    """Memory that calls draw their scratch from is full of NaN."""
    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 22, 1 << 24, 1 << 26):
        kept = [torch.full((n,), float("nan"), device=DEV) for _ in range(3)]
        del kept


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("count", [1, 2, 30])
@pytest.mark.parametrize("rows", [4, 16, 30, 120, 200, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_before_the_others(ops, full_scratch, dtype, count, rows, gated):
    g = torch.Generator().manual_seed(rows + count)
    K, outs = 128, (64, 64)
    x = torch.randn((rows, K), generator=g).to(DEV, dtype)
    w = (torch.randn((128, K), generator=g) / K ** 0.5).to(DEV, dtype)
    adapters = make_adapters(g, count, K, outs, 8, dtype, DEV)
    bank = make_bank(adapters, K, outs, 8, dtype, DEV)
    bad = [count + 5, count, 1000] if rows < 30 else [count + i for i in range(25)]
    of = (bad + [i % (count + 1) - 1 for i in range(count, count + rows)])[:rows]
    assert sum(a >= count for a in of) >= 3 and any(0 <= a < count for a in of)
    call = (lambda of: ops.adapted_gate_up_swiglu(x, w, 64, bank, rows_of_step(ops, [1] * rows, of, DEV))) if gated else (
        lambda of: ops.adapted_linear(x, w, bank, rows_of_step(ops, [1] * rows, of, DEV)))
    got = call(of)
    with pytest.raises(KernelError, match="does not hold"):
        ops.check()
    of = [-1 if a >= count else a for a in of]
    y, bound = product64(x, w, adapters, outs, of, dtype == torch.bfloat16)
    assert_within(got, *(gated64(y, bound) if gated else (y, bound)))
    ops.check()
