"""Products with adapters of millions of rows."""

import pytest
import torch

from adapter_helpers import assert_within, make_adapters, make_bank, product64
from kernel_rush_kawk_b200.csrc import load_kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_ten_million_rows():
    """As many sequences as the maps take, more tiles times sequences than 31 bits hold; rows from everywhere against the definition."""
    ops = load_kernels()
    n, each, K, N = 25000, 410, 64, 8
    M = n * each
    g = torch.Generator().manual_seed(5)
    x = torch.randn((M, K), generator=torch.Generator(DEV).manual_seed(5), device=DEV, dtype=torch.bfloat16)
    w = (torch.randn((N, K), generator=g) / K ** 0.5).to(DEV, torch.bfloat16)
    adapters = make_adapters(g, 3, K, (N,), 8, torch.bfloat16, DEV)
    bank = make_bank(adapters, K, (N,), 8, torch.bfloat16, DEV)
    of = torch.arange(n, dtype=torch.int32) % 4 - 1
    lengths = torch.full((n,), each, dtype=torch.int32, device=DEV)
    rows = ops.step_maps(torch.arange(n, dtype=torch.int32, device=DEV), torch.zeros_like(lengths), lengths, M, adapters=of.to(DEV)).adapters
    which, _ = ops._tiling(rows.heights, M, K, N)
    height, _, _, n_slots = rows.tiles(which)
    assert -(-M // height) * n_slots > 1 << 31
    got = ops.adapted_linear(x, w, bank, rows)
    ops.check()
    some = torch.cat([torch.arange(600), torch.arange(M - 600, M), torch.randint(0, M, (4000,), generator=g)])
    ref, bound = product64(x[some.to(DEV)], w, adapters, (N,), of[some // each].tolist(), True)
    assert_within(got[some.to(DEV)], ref, bound)
