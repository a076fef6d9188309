"""Products with adapters of several row tiles whose blocks of k are dealt out in shares, against the definition in 64 bits."""

import pytest
import torch

from adapter_helpers import assert_within, gated64, make_adapters, make_bank, per_row, product64, rows_of_step
from kernel_rush_kawk_b200.csrc import load_kernels
from test_adapted_shares import dealt, in_empty_parts

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    return load_kernels()


def inputs(seed, M, K, outs, rank):
    """Sequences that end inside tiles, three adapters and none, ranks of their own."""
    g = torch.Generator().manual_seed(seed)
    lengths = [M // 3, 1, 7, M // 5]
    lengths.append(M - sum(lengths))
    of = [2, 0, -1, 1, 0]
    x = torch.randn((M, K), generator=g).to(DEV, torch.bfloat16)
    w = (torch.randn((sum(outs), K), generator=g) / K ** 0.5).to(DEV, torch.bfloat16)
    adapters = make_adapters(g, 3, K, outs, rank, torch.bfloat16, DEV)
    return x, w, adapters, make_bank(adapters, K, outs, rank, torch.bfloat16, DEV), lengths, of


def in_shares(M, K, N):
    """(tiles taken whole, tiles in shares, whether these are in equal parts) of a product of several row tiles."""
    row_tiles, column_tiles, shared, k_blocks, _ = dealt(M, K, N, 3)
    rest = row_tiles * column_tiles - shared
    return row_tiles > 1, shared, rest, rest > 0 and rest * (74 // rest) * 10 >= 74 * 9


EMPTY = [(257, 13888, 256), (384, 14336, 256), (300, 17408, 256), (500, 17408, 256), (513, 9920, 256)]
EQUAL = [(257, 8192, 272), (1100, 8192, 272), (513, 9728, 256), (1100, 8192, 1536), (2103, 9728, 2560)]
RUNS = [(400, 8192, 784), (900, 9728, 272), (769, 8192, 5120)]


def product(ops, M, K, N, rank):
    outs = (N,) if M % 2 else (N // 2 + 24, N // 2 - 24)
    x, w, adapters, bank, lengths, of = inputs(M + K, M, K, outs, rank)
    got = ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV))
    ops.check()
    assert_within(got, *product64(x, w, adapters, outs, per_row(lengths, of), True), f"{M} rows of {K} x {N}")


def gate_up(ops, M, K, N, rank):
    outs = (N // 2, N // 2)
    x, w, adapters, bank, lengths, of = inputs(M + K + 1, M, K, outs, rank)
    got = ops.adapted_gate_up_swiglu(x, w, N // 2, bank, rows_of_step(ops, lengths, of, DEV))
    ops.check()
    assert_within(got, *gated64(*product64(x, w, adapters, outs, per_row(lengths, of), True)), f"{M} rows of {K} x {N}, gated")


@pytest.mark.parametrize("run", [product, gate_up])
@pytest.mark.parametrize("M,K,N", EMPTY)
def test_parts_without_k(ops, run, M, K, N):
    """Parts of k behind the last block add nothing, adapters least of all."""
    assert in_empty_parts(dealt(M, K, N, 3))
    run(ops, M, K, N, 16)


@pytest.mark.parametrize("run", [product, gate_up])
@pytest.mark.parametrize("M,K,N", EQUAL)
def test_equal_parts(ops, run, M, K, N):
    several, _, rest, equal = in_shares(M, K, N)
    assert several and rest and equal and not in_empty_parts(dealt(M, K, N, 3))
    run(ops, M, K, N, 80)


@pytest.mark.parametrize("run", [product, gate_up])
@pytest.mark.parametrize("M,K,N", RUNS)
def test_runs(ops, run, M, K, N):
    several, _, rest, equal = in_shares(M, K, N)
    assert several and rest and not equal
    run(ops, M, K, N, 24)
