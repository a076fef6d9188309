"""Float32 products with adapters, held to the bound of sums and factors that stay in 32 bits all the way: no first factor is rounded to fewer."""

import pytest
import torch

from adapter_helpers import assert_within, gated64, per_row, product64, rows_of_step
from kernel_rush_kawk_b200.csrc import load_kernels
from test_adapters_gpu import case, spread

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32 = torch.float32


@pytest.fixture(scope="module")
def ops():
    return load_kernels()


def test_the_bound_tells_16_bits_from_32():
    """On the formula alone: a first factor rounded to bfloat16 is far outside."""
    x, w, adapters, _ = case(40, F32, 192, (64, 40), [1] * 6, None, 16, 2)
    of = [0, 1, 0, 1, 0, 1]
    ref, bound = product64(x, w, adapters, (64, 40), of, False)
    y = x.double() @ w.double().T
    for r, a in enumerate(of):
        at = 0
        for n, (A, B, s) in zip((64, 40), adapters[a]):
            y[r, at:at + n] += (s * (x[r].double() @ A.double().T)).bfloat16().double() @ B.double().T
            at += n
    with pytest.raises(AssertionError, match="off by"):
        assert_within(y.float(), ref, bound)


@pytest.mark.parametrize("rows", [1, 2, 5, 9, 16])
@pytest.mark.parametrize("outs,K,rank", [((96, 40, 7), 36, 3), ((300, 20), 516, 17), ((16400, 33), 64, 8), ((65, 64, 63, 2), 128, 128), ((12300,), 1028, 40), ((70, 41), 260, 16)])
def test_few_rows(ops, rows, outs, K, rank):
    of = spread([1] * rows, 5)
    x, w, adapters, bank = case(41, F32, K, outs, [1] * rows, of, rank, 5, skip={(1, len(outs) - 1)})
    assert_within(ops.adapted_linear(x, w, bank, rows_of_step(ops, [1] * rows, of, DEV)), *product64(x, w, adapters, outs, of, False))


@pytest.mark.parametrize("rows", [1, 5, 16, 40])
@pytest.mark.parametrize("half,K,rank", [(100, 68, 5), (8200, 96, 16), (33, 1000, 64), (48, 77, 200)])
def test_gate_and_up(ops, rows, half, K, rank):
    of = spread([1] * rows, 5, 4)
    x, w, adapters, bank = case(42, F32, K, (half, half), [1] * rows, of, rank, 5, skip={(1, 1)})
    got = ops.adapted_gate_up_swiglu(x, w, half, bank, rows_of_step(ops, [1] * rows, of, DEV))
    assert_within(got, *gated64(*product64(x, w, adapters, (half, half), of, False)))


@pytest.mark.parametrize("lengths", [[1], [1] * 16, [1] * 33, [100, 1, 180]])
@pytest.mark.parametrize("outs,rank", [((64, 40, 24, 8), 130), ((128, 64), 256), ((264,), 200), ((16, 16, 16, 16), 72)])
def test_large_ranks_and_many_parts(ops, lengths, outs, rank):
    of = spread(lengths, 3)
    x, w, adapters, bank = case(43, F32, 192, outs, lengths, of, rank, 3, skip={(0, len(outs) - 1)})
    assert_within(ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV)), *product64(x, w, adapters, outs, per_row(lengths, of), False))


@pytest.mark.parametrize("length", [1, 3])
def test_a_thousand_sequences(ops, length):
    lengths, of = [length] * 1000, spread([1] * 1000, 150, 7)
    x, w, adapters, bank = case(44, F32, 96, (72, 24), lengths, of, 8, 150)
    assert_within(ops.adapted_linear(x, w, bank, rows_of_step(ops, lengths, of, DEV)), *product64(x, w, adapters, (72, 24), per_row(lengths, of), False))


@pytest.mark.parametrize("rows", [3, 20, 300])
def test_strided_rows_and_weights(ops, rows):
    of = spread([1] * rows, 3)
    x, w, adapters, bank = case(45, F32, 128, (96,), [1] * rows, of, 8, 3)
    wide_x, wide_w = torch.randn((rows, 141), device=DEV), torch.randn((96, 133), device=DEV)
    wide_x[:, 5:133], wide_w[:, 3:131] = x, w
    step = rows_of_step(ops, [1] * rows, of, DEV)
    ref, bound = product64(x, w, adapters, (96,), of, False)
    assert_within(ops.adapted_linear(wide_x[:, 5:133], w, bank, step), ref, bound)
    assert_within(ops.adapted_linear(wide_x[:, 5:133], wide_w[:, 3:131], bank, step), ref, bound)
