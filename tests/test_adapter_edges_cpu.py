"""Adapters at the edges of what banks, engines, files and the command line take (no GPU)."""

import pytest
import torch

from kernel_rush_kawk_b200.parts.adapters import AdapterBank, AdapterError


@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38, float("inf"), float("nan")])
def test_a_scale_that_32_bits_do_not_hold(scale):
    """Finite in 64 bits, an infinity where the bank holds it."""
    bank = AdapterBank(8, (4, 6), 2, 5, torch.float32, "cpu")
    with pytest.raises(AdapterError, match="finite"):
        bank.put(1, 1, torch.randn(5, 8), torch.randn(6, 5), scale)
    assert not bank.scale.any() and not bank.ranks.any()
    bank.put(1, 1, torch.randn(5, 8), torch.randn(6, 5), torch.finfo(torch.float32).max)
    assert torch.isfinite(bank.scale).all()
