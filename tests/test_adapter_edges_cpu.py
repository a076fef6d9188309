"""Adapters at the edges of what banks, engines, files and the command line take (no GPU)."""

import pytest
import torch

from adapter_helpers import random_factors
from helpers import prompts_for
from kernel_rush_kawk_b200.parts.adapters import AdapterBank, AdapterError
from test_adapted_engine_cpu import NAME, make, plain_of


@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38, float("inf"), float("nan")])
def test_a_scale_that_32_bits_do_not_hold(scale):
    """Finite in 64 bits: refused before anything is written, like an infinity."""
    bank = AdapterBank(8, (4, 6), 2, 5, torch.float32, "cpu")
    with pytest.raises(AdapterError, match="finite"):
        bank.put(1, 1, torch.randn(5, 8), torch.randn(6, 5), scale)
    assert not any(t.any() for t in (bank.a, bank.b, bank.scale, bank.ranks))
    bank.put(1, 1, torch.randn(5, 8), torch.randn(6, 5), torch.finfo(torch.float32).max)
    assert torch.isfinite(bank.scale).all()


def test_an_adapter_that_is_not_all_there_has_no_name(folders, monkeypatch):
    """Copies that fail half way through: the name stands for nothing, and may be loaded again."""
    engine = make(folders)
    cfg, w = plain_of(folders)
    old, new = random_factors(cfg, w, 1, 4), random_factors(cfg, w, 2, 4)
    engine.load_adapter("a", old)
    engine.load_adapter("b", old)
    prompt = prompts_for(NAME, [9])
    before = engine.generate_all(prompt, 4, adapters="b")
    put, calls = AdapterBank.put, []

    def failing(self, *args):
        calls.append(args)
        if len(calls) == 4:
            raise torch.OutOfMemoryError("no room for the copy")
        put(self, *args)

    monkeypatch.setattr(AdapterBank, "put", failing)
    with pytest.raises(torch.OutOfMemoryError):
        engine.load_adapter("a", new)
    monkeypatch.undo()
    assert sorted(engine.adapters) == ["b"]
    with pytest.raises(AdapterError, match="no adapter 'a'"):
        engine.generate_all(prompt, 4, adapters="a")
    assert engine.generate_all(prompt, 4, adapters="b") == before
    engine.load_adapter("a", new)
    other = make(folders)
    other.load_adapter("x", new)
    assert engine.generate_all(prompt, 4, adapters="a") == other.generate_all(prompt, 4, adapters="x")
