"""Adapters at the edges of what banks, engines, files and the command line take (no GPU)."""

import pytest
import torch

from adapter_helpers import random_factors, write_adapter
from helpers import prompts_for
from kernel_rush_kawk_b200.parts.adapters import AdapterBank, AdapterError
from kernel_rush_kawk_b200.weights.adapters import read_adapter
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


def test_files_of_more_than_products(tmp_path):
    """Adapters whose weights are changed for them, or that do not run on every token, would be taken for others."""
    factors = {"model.layers.0.mlp.down_proj.weight": (torch.randn(3, 8), torch.randn(6, 3), 1.0)}
    refused = [dict(init_lora_weights=v) for v in ("pissa", "pissa_niter_16", "olora", "loftq", "corda")] + [
        dict(alora_invocation_tokens=[7, 8]), dict(layer_replication=[[0, 2]]), dict(use_qalora=True), dict(lora_bias=True), dict(trainable_token_indices=[1]),
        dict(peft_type="LOHA")]
    for i, config in enumerate(refused):
        with pytest.raises(AdapterError, match="not taken"):
            read_adapter(write_adapter(tmp_path / f"r{i}", factors, **config))
    for i, config in enumerate([dict(init_lora_weights=v) for v in (True, False, None, "gaussian", "eva", "orthogonal")] + [
            dict(peft_type="LORA", use_qalora=False, alora_invocation_tokens=None, layer_replication=None, lora_bias=False, trainable_token_indices=None)]):
        assert set(read_adapter(write_adapter(tmp_path / f"t{i}", factors, **config))) == set(factors)


@pytest.mark.parametrize("given", [["{0}"], ["{0}="], ["=x"], ["-={0}"], ["x={0}", "x={0}"], ["x={0}", "y"]])
def test_command_line_adapters_have_a_name_and_a_folder(folders, tmp_path, capsys, monkeypatch, given):
    """Without a folder the current one would be read; of one name given twice, or of '-', one adapter could not be asked for."""
    from kernel_rush_kawk_b200.cli import main

    folder = write_adapter(tmp_path / "a", {"model.layers.0.mlp.down_proj.weight": (torch.randn(3, 8), torch.randn(6, 3), 1.0)})
    monkeypatch.chdir(folder)
    with pytest.raises(SystemExit):
        main(["generate", "--model", str(folders[NAME]), "--prompt-ids", "1,2"] + ["--adapter=" + a.format(folder) for a in given])
    assert "NAME=DIR" in capsys.readouterr().err.splitlines()[-1]
