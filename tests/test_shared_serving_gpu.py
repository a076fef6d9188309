"""Shared prefixes and evictions as a server runs them, on the GPU: with few captured steps kept."""

import pytest

from helpers import assert_greedy_token, prompts_for, windows_of
import plain_qwen3 as plain

pytestmark = pytest.mark.gpu


def engine_of(folders, name, **kw):
    from kernel_rush_kawk_b200 import Engine

    args = dict(dtype="bfloat16", max_slots=12)
    args.update(kw)
    return Engine(folders[name], **args)


def family(name, length, tails, seed):
    doc = prompts_for(name, [length], seed)[0]
    return [doc + t for t in prompts_for(name, tails, seed + 1)]


def assert_greedy(folder, name, prompts, steps, what):
    """Every token that was drawn is the plain decoder's largest, or ties with it within the arithmetic."""
    cfg, w = plain.read_folder(folder)
    for i, p in enumerate(prompts):
        seq = list(p)
        for t, step in enumerate(steps):
            if step[i] is None:
                break
            assert_greedy_token(cfg, w, seq, step[i], "bfloat16", windows_of(name), f"{what}, request {i} step {t}")
            seq.append(step[i])


def test_few_captured_steps_of_groups_are_kept(folders, monkeypatch):
    """Sequences end one by one, so that every few steps another number of them goes on; the steps captured for those used last stay."""
    from kernel_rush_kawk_b200.cache import prefix
    from kernel_rush_kawk_b200.engine.step import Stepper

    monkeypatch.setattr(prefix, "SHARE_BYTES", 0)
    monkeypatch.setattr(prefix, "JOIN_STEPS", -1e9)
    monkeypatch.setattr(Stepper, "MAX_GROUP_GRAPHS", 2)
    name = "tiny_a"
    engine = engine_of(folders, name)
    prompts = family(name, 130, [3, 12, 1, 30, 7], 21)
    steps = list(engine.generate(prompts, 10, share_prefix=True))
    stops = {steps[2][0], steps[4][1], steps[6][2], steps[8][3]}
    for _ in range(2):
        got = list(engine.generate(prompts, 10, share_prefix=True, stop_token_ids=stops))
        assert 1 <= sum(isinstance(key, tuple) for key in engine.stepper._graphs) <= 2
        assert_greedy(folders[name], name, prompts, got, "sequences that end")
        for i in range(len(prompts)):
            mine = [s[i] for s in got if s[i] is not None]
            assert len(mine) == 10 or mine[-1] in stops
    assert_greedy(folders[name], name, prompts, steps, "few captured steps")
    assert engine.cache.live == 0
    engine.ops.check()
