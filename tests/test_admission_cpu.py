"""What requests are counted to need of the cache (no GPU): the pages of sequences that give keys up, the pools that are built for them, and the
batches that they form. Whole generations run with the kernels' plain restatement."""

import random

import pytest
import torch

from cache_engine_helpers import CacheTorchOps
from helpers import prompts_for
from kernel_rush_kawk_b200 import Engine, KeyEviction
from kernel_rush_kawk_b200.cache import PAGE
from kernel_rush_kawk_b200.engine.generate import pages_needed, rows_held, split_into_batches


def cpu_engine(folders, name, **kw):
    args = dict(dtype="float32", device="cpu", ops=CacheTorchOps(torch.float32), max_slots=8, use_cuda_graphs=False)
    args.update(kw)
    return Engine(folders[name], **args)


# -- keys that are given up ------------------------------------------------------------------------------
def most_rows(prompt, new, eviction, pieces):
    """The most rows that a sequence holds, step by step: its prompt in these pieces, then token by token."""
    held = most = 0
    for n in list(pieces) + [1] * (new - 1):
        if held >= eviction.keep + eviction.every:
            held = eviction.keep
        held += n
        most = max(most, held)
    return most


def test_rows_that_an_evicting_sequence_comes_to_hold():
    rng = random.Random(2)
    for _ in range(3000):
        keep = rng.randint(1, 60)
        eviction = KeyEviction(keep=keep, recent=rng.randint(0, keep), every=rng.randint(1, 40))
        prompt, new, at_once = rng.randint(1, 200), rng.randint(1, 120), rng.choice([1, 7, 32, 64, 500])
        bound = rows_held(prompt, new, eviction, at_once)
        assert bound <= prompt + new - 1
        pieces, left = [], prompt  # of any sizes up to a pass's
        while left:
            pieces.append(min(left, rng.choice([at_once, rng.randint(1, at_once)])))
            left -= pieces[-1]
        assert most_rows(prompt, new, eviction, pieces) <= bound
        if prompt <= at_once:  # one pass: the bound is what it holds
            assert bound == max(most_rows(prompt, new, eviction, [prompt]), min(prompt + new - 1, keep + eviction.every))
    assert rows_held(70, 10) == 79 and pages_needed(70, 10) == 2
    assert rows_held(70, 10000, KeyEviction(keep=100, every=20), 64) == 120
    assert split_into_batches([100, 100, 100], 5000, 8, 6, KeyEviction(keep=100, every=20), 512) == [[0, 1, 2]]


def test_a_pool_that_the_kept_keys_fit_takes_longer_requests(folders):
    """The command line's way in serves what a generation serves."""
    name, eviction = "tiny_a", KeyEviction(keep=40, recent=10, every=24)
    prompts = prompts_for(name, [30, 100, 5], 3)
    engine = cpu_engine(folders, name, eviction=eviction, max_tokens=2 * PAGE, max_slots=4)
    one_by_one = [[s[0] for s in engine.generate([p], 60)] for p in prompts]
    assert all(len(t) == 60 for t in one_by_one)
    assert engine.generate_all(prompts, 60) == one_by_one
    engine.cache.check()
    with pytest.raises(ValueError, match="needs 192 cached tokens; the cache holds 128"):
        engine.generate_all(prompts_for(name, [130], 3), 2)  # a prompt that one pass brings has all of its keys at once


@pytest.mark.parametrize("rows", [32, 4096])
def test_pools_are_as_large_as_what_the_sequences_hold(folders, rows):
    """A pool without a fixed size: no more pages than the rows that are held, prompts in one pass or in pieces, and these are enough."""
    name, eviction = "tiny_b", KeyEviction(keep=40, recent=10, every=9)
    prompts = prompts_for(name, [100, 50, 7], 4)
    engine = cpu_engine(folders, name, eviction=eviction, max_step_rows=rows)
    want = list(engine.generate(prompts, 60))
    assert len(want) == 60
    assert engine.cache.n_pages == 4, "100 rows (80 in pieces of 32: 48 held and a piece), 50 and 49 (40 kept and 9 more)"
    engine.cache.check()
    plenty = cpu_engine(folders, name, eviction=eviction, max_step_rows=rows, max_tokens=64 * 40)
    assert list(plenty.generate(prompts, 60)) == want
    assert cpu_engine(folders, name, eviction=eviction, max_step_rows=rows).generate_all(prompts, 60) == [[s[i] for s in want] for i in range(3)]


def test_sums_and_positions_are_no_wider_than_the_pool(folders):
    """A slot never holds more rows than the pool has pages for; a pass bounds it where that is less."""
    prompts = prompts_for("tiny_a", [30, 20], 3)
    engine = cpu_engine(folders, "tiny_a", eviction=KeyEviction(keep=50, recent=10, every=9))
    list(engine.generate(prompts, 50))
    assert engine.cache.n_pages == 2, "59 rows each at most"
    assert engine.cache.view(0).scores.shape == engine.cache.view(0).positions.shape == (8, 2, 2 * PAGE)
    engine = cpu_engine(folders, "tiny_a", eviction=KeyEviction(keep=50, recent=10, every=9), max_step_rows=60, max_tokens=64 * 40)
    assert engine.cache.width == 2, "50 + 9 - 1 rows before a pass, and the pass"
