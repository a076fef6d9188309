"""What requests are counted to need of the cache (no GPU): the pages of sequences that give keys up, the pools that are built for them, and the
batches that they form. Whole generations run with the kernels' plain restatement."""

import random

import pytest
import torch

from cache_engine_helpers import CacheTorchOps
from helpers import prompts_for
from kernel_rush_kawk_b200 import Engine, KeyEviction
from kernel_rush_kawk_b200.cache import PAGE
from kernel_rush_kawk_b200.engine.generate import pages_needed, rows_held, shared_pages, split_into_batches
from test_generate_loop import make


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


# -- beginnings that are shared -----------------------------------------------------------------------------
def test_shared_pages_are_counted_once():
    """What a batch is counted to need is what it comes to hold, to the page, and a pool of that size runs it."""
    rng = random.Random(5)
    for _ in range(120):
        stems = [[rng.randint(0, 1) for _ in range(rng.randint(1, 300))] for _ in range(2)]
        prompts = [rng.choice(stems)[:rng.randint(1, 300)] + [rng.randint(0, 1) for _ in range(rng.randint(0, 70))] for _ in range(rng.randint(1, 7))]
        new = rng.randint(1, 80)
        pages = shared_pages(prompts, new)
        assert pages <= sum(pages_needed(len(p), new) for p in prompts)
        script = {i: [3] * new for i in range(len(prompts))}
        loop, cache, stepper, _ = make(script, max_tokens=pages * PAGE, max_slots=8)
        step, held = stepper.step, []
        stepper.step = lambda entries: (step(entries), held.append(cache.n_pages - cache.free_pages()))[0]
        assert len(list(loop.run_batch(prompts, new, share_prefix=True))) == new
        assert max(held) == pages
        cache.check()
        assert loop.run_requests(prompts, new, share_prefix=True) == [script[i] for i in range(len(prompts))]
    doc = list(range(320))
    prompts = [doc + [i] * 3 for i in range(8)]
    assert sum(pages_needed(len(p), 2) for p in prompts) == 48 and shared_pages(prompts, 2) == 5 + 8


def test_batches_of_requests_that_share():
    """As many neighbours as slots and pages take, the shared pages counted once; each batch of those that are tried fits."""
    doc = list(range(320))
    prompts = [doc + [i] * 3 for i in range(8)]
    lens = [len(p) for p in prompts]
    split = lambda slots, pages, ps=prompts: split_into_batches([len(p) for p in ps], 2, slots, pages, prompts=ps)
    assert split(8, 13) == [list(range(8))] and split(8, 14) == [list(range(8))]
    assert split(3, 13) == [[0, 1, 2], [3, 4, 5], [6, 7]]
    assert split(8, 10) == [[0, 1, 2, 3, 4], [5, 6, 7]]
    assert split_into_batches(lens, 2, 8, 14) == [[0, 1], [2, 3], [4, 5], [6, 7]], "not shared: six pages each"
    with pytest.raises(ValueError, match="request 2 needs 640"):
        split(8, 8, prompts[:2] + [list(range(600))])
    rng = random.Random(6)
    for _ in range(200):
        stems = [[rng.randint(0, 1) for _ in range(200)] for _ in range(2)]
        some = [rng.choice(stems)[:rng.randint(1, 200)] + [rng.randint(0, 1)] for _ in range(rng.randint(1, 12))]
        slots, pages = rng.randint(1, 12), rng.randint(4, 20)
        batches = split(slots, pages, some)
        assert [i for b in batches for i in b] == list(range(len(some)))
        assert all(1 <= len(b) <= slots and shared_pages([some[i] for i in b], 2) <= pages for b in batches)
        plain = split_into_batches([len(p) for p in some], 2, slots, pages)
        assert len(batches) <= len(plain), "sharing costs no batch"


def test_a_pool_that_the_shared_pages_fit_runs_all_at_once(folders):
    name = "tiny_a"
    doc = prompts_for(name, [200], 5)[0]
    prompts = [doc + t for t in prompts_for(name, [3, 9, 1, 30, 2, 5, 4, 60], 6)]
    want = [list(s) for s in zip(*cpu_engine(folders, name, max_tokens=64 * 60).generate(prompts, 4))]
    engine = cpu_engine(folders, name, max_tokens=14 * PAGE)
    before = engine.loop.steps
    assert engine.generate_all(prompts, 4, share_prefix=True) == want
    assert engine.loop.steps - before == 4, "one batch"
    pool = cpu_engine(folders, name)
    assert [list(s) for s in zip(*pool.generate(prompts, 4, share_prefix=True))] == want
    assert pool.cache.n_pages == 3 + 8 + 1, "three pages of the document, one of each prompt's own, a second of the longest's"
    pool = cpu_engine(folders, name)
    assert pool.generate_all(prompts, 4, share_prefix=True) == want and pool.cache.n_pages == 12
    assert pool.generate_all(prompts, 4) == want and pool.cache.n_pages == sum(pages_needed(len(p), 4) for p in prompts), "the pool grows when it must"
    pool = cpu_engine(folders, name)
    assert pool.generate_all(prompts, 4, share_prefix=True, max_batch=3) == want and pool.cache.n_pages < 12


def test_speeds_count_the_tokens_that_ran():
    """A batch's prompt tokens are all of them; its speed is by those that went through the model."""
    doc = list(range(320))
    prompts = [doc + [i] * 3 for i in range(8)] + [[7, 8]]
    loop, _, stepper, _ = make({i: [3] for i in range(9)}, max_slots=9)
    list(loop.run_batch(prompts, 1, share_prefix=True))
    ran = sum(len(tokens) for call in stepper.calls for _, tokens, _ in call)
    assert ran == 320 + 8 * 3 + 2
    stats = loop.stats
    assert stats.prompt_tokens == 8 * 323 + 2 and stats.shared_tokens == 7 * 320
    assert stats.prefill_tokens_per_s == pytest.approx(ran * 1000 / stats.prefill_ms) and "(2240 shared)" in stats.line()
    loop, _, _, _ = make({i: [3] for i in range(9)}, max_tokens=64 * 60, max_slots=9)
    list(loop.run_batch(prompts, 1))
    assert loop.stats.shared_tokens == 0 and loop.stats.prefill_tokens_per_s == pytest.approx(2586 * 1000 / loop.stats.prefill_ms)
    assert "shared" not in loop.stats.line()


@pytest.mark.parametrize("preset,why", [("zadunex_tiny", "'mamba2' layer keeps other things than keys"), ("taredra_tiny", "'parallel' layer keeps other things than keys"),
                                        ("disorax_tiny", "keeps a window of keys"), ("zefapel_tiny", "'gla' layer keeps other things than keys")])
def test_models_whose_layers_keep_other_things_evict_no_keys(preset, why):
    with pytest.raises(ValueError, match=why):
        Engine.from_random(preset, dtype="float32", device="cpu", ops=CacheTorchOps(torch.float32), eviction=KeyEviction(64))


@pytest.mark.parametrize("options", ["--keep-keys 0", "--keep-keys 10 --keep-recent 11", "--keep-keys 10 --keep-recent -1"])
def test_the_command_line_says_what_keeps_nothing(options, capsys):
    from kernel_rush_kawk_b200.cli import main

    with pytest.raises(SystemExit):
        main(f"generate --random tiny_a --prompt-ids 1 {options}".split())
    assert "at least one key stays" in capsys.readouterr().err
