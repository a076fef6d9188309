"""Shared pages, forks and evictions around the kernels (no GPU): the ledger's counts, what is refused, how prompts are grouped,
and whole generations with the kernels' plain restatement."""

import random

import pytest
import torch

from cache_engine_helpers import CacheTorchOps, PlainEvicting
from helpers import assert_close, prompts_for
from kernel_rush_kawk_b200 import KeyEviction
from kernel_rush_kawk_b200.cache import PAGE, CacheError, PageLedger, PrefixGroups, SequenceCache
from kernel_rush_kawk_b200.engine.generate import shared_prefixes
from kernel_rush_kawk_b200.parts.base import KVNeed, StateNeed


@pytest.fixture(autouse=True)
def always_shared(monkeypatch):
    """Tiny models take the paths that large ones do."""
    from kernel_rush_kawk_b200.cache import prefix

    monkeypatch.setattr(prefix, "SHARE_BYTES", 0)
    monkeypatch.setattr(prefix, "JOIN_STEPS", -1e9)


def cpu_engine(folders, name, dtype="float32", **kw):
    from kernel_rush_kawk_b200 import Engine

    ops = CacheTorchOps(torch.float32 if dtype == "float32" else torch.bfloat16)
    args = dict(dtype=dtype, device="cpu", ops=ops, max_tokens=64 * 40, max_slots=8, use_cuda_graphs=False)
    args.update(kw)
    return Engine(folders[name], **args)


# -- pages held by several -------------------------------------------------------------------------------
def test_a_shared_page_goes_back_with_its_last_holder():
    led = PageLedger(n_pages=10, n_slots=4, width=5, page_size=PAGE, ring=None)
    led.grow(0, 3 * PAGE)
    assert led.share(0, 1, 2) == [(0, led.pages[0][0]), (1, led.pages[0][1])]
    led.share(1, 2, 1)
    led.grow(1, 3 * PAGE)
    led.check()
    assert led.pool.held == 4
    led.release(0)
    led.check()
    assert led.pool.held == 3
    led.shrink(1, PAGE)
    led.check()
    assert led.pool.held == 1 and led.pages[1] == led.pages[2]
    led.release(2)
    led.check()
    led.release(1)
    led.check()
    assert led.pool.held == 0 and not led.holders
    led.grow(3, PAGE)
    with pytest.raises(CacheError):
        led.share(3, 0, 2)  # more than there are
    with pytest.raises(CacheError):
        led.share(0, 3, 0)  # a slot with pages of its own
    with pytest.raises(CacheError):
        PageLedger(4, 2, 2, PAGE, ring=2).share(0, 1, 0)
    led.pages[0] = [led.pages[3][0]]
    with pytest.raises(CacheError, match="held by two slots"):
        led.check()


def make_cache(needs=None, **kw):
    args = dict(max_tokens=64 * 20, max_slots=6, max_context=64 * 8, device="cpu", dtype=torch.bfloat16)
    args.update(kw)
    return SequenceCache(needs or [KVNeed(2, 16), KVNeed(2, 16)], **args)


def test_forks_hold_the_same_pages_until_they_are_freed():
    cache = make_cache([KVNeed(2, 16), StateNeed((3,))])
    a = cache.alloc()
    cache.reserve(a, 130)
    cache.advance(a, 128)
    cache._state_groups[0].state[:, a] = 5
    b, c = cache.fork(a, 128), cache.fork(a, 128)
    cache.sync()
    assert (cache.view(1).state[[b, c]] == 5).all() and cache.length[b] == 128
    assert cache.view(0).table[b, :2].tolist() == cache.view(0).table[a, :2].tolist()
    for s in (b, c):
        cache.reserve(s, 129)
    assert len({cache.view(0).table.data_ptr()}) == 1
    host = cache._kv_groups[0].table_host
    assert len({host[s, 2] for s in (a, b, c)}) == 3, "what follows is each one's own"
    assert cache.shared_groups([a, b, c]) == ([3], [128])
    d = cache.alloc()
    assert cache.shared_groups([b, d, a, c]) == ([1, 1, 2], [0, 0, 128])
    cache.free(a)
    cache.check()
    assert cache.shared_groups([b, c]) == ([2], [128])
    again = cache.alloc()  # the slot that the source had
    assert again == a and cache.shared_groups([again, b]) == ([1, 1], [0, 0])
    for s in (again, b, c, d):
        cache.free(s)
    cache.check()
    assert cache.free_pages() == cache.n_pages


def test_forks_of_forks():
    cache = make_cache()
    a = cache.alloc()
    cache.reserve(a, 300)
    cache.advance(a, 300)
    b = cache.fork(a, 256)
    c = cache.fork(b, 256)
    short = cache.fork(a, 128)  # shares less than the family does: pages, but no group
    assert cache.shared_groups([a, b, c, short]) == ([3, 1], [256, 0])
    cache.reserve(c, 320)
    cache.advance(c, 64)
    long = cache.fork(c, 320)  # shares more with c, and what all share with all
    assert cache.shared_groups([a, c, long]) == ([3], [256])
    none = cache.fork(a, 0)
    assert cache.shared_groups([a, none]) == ([1, 1], [0, 0])
    for s in (a, b, c, short, long, none):
        cache.free(s)
    cache.check()


def test_forks_that_are_refused():
    cache = make_cache([KVNeed(2, 16), StateNeed((3,))])
    a = cache.alloc()
    cache.reserve(a, 200)
    cache.advance(a, 200)
    for length in (-64, 1, 63, 256, 128):  # 128: the state there is gone
        with pytest.raises(CacheError):
            cache.fork(a, length)
    with pytest.raises(CacheError, match="not held"):
        cache.fork(a + 1, 0)
    window = make_cache([KVNeed(2, 16, window=100)])
    assert not window.can_share()
    with pytest.raises(CacheError):
        window.fork(window.alloc(), 0)
    evicting = make_cache(eviction=KeyEviction(64))
    assert not evicting.can_share()
    with pytest.raises(CacheError):
        evicting.fork(evicting.alloc(), 0)
    with pytest.raises(CacheError):
        make_cache([KVNeed(2, 16, window=100)], eviction=KeyEviction(64))
    assert cache.live == 1, "a refused fork takes no slot"


def test_random_forks_lose_no_page():
    rng = random.Random(4)
    cache = make_cache(max_tokens=64 * 60, max_slots=10)
    live = []
    for _ in range(600):
        what = rng.random()
        if live and what < 0.35:
            cache.free(live.pop(rng.randrange(len(live))))
        elif len(live) < 10 and what < 0.7:
            if live and rng.random() < 0.7:
                source = rng.choice(live)
                live.append(cache.fork(source, cache.length[source] // PAGE * PAGE))
            else:
                live.append(cache.alloc())
        elif live:
            s = rng.choice(live)
            n = rng.randint(0, 512 - cache.length[s])
            try:
                cache.reserve(s, cache.length[s] + n)
                cache.advance(s, n)
            except CacheError:
                pass
        cache.check()
        for sizes, lengths in [cache.shared_groups(live)]:
            at = 0
            for size, length in zip(sizes, lengths):
                pages = [cache._kv_groups[0].ledger.pages[s][:length // PAGE] for s in live[at:at + size]]
                assert all(p == pages[0] for p in pages), "a group's members hold the same pages"
                at += size
    for s in live:
        cache.free(s)
    cache.check()
    assert cache.free_pages() == cache.n_pages


def test_groups_refuse_what_is_none():
    for sizes, lengths in [([], []), ([1], [64, 64]), ([0], [64]), ([2], [63]), ([2], [-64])]:
        with pytest.raises(CacheError):
            PrefixGroups(sizes, lengths, "cpu")
    g = PrefixGroups([2, 1], [128, 0], "cpu")
    assert g.cu.tolist() == [0, 2, 3] and g.length.tolist() == [128, 0] and g.group.tolist() == [0, 0, 1]
    g.update(PrefixGroups([1, 2], [64, 192], "cpu"))
    assert g.cu.tolist() == [0, 1, 3] and g.lengths == (64, 192)
    for other in (PrefixGroups([3], [64], "cpu"), PrefixGroups([2, 2], [64, 64], "cpu"), PrefixGroups([1, 2], [0, 0], "cpu")):
        with pytest.raises(CacheError):
            g.update(other)


def test_evictions_that_make_no_sense_are_refused():
    for kw in [dict(keep=0), dict(keep=5, recent=6), dict(keep=5, recent=-1), dict(keep=5, every=0), dict(keep=5, observe=0)]:
        with pytest.raises(CacheError):
            KeyEviction(**kw)


# -- how prompts are grouped -----------------------------------------------------------------------------------
def test_prompts_that_begin_alike_form_groups():
    doc, other = list(range(200)), list(range(500, 700))
    assert shared_prefixes([[1, 2], [1, 2]]) == [([0], 0), ([1], 0)], "less than a page"
    groups = shared_prefixes([doc + [7], other, doc + [3, 4], [9], doc])
    assert sorted((sorted(m), n) for m, n in groups) == [([0, 2, 4], 192), ([1], 0), ([3], 0)]
    # a prompt is never shared whole: its last token's logits are asked for
    assert shared_prefixes([doc[:128]] * 3) == [([0, 1, 2], 64)]
    assert shared_prefixes([doc[:129]] * 2) == [([0, 1], 128)]
    assert [n for _, n in shared_prefixes([doc[:64], doc[:64]])] == [0, 0]
    # two that share three pages do not give them up for a third that shares one
    a, b, c = doc[:64] + other[:64], doc[:199], doc[:198] + [0]
    assert sorted((sorted(m), n) for m, n in shared_prefixes([a, b, c])) == [([0], 0), ([1, 2], 192)]


def test_groups_share_what_they_say():
    rng = random.Random(1)
    for _ in range(200):
        stems = [[rng.randint(0, 1) for _ in range(rng.randint(1, 300))] for _ in range(3)]
        prompts = [rng.choice(stems)[:rng.randint(1, 300)] + [rng.randint(0, 1) for _ in range(rng.randint(0, 80))] for _ in range(rng.randint(1, 9))]
        groups = shared_prefixes(prompts)
        assert sorted(i for m, _ in groups for i in m) == list(range(len(prompts)))
        for members, n in groups:
            assert n % PAGE == 0 and (n > 0) == (len(members) > 1)
            assert all(prompts[i][:n] == prompts[members[0]][:n] and len(prompts[i]) > n for i in members)


# -- generations ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_shared_prefixes_generate_the_same(folders, dtype):
    name = "tiny_a"
    doc = prompts_for(name, [150], 5)[0]
    prompts = [doc + t for t in prompts_for(name, [3, 40, 1], 6)] + prompts_for(name, [20, 5], 7) + [doc[:130]]
    engine = cpu_engine(folders, name, dtype)
    want = list(engine.generate(prompts, 5))
    before = engine.stepper.passes
    got = list(engine.generate(prompts, 5, share_prefix=True))
    assert got == want
    assert engine.cache.live == 0 and engine.stepper.passes > before
    assert (engine.ops.calls["shared"] > 0) == (dtype == "bfloat16"), "32-bit steps stay what they are without sharing"
    engine.cache.check()
    sampled = list(engine.generate(prompts, 4, temperature=0.9, seed=3))
    assert list(engine.generate(prompts, 4, temperature=0.9, seed=3, share_prefix=True)) == sampled, "a request's draws are its own"
    assert engine.generate_all(prompts, 3, share_prefix=True, max_batch=3) == engine.generate_all(prompts, 3, max_batch=3)


def test_shared_prefixes_with_stops_and_an_early_end(folders):
    name = "tiny_b"
    doc = prompts_for(name, [70], 8)[0]
    prompts = [doc + [i] for i in range(4)]
    engine = cpu_engine(folders, name, "bfloat16")
    want = list(engine.generate(prompts, 6))
    stop = [want[1][0], want[2][2]]
    assert list(engine.generate(prompts, 6, stop_token_ids=stop, share_prefix=True)) == list(engine.generate(prompts, 6, stop_token_ids=stop))
    run = engine.generate(prompts, 6, share_prefix=True)
    next(run)
    run.close()
    assert engine.cache.live == 0
    engine.cache.check()


def test_windows_share_no_prefix(folders):
    engine = cpu_engine(folders, "tiny_w")
    with pytest.raises(ValueError, match="window"):
        list(engine.generate([[1, 2]], 2, share_prefix=True))
    assert engine.cache.live == 0


@pytest.mark.parametrize("name", ["tiny_a", "tiny_b"])
@pytest.mark.parametrize("observe", [None, 5])
def test_evicting_steps_agree_with_plain(folders, name, observe):
    from kernel_rush_kawk_b200 import StepEntry

    eviction = KeyEviction(keep=40, recent=12, every=9, observe=observe)
    engine = cpu_engine(folders, name, eviction=eviction)
    seqs = prompts_for(name, [95, 30], seed=31)
    plains = [PlainEvicting(folders[name], 40, 12, 9, observe) for _ in seqs]
    slots = [engine.cache.alloc() for _ in seqs]
    steps = [(60, 4), (61, 5), (75, 20)] + [(75 + i, 20 + i) for i in range(1, 11)] + [(95, 30)]
    done = [0, 0]
    for to in steps:
        entries, refs = [], []
        for i in (0, 1):
            if to[i] > done[i]:
                entries.append(StepEntry(slots[i], seqs[i][done[i]:to[i]], list(range(to[i] - done[i]))))
                refs.append(plains[i].step(seqs[i][done[i]:to[i]]))
                done[i] = to[i]
        assert_close(engine.step(entries), torch.cat(refs).float(), "float32", f"up to {to}")
        for i in (0, 1):
            n = engine.cache.length[slots[i]]
            assert n == len(plains[i].rows[0][0]) and n + engine.cache.evicted[slots[i]] == done[i]
            assert len(engine.cache._kv_groups[0].ledger.pages[slots[i]]) == -(-n // PAGE)
            for layer in range(plains[i].cfg.layers):
                for h in range(plains[i].cfg.kv_heads):
                    got = engine.cache.view(layer).positions[slots[i], h, :n].tolist()
                    assert sorted(got) == sorted(plains[i].held(layer, h))
    assert engine.ops.calls["evict"] > 1
    for s in slots:
        engine.cache.free(s)
    engine.cache.check()


def test_an_eviction_that_never_comes_changes_nothing(folders):
    name = "tiny_a"
    prompts = prompts_for(name, [50, 7], 9)
    want = list(cpu_engine(folders, name).generate(prompts, 8))
    assert list(cpu_engine(folders, name, eviction=KeyEviction(keep=500)).generate(prompts, 8)) == want


def test_an_evicting_cache_holds_longer_sequences_than_it_has_pages_for(folders):
    """Rows are bounded, positions are not: pages for 128 rows serve a sequence of 400."""
    engine = cpu_engine(folders, "tiny_a", eviction=KeyEviction(keep=40, recent=10, every=24), max_tokens=128, max_slots=1)
    slot = engine.cache.alloc()
    from kernel_rush_kawk_b200 import StepEntry
    for _ in range(20):
        engine.step([StepEntry(slot, list(range(20)), [19])])
    assert engine.cache.length[slot] + engine.cache.evicted[slot] == 400 and engine.cache.length[slot] < 84
    with pytest.raises(CacheError, match="exceeds the longest"):
        engine.cache.reserve(slot, engine.max_context - 380 + engine.cache.length[slot])


def test_models_that_cannot_evict_are_refused(folders):
    with pytest.raises(ValueError, match="window"):
        cpu_engine(folders, "tiny_w", eviction=KeyEviction(64))
    engine = cpu_engine(folders, "tiny_a", eviction=KeyEviction(64))
    with pytest.raises(ValueError, match="evicted"):
        list(engine.generate([[1, 2]], 2, share_prefix=True))


def test_the_command_line_takes_the_options():
    from kernel_rush_kawk_b200.cli import build_parser, main

    args = build_parser().parse_args("generate --random tiny_a --prompt-ids 1 --share-prefix".split())
    assert args.share_prefix and args.keep_keys is None
    for bad in ("--keep-recent 5", "--keep-keys 64 --share-prefix"):
        with pytest.raises(SystemExit):
            main(f"generate --random tiny_a --prompt-ids 1 {bad}".split())


def test_the_lines_between_shared_and_alone(monkeypatch):
    """Both sides of the measured lines, at sizes that were measured."""
    from kernel_rush_kawk_b200.cache import prefix

    monkeypatch.undo()
    single = lambda n, p, row=4096: prefix.single_tokens_share([n], [p], row)
    assert [single(2, 2048), single(2, 8192), single(8, 1024), single(8, 4096), single(64, 64), single(64, 8192)] == [False, True, False, True, False, True]
    assert not single(1, 1 << 20) and not prefix.single_tokens_share([1, 1], [0, 0], 4096)
    longer = lambda n, t, p, per=4, kv=8: prefix.longer_steps_share([n], [p], [t] * n, per, kv)
    assert [longer(2, 4, 4096), longer(4, 60, 4096), longer(2, 250, 4096)] == [True] * 3
    assert [longer(16, 60, 4096), longer(4, 250, 4096), longer(32, 60, 4096), longer(16, 16, 256)] == [False] * 4
    assert prefix.longer_steps_share([16], [4096], [90 - 90 * i // 32 for i in range(16)], 4, 8)
