"""Shared prefixes and evictions through the engine on the GPU: whole generations and steps against the plain decoders."""

import pytest
import torch

from cache_engine_helpers import PlainEvicting
from helpers import assert_close, assert_greedy_token, plain_logits, prompts_for, windows_of
import plain_qwen3 as plain

pytestmark = pytest.mark.gpu

NAMES = ["tiny_a", "tiny_b"]


@pytest.fixture(autouse=True)
def always_shared(monkeypatch):
    """Tiny models take the paths that large ones do."""
    from kernel_rush_kawk_b200.cache import prefix

    monkeypatch.setattr(prefix, "SHARE_BYTES", 0)
    monkeypatch.setattr(prefix, "JOIN_STEPS", -1e9)


def engine_of(folders, name, **kw):
    from kernel_rush_kawk_b200 import Engine

    args = dict(dtype="bfloat16", max_slots=12)
    args.update(kw)
    return Engine(folders[name], **args)


def family(name, length, tails, seed):
    doc = prompts_for(name, [length], seed)[0]
    return [doc + t for t in prompts_for(name, tails, seed + 1)]


@pytest.mark.parametrize("name", NAMES)
def test_float32_generations_are_the_same_shared_or_not(folders, name):
    prompts = family(name, 150, [3, 40, 1], 5) + prompts_for(name, [20], 7) + family(name, 66, [9, 9], 9)
    engine = engine_of(folders, name, dtype="float32")
    want = list(engine.generate(prompts, 6))
    assert list(engine.generate(prompts, 6, share_prefix=True)) == want
    from kernel_rush_kawk_b200 import StepEntry
    engine.open_cache(64 * 60, 8)
    whole, first = engine.cache.alloc(), engine.cache.alloc()
    a = engine.step([StepEntry(whole, prompts[0], [len(prompts[0]) - 1])])
    engine.step([StepEntry(first, prompts[0][:128], [])])
    forks = [engine.cache.fork(first, 128) for _ in range(2)]
    b = engine.step([StepEntry(s, prompts[0][128:], [len(prompts[0]) - 129]) for s in forks])
    assert torch.equal(a, b[:1]) and torch.equal(a, b[1:]), "32-bit logits are equal to the bit, shared or not"


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("graphs", [True, False])
def test_bfloat16_steps_behind_a_shared_prefix_agree_with_plain(folders, name, graphs):
    from kernel_rush_kawk_b200 import StepEntry

    engine = engine_of(folders, name, use_cuda_graphs=graphs, max_tokens=64 * 60)
    seqs = family(name, 192, [4, 70, 33], 15)
    alone = prompts_for(name, [90], 16)[0]
    refs = [plain_logits(folders[name], name, s + prompts_for(name, [6], 17)[0], "bfloat16") for s in seqs]
    more = prompts_for(name, [6], 17)[0]
    first = engine.cache.alloc()
    engine.step([StepEntry(first, seqs[0][:192], [])])
    slots = [first] + [engine.cache.fork(first, 192) for _ in seqs[1:]]
    other = engine.cache.alloc()
    out = engine.step([StepEntry(s, q[192:], [len(q) - 193]) for s, q in zip(slots, seqs)] + [StepEntry(other, alone, [89])])
    for i, q in enumerate(seqs):
        assert_close(out[i:i + 1], refs[i][len(q) - 1:len(q)], "bfloat16", f"the questions' step, {i}")
    ref = plain_logits(folders[name], name, alone + more, "bfloat16")
    for t, tok in enumerate(more):
        out = engine.step([StepEntry(s, [tok], [0]) for s in slots] + [StepEntry(other, [tok], [0])])
        for i, q in enumerate(seqs):
            assert_close(out[i:i + 1], refs[i][len(q) + t:len(q) + t + 1], "bfloat16", f"token {t} of sequence {i}")
        assert_close(out[3:], ref[90 + t:91 + t], "bfloat16", "the sequence beside them")
    engine.cache.free(first)  # the others go on without it
    out = engine.step([StepEntry(s, [1], [0]) for s in slots[1:]])
    for i in (1, 2):
        want = plain_logits(folders[name], name, seqs[i] + more + [1], "bfloat16")[-1:]
        assert_close(out[i - 1:i], want, "bfloat16", "after the first has gone")
    engine.cache.check()


@pytest.mark.parametrize("name", NAMES)
def test_bfloat16_generations_behind_shared_prefixes(folders, name):
    """Greedy tokens, run ahead from captured steps, while sequences end one by one; then the captured steps again for other groups."""
    cfg, w = plain.read_folder(folders[name])
    engine = engine_of(folders, name)
    for seed, length in ((21, 130), (22, 200)):
        prompts = family(name, length, [3, 12, 1, 30], seed) + prompts_for(name, [20], seed + 5) + family(name, 70, [5, 6], seed + 9)
        steps = list(engine.generate(prompts, 8, share_prefix=True))
        stop = [steps[2][0], steps[4][1]]
        for i, p in enumerate(prompts):
            seq = list(p)
            for t in range(0, 8):
                assert_greedy_token(cfg, w, seq, steps[t][i], "bfloat16", windows_of(name), f"request {i} step {t}")
                seq.append(steps[t][i])
        again = list(engine.generate(prompts, 8, share_prefix=True, stop_token_ids=stop))
        for i in range(len(prompts)):
            got = [s[i] for s in again if s[i] is not None]
            assert got == [s[i] for s in steps][:len(got)] and (len(got) == 8 or got[-1] in stop)
        assert engine.cache.live == 0
        engine.cache.check()
    from kernel_rush_kawk_b200.cache.prefix import PrefixGroups  # noqa: F401
    assert any(isinstance(key, tuple) for key in engine.stepper._graphs), "steps of groups were captured"


def test_samples_of_one_prompt(folders):
    """A prompt given several times draws as many samples, each the one that its request would draw alone."""
    engine = engine_of(folders, "tiny_a", dtype="float32")
    prompt = prompts_for("tiny_a", [140], 3)[0]
    want = list(engine.generate([prompt] * 5, 7, temperature=1.0, seed=9))
    assert list(engine.generate([prompt] * 5, 7, temperature=1.0, seed=9, share_prefix=True)) == want
    assert len({tuple(s[i] for s in want) for i in range(5)}) > 1


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("observe", [None, 5])
def test_evicting_float32_steps_agree_with_plain(folders, name, observe):
    from kernel_rush_kawk_b200 import KeyEviction, StepEntry

    engine = engine_of(folders, name, dtype="float32", eviction=KeyEviction(keep=80, recent=20, every=9, observe=observe), max_tokens=64 * 20)
    seqs = prompts_for(name, [240, 100], seed=31)
    plains = [PlainEvicting(folders[name], 80, 20, 9, observe) for _ in seqs]
    slots = [engine.cache.alloc() for _ in seqs]
    done = [0, 0]
    for to in [(150, 4), (151, 70), (215, 71)] + [(215 + i, 71 + i) for i in range(1, 25)] + [(240, 100)]:
        entries, refs = [], []
        for i in (0, 1):
            if to[i] > done[i]:
                entries.append(StepEntry(slots[i], seqs[i][done[i]:to[i]], list(range(to[i] - done[i]))))
                refs.append(plains[i].step(seqs[i][done[i]:to[i]]))
                done[i] = to[i]
        assert_close(engine.step(entries), torch.cat(refs).float(), "float32", f"up to {to}")
        for i in (0, 1):
            n = engine.cache.length[slots[i]]
            for layer in range(plains[i].cfg.layers):
                for h in range(plains[i].cfg.kv_heads):
                    assert sorted(engine.cache.view(layer).positions[slots[i], h, :n].tolist()) == sorted(plains[i].held(layer, h))
    engine.cache.check()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_evicting_generations_are_the_same_run_ahead_or_step_by_step(folders, dtype):
    """The generation loop queues steps and evictions ahead of the host; one step at a time, without captured steps, and the steps that feed
    themselves on the device give the same tokens and leave the same cache."""
    from kernel_rush_kawk_b200 import KeyEviction, StepEntry

    name, eviction = "tiny_a", KeyEviction(keep=70, recent=16, every=7)
    prompts = prompts_for(name, [200, 30, 75], 41)
    engine = engine_of(folders, name, dtype=dtype, eviction=eviction, max_tokens=64 * 40)
    want = list(engine.generate(prompts, 40))
    plainly = engine_of(folders, name, dtype=dtype, eviction=eviction, use_cuda_graphs=False, max_tokens=64 * 40)
    assert list(plainly.generate(prompts, 40)) == want
    slots = [engine.cache.alloc() for _ in prompts]
    first = engine.step([StepEntry(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)]).argmax(dim=-1).tolist()
    assert first == want[0]
    rest = engine.stepper.decode_on_device(slots, first, 39)
    assert rest.tolist() == want[1:]
    for s, p in zip(slots, prompts):
        n = engine.cache.length[s]
        assert n < 77 + 1 and n + engine.cache.evicted[s] == len(p) + 39
        positions = engine.cache.view(1).positions[s, :, :n]
        last = len(p) + 39
        for h in range(positions.shape[0]):
            got = positions[h].tolist()
            assert len(set(got)) == n and set(range(last - 16, last)) <= set(got)
        sums = engine.cache.view(1).scores[s, :, :n]
        assert (sums >= 0).all() and torch.isfinite(sums).all()
        engine.cache.free(s)
    engine.ops.check()
    engine.cache.check()


def test_an_eviction_that_never_comes_changes_no_float32_logits(folders):
    from kernel_rush_kawk_b200 import KeyEviction

    prompts = prompts_for("tiny_b", [100, 7], 9)
    want = list(engine_of(folders, "tiny_b", dtype="float32").generate(prompts, 8))
    assert list(engine_of(folders, "tiny_b", dtype="float32", eviction=KeyEviction(keep=500)).generate(prompts, 8)) == want


def test_forks_of_a_hybrid_decoder():
    """A decoder with recurrent state beside attention over every key: forks take copies of the state, and go on as the whole prompts do."""
    from kernel_rush_kawk_b200 import Engine

    engine = Engine.from_random("zadunex_tiny", dtype="float32", max_slots=6, seed=3, std=0.08)
    g = torch.Generator().manual_seed(1)
    doc = torch.randint(0, engine.config.vocab, (140,), generator=g).tolist()
    prompts = [doc + [i, i + 1] for i in range(3)]
    engine._ensure_cache([len(p) for p in prompts], 6)
    if not engine.cache.can_share():
        pytest.skip("this preset keeps windows")
    want = list(engine.generate(prompts, 6))
    assert list(engine.generate(prompts, 6, share_prefix=True)) == want
