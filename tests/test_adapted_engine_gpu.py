"""Engines with low-rank adapters on the GPU against plain decoders whose weights have the adapters merged in."""

import json

import pytest
import torch

import plain_qwen3 as plain
from adapter_helpers import merged, random_factors, write_adapter
from helpers import assert_close, assert_greedy_token, prompts_for, windows_of

pytestmark = pytest.mark.gpu


def make(folders, name, dtype, **kw):
    from kernel_rush_kawk_b200 import AdapterRoom, Engine

    args = dict(dtype=dtype, max_slots=12, adapters=AdapterRoom(4, 6))
    args.update(kw)
    return Engine(folders[name], **args)


def load(folders, engine, name):
    cfg, w = plain.read_folder(folders[name])
    factors = {"one": random_factors(cfg, w, 1, 4), "two": random_factors(cfg, w, 2, 6, keys=("q_proj", "v_proj", "down_proj")),
               "last": random_factors(cfg, w, 3, 2, layers={cfg.layers - 1})}
    for key, f in factors.items():
        if engine.dtype == torch.bfloat16:  # what the engine holds
            f = factors[key] = {n: (a.bfloat16().float(), b.bfloat16().float(), s) for n, (a, b, s) in f.items()}
        engine.load_adapter(key, f)
    return cfg, w, factors


def logits_of(cfg, w, ids, dtype, name):
    """As the plain implementation has them for the path."""
    if dtype == "float32":
        return plain.forward_logits(cfg, w, ids, torch.float64, None, windows_of(name)).float()
    return plain.forward_logits(cfg, w, ids, torch.float32, torch.bfloat16, windows_of(name)).float()


@pytest.mark.parametrize("name", ["tiny_a", "tiny_b", "tiny_w"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [True, False])
def test_logits(folders, name, dtype, graphs):
    """Prompts in pieces, then single tokens, of sequences with adapters and without, some joining later."""
    from kernel_rush_kawk_b200 import StepEntry

    engine = make(folders, name, dtype, max_tokens=4096, use_cuda_graphs=graphs)
    cfg, w, factors = load(folders, engine, name)
    names = ["one", None, "two", "last", "one"]
    seqs = prompts_for(name, [40, 75, 12, 66, 21], seed=3)
    slots = [engine.cache.alloc(engine.adapters.get(k, -1)) for k in names]
    got = [[] for _ in seqs]
    done = [0] * 5
    for to in [(30, 64, 0, 1, 0), (31, 65, 4, 2, 0), (32, 66, 5, 60, 17)] + [(32 + i, 66 + i, 5 + i, 60 + i, 17 + i) for i in range(1, 5)] + [(40, 75, 12, 66, 21)]:
        entries = [(i, StepEntry(slots[i], seqs[i][done[i]:to[i]], list(range(to[i] - done[i])))) for i in range(5) if to[i] > done[i]]
        out = engine.step([e for _, e in entries]).float().cpu()
        row = 0
        for i, e in entries:
            got[i].append(out[row:row + len(e.tokens)])
            row += len(e.tokens)
            done[i] = to[i]
    for i, k in enumerate(names):
        assert_close(torch.cat(got[i]), logits_of(cfg, merged(w, factors.get(k)), seqs[i], dtype, name), dtype, f"{name} sequence {i} ({k})")
    for s in slots:
        engine.cache.free(s)
    engine.cache.check()


def test_float32_sequences_without_adapters_are_as_ever(folders):
    """To the bit, in the company of others that have some; and an engine without any loaded is one without room."""
    name = "tiny_b"
    prompts = prompts_for(name, [30, 9, 70, 2], seed=5)
    from kernel_rush_kawk_b200 import Engine, StepEntry

    bare, roomy = Engine(folders[name], dtype="float32", max_tokens=2048), make(folders, name, "float32", max_tokens=2048)
    load(folders, roomy, name)

    def run(engine, adapters):
        slots = [engine.cache.alloc(a) for a in adapters]
        outs = [engine.step([StepEntry(s, p, list(range(len(p)))) for s, p in zip(slots, prompts)]).clone()]
        for t in (5, 6):
            outs.append(engine.step([StepEntry(s, [t], [0]) for s in slots]).clone())
        for s in slots:
            engine.cache.free(s)
        return outs

    ref, none, mixed = run(bare, [-1] * 4), run(roomy, [-1] * 4), run(roomy, [0, -1, 1, -1])
    rows = [list(range(30, 39)) + [109, 110], [1, 3], [1, 3]]
    for a, b, c, r in zip(ref, none, mixed, rows):
        assert torch.equal(a, b)
        assert torch.equal(a[r], c[r]) and not torch.equal(a, c)


@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generations(folders, share, dtype):
    name = "tiny_a"
    engine = make(folders, name, dtype)
    cfg, w, factors = load(folders, engine, name)
    doc = prompts_for(name, [130], 7)[0]
    tails = prompts_for(name, [3, 12, 1, 30, 7, 5], 8)
    prompts = [doc + t for t in tails[:4]] + tails[4:]
    for names in (["one", None, "one", "two", "last", None], [None, "two", "two", "two", "one", "one"], [None] * 6):
        steps = list(engine.generate(prompts, 6, adapters=names, share_prefix=share))
        for i, (p, k) in enumerate(zip(prompts, names)):
            seq, mine = list(p), merged(w, factors.get(k))
            for t, step in enumerate(steps):
                assert_greedy_token(cfg, mine, seq, step[i], dtype, windows_of(name), f"request {i} ({k}) step {t}")
                seq.append(step[i])
    assert engine.cache.live == 0
    engine.ops.check()


def test_captured_steps_follow_adapters_that_change(folders):
    """The same captured step of four sequences, with other adapters each time, and another adapter in an old place."""
    name = "tiny_a"
    engine = make(folders, name, "bfloat16")
    cfg, w, factors = load(folders, engine, name)
    prompts = prompts_for(name, [9, 20, 5, 33], seed=11)
    for turn, names in enumerate((["one", "two", None, "last"], ["two", "two", "one", None], ["one", "one", "one", "one"])):
        if turn == 2:
            engine.drop_adapter("one")
            fresh = {n: (a.bfloat16().float(), b.bfloat16().float(), s) for n, (a, b, s) in random_factors(cfg, w, 9, 3, keys=("k_proj", "up_proj")).items()}
            engine.load_adapter("one", fresh)
            factors["one"] = fresh
        steps = list(engine.generate(prompts, 8, adapters=names))
        for i, (p, k) in enumerate(zip(prompts, names)):
            seq, mine = list(p), merged(w, factors.get(k))
            for t, step in enumerate(steps):
                assert_greedy_token(cfg, mine, seq, step[i], "bfloat16", windows_of(name), f"turn {turn} request {i} ({k}) step {t}")
                seq.append(step[i])
    assert sum("adapted" in str(key) for key in engine.stepper._graphs) == 1
    engine.ops.check()


def test_command_line(folders, tmp_path, capsys):
    from kernel_rush_kawk_b200.cli import main

    name = "tiny_a"
    cfg, w = plain.read_folder(folders[name])
    factors = random_factors(cfg, w, 1, 5)
    folder = write_adapter(tmp_path / "a", factors, alpha=4.0)
    scaled = {n: (a, b, 4.0 / a.shape[0]) for n, (a, b, _) in factors.items()}
    prompts = prompts_for(name, [4, 6], seed=12)
    args = ["generate", "--model", str(folders[name]), "--dtype", "float32", "--max-new-tokens", "5", "--adapter", f"mine={folder}", "--use-adapter", "mine",
            "--use-adapter", "-"]
    for p in prompts:
        args += ["--prompt-ids", ",".join(map(str, p))]
    assert main(args) == 0
    lines = [json.loads(line) for line in capsys.readouterr().out.splitlines() if line.startswith("{")]
    for p, line, weights in zip(prompts, lines, (merged(w, scaled), w)):
        assert line["prompt"] == p
        seq = list(p)
        for t, tok in enumerate(line["tokens"]):
            assert_greedy_token(cfg, weights, seq, tok, "float32", windows_of(name), f"step {t}")
            seq.append(tok)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_maps_then_rows_then_both_products(folders, dtype):
    """The operators one after the other, as a program calls them: rows found by their lengths, written into the cache by their places, a feed-forward with adapters."""
    from adapter_helpers import assert_within, gated64, make_adapters, make_bank, per_row, product64
    from kernel_rush_kawk_b200.csrc import load_kernels

    ops, dev = load_kernels(), "cuda:0"
    dt = torch.bfloat16 if dtype == "bfloat16" else torch.float32
    g = torch.Generator().manual_seed(0)
    starts, lengths, of, slots = [60, 0, 5, 128], [70, 3, 1, 64], [1, -1, 0, 1], [2, 0, 3, 1]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    table = torch.zeros((4, 4), dtype=torch.int32, device=dev)
    table[2, 0], table[3, 0], table[1, 0], table[1, 1] = 6, 1, 2, 3
    rows = sum(lengths)
    maps = ops.step_maps(ints(slots), ints(starts), ints(lengths), rows, table=table, pages=ints([4, 5, 0, 7]), adapters=ints(of))
    x = torch.randn((rows, 64), generator=g).to(dev, dt)
    cache = torch.zeros((8 * 64, 64), dtype=dt, device=dev)
    cache[maps.row_place] = x
    at = 0
    for s, start, n in zip(slots, starts, lengths):
        for p in (0, n - 1):
            place = int(table[s, (start + p) // 64]) * 64 + (start + p) % 64
            assert torch.equal(cache[place], x[at + p])
        at += n
    up = make_adapters(g, 2, 64, (128, 128), 8, dt, dev)
    w_up = (torch.randn((256, 64), generator=g) / 8).to(dev, dt)
    act = ops.adapted_gate_up_swiglu(x, w_up, 128, make_bank(up, 64, (128, 128), 8, dt, dev), maps.adapters)
    assert_within(act, *gated64(*product64(x, w_up, up, (128, 128), per_row(lengths, of), True)))
    down = make_adapters(g, 2, 128, (64,), 8, dt, dev)
    w_down = (torch.randn((64, 128), generator=g) / 11).to(dev, dt)
    out = ops.adapted_linear(act, w_down, make_bank(down, 128, (64,), 8, dt, dev), maps.adapters)
    assert_within(out, *product64(act, w_down, down, (64,), per_row(lengths, of), True))
    ops.check()
