"""Engines with low-rank adapters on the CPU, with a stand-in for the kernels: which sequence runs with which adapter, what shares pages, what is refused, and
adapters read from files."""

import json
from dataclasses import replace

import pytest
import torch

import plain_qwen3 as plain
from adapter_helpers import maps_by_hand, merged, random_factors, write_adapter
from cache_engine_helpers import CacheTorchOps
from helpers import prompts_for
from kernel_rush_kawk_b200 import AdapterError, AdapterRoom, Engine, KeyEviction, StepEntry
from kernel_rush_kawk_b200.csrc.adapter_ops import StepMaps
from kernel_rush_kawk_b200.engine.generate import shared_pages, shared_prefixes
from kernel_rush_kawk_b200.engine.model import Model, PartTree
from kernel_rush_kawk_b200.weights.adapters import read_adapter


class AdapterTorchOps(CacheTorchOps):
    """The stand-in with maps and adapted products."""

    def __init__(self, dtype=torch.float32):
        super().__init__(dtype)
        self.calls.update(maps=0, pages=0, adapted=0)

    def step_maps(self, slots, starts, lengths, n_rows, table=None, pages=None, adapters=None, out=None):
        self.calls["maps"] += 1
        assert int(lengths.sum()) == n_rows
        out = out or StepMaps(n_rows, lengths.shape[0], "cpu", table is not None, adapters is not None)
        rows = None if table is None else table.tolist()
        if table is not None:
            need = sum(-(-(s + n) // 64) - -(-s // 64) for s, n in zip(starts.tolist(), lengths.tolist()))
            assert pages.shape[0] == need, "the pages are the ones that the lengths ask for"
            self.calls["pages"] += need
        cu, seq, pos, place, of = maps_by_hand(slots.tolist(), starts.tolist(), lengths.tolist(), rows, None if pages is None else pages.tolist(),
                                               None if adapters is None else adapters.tolist())
        for to, values in ((out.cu_q, cu), (out.row_seq, seq), (out.row_pos, pos)):
            to.copy_(torch.tensor(values, dtype=torch.int32))
        if table is not None:
            table.copy_(torch.tensor(rows, dtype=torch.int32))
            out.row_place.copy_(torch.tensor(place, dtype=torch.int64))
        if adapters is not None:
            out.adapters.row_adapter.copy_(torch.tensor(of, dtype=torch.int32))
        return out

    def adapted_linear(self, x, w, bank, rows):
        self.calls["adapted"] += 1
        x = self._resolve(x)
        y = self.linear(x, w, out_float32=True)
        for r, a in enumerate(rows.row_adapter.tolist()):
            for p in range(bank.parts) if a >= 0 else ():
                n = int(bank.ranks[a, p])
                A, B = bank.a[a, p * bank.rank:p * bank.rank + n].float(), bank.b[a, bank.begin[p]:bank.begin[p + 1], :n].float()
                y[r, bank.begin[p]:bank.begin[p + 1]] += bank.scale[a, p] * (x[r].float() @ A.T @ B.T)
        return y.to(self.dtype)

    def adapted_gate_up_swiglu(self, x, w_gate_up, intermediate, bank, rows):
        y = self.adapted_linear(x, w_gate_up, bank, rows).float()
        return (torch.nn.functional.silu(y[:, :intermediate]) * y[:, intermediate:]).to(self.dtype)


NAME = "tiny_a"


def make(folders, ops=None, name=NAME, **kw):
    args = dict(dtype="float32", max_slots=8, device="cpu", ops=ops or AdapterTorchOps(), use_cuda_graphs=False, adapters=AdapterRoom(3, 6))
    args.update(kw)
    return Engine(folders[name], **args)


def plain_of(folders, name=NAME):
    return plain.read_folder(folders[name])


def greedy(cfg, w, prompt, n):
    seq = list(prompt)
    for _ in range(n):
        seq.append(int(plain.forward_logits(cfg, w, seq, torch.float64)[-1].argmax()))
    return seq[len(prompt):]


def loaded(folders, engine, name=NAME):
    cfg, w = plain_of(folders, name)
    factors = {"one": random_factors(cfg, w, 1, 4), "two": random_factors(cfg, w, 2, 6, keys=("q_proj", "v_proj", "down_proj")),
               "last": random_factors(cfg, w, 3, 2, layers={cfg.layers - 1})}
    for key, f in factors.items():
        engine.load_adapter(key, f)
    return cfg, w, factors


@pytest.mark.parametrize("name", ["tiny_a", "tiny_b"])
def test_every_prompt_runs_with_its_adapter(folders, name):
    ops = AdapterTorchOps()
    engine = make(folders, ops, name)
    cfg, w, factors = loaded(folders, engine, name)
    prompts = prompts_for(name, [5, 70, 3, 9, 64], seed=1)
    names = ["one", None, "two", "last", "one"]
    outs = engine.generate_all(prompts, 4, adapters=names)
    assert ops.calls["adapted"] > 0 and ops.calls["maps"] > 0 and ops.calls["pages"] > 0
    for p, key, out in zip(prompts, names, outs):
        assert out == greedy(cfg, merged(w, factors.get(key)), p, 4), key
    assert len({tuple(engine.generate_all([prompts[0]], 6, adapters=k)[0]) for k in (None, "one", "two", "last")}) > 1, "adapters change what is said"
    before = ops.calls["adapted"]
    assert engine.generate_all(prompts, 3) == [greedy(cfg, w, p, 3) for p in prompts]
    assert engine.generate_all(prompts, 3, adapters=[None] * 5) == [greedy(cfg, w, p, 3) for p in prompts]
    assert ops.calls["adapted"] == before, "steps without any adapter run as in an engine without room"
    assert set(engine.cache.adapter) == {-1}


def test_batches_keep_their_prompts_adapters(folders):
    engine = make(folders)
    cfg, w, factors = loaded(folders, engine)
    prompts = prompts_for(NAME, [4, 6, 8, 3, 5], seed=2)
    names = ["two", "one", None, "one", "last"]
    assert engine.generate_all(prompts, 3, adapters=names, max_batch=2) == [greedy(cfg, merged(w, factors.get(k)), p, 3) for p, k in zip(prompts, names)]


def test_what_begins_alike_is_shared_by_one_adapter_alone(folders):
    doc = prompts_for(NAME, [130], 3)[0]
    prompts = [doc + t for t in prompts_for(NAME, [3, 5, 2, 4], 4)]
    assert shared_prefixes(prompts, [0, -1, 0, -1]) == [([1, 3], 128), ([0, 2], 128)] or shared_prefixes(prompts, [0, -1, 0, -1]) == [([3, 1], 128), ([2, 0], 128)] \
        or {frozenset(m) for m, s in shared_prefixes(prompts, [0, -1, 0, -1]) if s == 128} == {frozenset((1, 3)), frozenset((0, 2))}
    assert all(s == 0 for _, s in shared_prefixes(prompts, [0, 1, 2, -1]))
    assert shared_prefixes(prompts) == shared_prefixes(prompts, [2] * 4)
    assert shared_pages(prompts, 1, [0, -1, 0, -1]) == shared_pages(prompts, 1) + 2
    engine = make(folders)
    cfg, w, factors = loaded(folders, engine)
    names = ["one", None, "one", "two"]
    outs = engine.generate_all(prompts, 3, adapters=names, share_prefix=True)
    assert outs == [greedy(cfg, merged(w, factors.get(k)), p, 3) for p, k in zip(prompts, names)]
    assert engine.last_stats.shared_tokens == 128


def test_adapters_come_and_go(folders):
    engine = make(folders, adapters=AdapterRoom(2, 6))
    cfg, w = plain_of(folders)
    prompt = prompts_for(NAME, [7], 5)[0]
    sets = [random_factors(cfg, w, s, 5, keys=keys) for s, keys in ((1, ("q_proj", "o_proj")), (2, ("up_proj",)), (3, ("gate_proj", "down_proj", "k_proj")))]
    engine.load_adapter("a", sets[0])
    engine.load_adapter("b", sets[1])
    with pytest.raises(AdapterError, match="no room"):
        engine.load_adapter("c", sets[2])
    engine.drop_adapter("a")
    engine.load_adapter("c", sets[2])
    engine.load_adapter("b", sets[0], scale=0.5)  # another in its place, with another scale
    half = {k: (a, b, 0.5) for k, (a, b, _) in sets[0].items()}
    for key, f in (("c", sets[2]), ("b", half)):
        assert engine.generate_all([prompt], 4, adapters=key) == [greedy(cfg, merged(w, f), prompt, 4)], key
    with pytest.raises(AdapterError, match="no adapter 'a'"):
        engine.generate_all([prompt], 4, adapters="a")
    with pytest.raises(AdapterError):
        engine.drop_adapter("a")
    running = engine.generate([prompt], 5, adapters=["b"])
    next(running)
    for call in (lambda: engine.load_adapter("b", sets[1]), lambda: engine.drop_adapter("b")):
        with pytest.raises(AdapterError, match="in use"):
            call()
    engine.drop_adapter("c")
    running.close()
    engine.drop_adapter("b")
    assert engine.adapters == {}


def test_forks_go_on_with_their_adapter(folders):
    engine = make(folders, max_tokens=64 * 12)
    cfg, w, factors = loaded(folders, engine)
    cache = engine.cache
    doc, tail = prompts_for(NAME, [64, 5], 6)
    slot = cache.alloc(engine.adapters["two"])
    engine.step([StepEntry(slot, doc, [])])
    fork = cache.fork(slot, 64)
    logits = engine.step([StepEntry(fork, tail, [4])])
    ref = plain.forward_logits(cfg, merged(w, factors["two"]), doc + tail, torch.float64)[-1]
    assert torch.allclose(logits[0].double(), ref, atol=1e-4)
    cache.free(slot)
    cache.free(fork)
    assert cache.adapter[slot] == cache.adapter[fork] == -1
    cache.check()


def test_with_eviction(folders):
    """Rows that lie elsewhere than their positions: maps and adapters go by what is held."""
    engine = make(folders, eviction=KeyEviction(keep=100, recent=50, every=20))
    cfg, w, factors = loaded(folders, engine)
    prompt = prompts_for(NAME, [90], 7)[0]
    assert engine.generate_all([prompt, prompt], 5, adapters=["one", None]) == [greedy(cfg, merged(w, factors["one"]), prompt, 5), greedy(cfg, w, prompt, 5)]


def test_pages_entered_from_lengths_are_the_ledgers(folders):
    ops = AdapterTorchOps()
    engine = make(folders, ops, max_tokens=64 * 30, adapters=None)
    cache, group = engine.cache, engine.cache._kv_groups[0]
    slots = [cache.alloc() for _ in range(3)]
    toks = prompts_for(NAME, [200, 70, 129], 8)
    done = [0, 0, 0]
    for pieces in ((63, 1, 64), (2, 60, 65), (100, 9, 0), (35, 0, 0)):
        engine.step([StepEntry(s, t[d:d + n], []) for s, t, d, n in zip(slots, toks, done, pieces) if n])
        done = [d + n for d, n in zip(done, pieces)]
        for s in slots:
            pages = group.ledger.pages[s]
            assert group.table[s, :len(pages)].tolist() == pages == group.table_host[s, :len(pages)].tolist()
        assert not group.dirty
    cache.reserve(slots[1], 200)  # ahead of its tokens, as queued single-token steps do
    engine.step([StepEntry(slots[1], [3, 4], []), StepEntry(slots[2], [5], [])])
    for s in slots:
        pages = group.ledger.pages[s]
        assert group.table[s, :len(pages)].tolist() == pages
    assert ops.calls["maps"] == 5 and ops.calls["pages"] > 0 and not group.dirty


def test_refusals(folders):
    cfg, w = plain_of(folders)
    factors = random_factors(cfg, w, 1, 4)
    engine = make(folders)
    name = next(iter(factors))
    a, b, s = factors[name]
    for bad in ({}, {"model.norm.weight": (a, b, s)}, {name: (a[:, :-1], b, s)}, {name: (a, b[:-1], s)}, {name: (a[:0], b[:, :0], s)},
                {name: (torch.randn(7, a.shape[1]), torch.randn(b.shape[0], 7), s)}, {name: (a[0], b, s)}):
        with pytest.raises(AdapterError):
            engine.load_adapter("x", bad)
    assert engine.adapters == {} and not any(bank.ranks.any() for bank, _ in engine._beside.values())
    with pytest.raises(AdapterError):
        make(folders, adapters=None).load_adapter("x", factors)
    for room in ((0, 4), (1, 0), (1, 300)):
        with pytest.raises(AdapterError):
            AdapterRoom(*room)
    engine.load_adapter("x", factors)
    said = engine.generate_all([[1, 2, 3]], 3, adapters="x")
    last = list(factors)[-1]
    broken = dict(factors) | {last: (factors[last][0], torch.full_like(factors[last][1], float("nan")), 1.0)}
    with pytest.raises(AdapterError, match="finite"):
        engine.load_adapter("x", broken)  # and what the name had before is all there
    assert engine.generate_all([[1, 2, 3]], 3, adapters="x") == said
    with pytest.raises(AdapterError, match="2 adapters for 1"):
        engine.generate_all([[1, 2]], 2, adapters=["x", None])
    with pytest.raises(AdapterError):
        list(engine.generate([[1, 2]], 2, adapters=["y"]))


def test_models_whose_layers_take_none(tmp_path):
    from kernel_rush_kawk_b200 import write_model_folder
    from kernel_rush_kawk_b200.config.registry import preset_config

    folder = write_model_folder(tmp_path / "m", preset_config("taredra_tiny"), seed=1)
    with pytest.raises(ValueError, match="cannot stand beside"):
        Engine(folder, dtype="float32", device="cpu", ops=AdapterTorchOps(), adapters=AdapterRoom(1, 4))


def test_adapters_from_files(folders, tmp_path):
    cfg, w = plain_of(folders)
    factors = random_factors(cfg, w, 4, 5)
    folder = write_adapter(tmp_path / "a", factors, alpha=3.0)
    got = read_adapter(folder)
    assert set(got) == set(factors)
    for name, (a, b, s) in got.items():
        assert torch.equal(a, factors[name][0]) and torch.equal(b, factors[name][1]) and s == 3.0 / a.shape[0]
    assert read_adapter(write_adapter(tmp_path / "b", factors, 3.0, prefix="", use_rslora=True))[name][2] == 3.0 / a.shape[0] ** 0.5
    engine = make(folders)
    engine.load_adapter("file", folder)
    prompt = prompts_for(NAME, [6], 9)[0]
    assert engine.generate_all([prompt], 3, adapters="file") == [greedy(cfg, merged(w, got), prompt, 3)]
    for i, config in enumerate((dict(bias="all"), dict(use_dora=True), dict(alpha_pattern={"q_proj": 4}), dict(modules_to_save=["lm_head"]))):
        with pytest.raises(AdapterError):
            read_adapter(write_adapter(tmp_path / f"c{i}", factors, **config))
    (folder / "adapter_config.json").write_text(json.dumps({"r": 4}))
    with pytest.raises(AdapterError, match="lora_alpha"):
        read_adapter(folder)
    (folder / "adapter_config.json").write_text("{")
    with pytest.raises(AdapterError):
        read_adapter(folder)
    with pytest.raises(AdapterError):
        read_adapter(tmp_path / "nowhere")
    empty = tmp_path / "empty"
    empty.mkdir()
    (empty / "adapter_config.json").write_text(json.dumps({"lora_alpha": 4}))
    with pytest.raises(AdapterError, match="no .*safetensors"):
        read_adapter(empty)
    from safetensors.torch import save_file
    module = next(iter(factors)).removesuffix(".weight")
    for tensors in ({module + ".lora_A.weight": factors[name][0]}, {module + ".lora_magnitude_vector": torch.ones(3)}, {"x": torch.ones(2)},
                    {module + ".lora_A.weight": torch.ones(3, 4), module + ".lora_B.weight": torch.ones(4, 2)}):
        save_file(tensors, str(empty / "t.safetensors"))
        with pytest.raises(AdapterError):
            read_adapter(empty)
    (empty / "t.safetensors").write_bytes(b"12345678")
    with pytest.raises(AdapterError, match="cannot be read"):
        read_adapter(empty)


def test_command_line(folders, tmp_path, capsys):
    from kernel_rush_kawk_b200.cli import main

    cfg, w = plain_of(folders)
    folder = write_adapter(tmp_path / "a", random_factors(cfg, w, 4, 5))
    base = ["generate", "--model", str(folders[NAME]), "--prompt-ids", "1,2"]
    for more in (["--use-adapter", "x"], ["--adapter", "x=/nowhere"], ["--adapter", f"x={folder}", "--use-adapter", "y"],
                 ["--adapter", f"x={folder}", "--use-adapter", "x", "--use-adapter", "x"]):
        with pytest.raises(SystemExit):
            main(base + more)
    capsys.readouterr()


def test_a_weight_of_two_layers_takes_none(folders):
    """Two layers that have one checkpoint tensor between them: an adapter would have to stand beside both."""
    engine = make(folders)
    plan = engine.plan
    layers = list(plan.layers)
    layers[1] = replace(layers[1], feed_forward=replace(layers[1].feed_forward, tensors=layers[0].feed_forward.tensors))
    plan = replace(plan, layers=tuple(layers))
    tensors = {name: torch.zeros(spec.shape) for name, spec in PartTree(plan).expected_tensors().items()}
    where = Model(plan, engine.model.runtime, tensors).open_adapters(AdapterRoom(1, 4))
    gone = set(engine._beside) - set(where)
    assert gone == set(layers[0].feed_forward.tensors.values()) | set(engine.plan.layers[1].feed_forward.tensors.values()) and where


def test_passes_of_more_sequences_than_the_maps_take(folders):
    """Their rows are described by the host, as where there are no such maps."""
    ops = AdapterTorchOps()
    engine = make(folders, ops=ops)
    prompts = prompts_for(NAME, [9, 70, 4], 8)
    expected = engine.generate_all(prompts, 3)
    made = ops.calls["maps"]
    assert made > 0
    ops.MOST_SEQUENCES = 2
    assert engine.generate_all(prompts, 3) == expected and ops.calls["maps"] == made
