"""Shared prefixes and evictions as a server runs them, on the GPU: under the lines that ship, with few captured steps kept, and against the plain
decoders."""

import pytest
import torch

from helpers import assert_close, assert_greedy_token, prompts_for, windows_of
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


@pytest.fixture(scope="module")
def wide_heads(tmp_path_factory):
    """Two layers of 16 heads over 8 of 128 elements: small, but as many bytes a position as a large model's layers have."""
    from kernel_rush_kawk_b200 import Qwen3Config, write_model_folder

    config = Qwen3Config.from_dict({"architectures": ["Qwen3ForCausalLM"], "model_type": "qwen3", "hidden_size": 128, "intermediate_size": 256, "num_hidden_layers": 2,
                                    "num_attention_heads": 16, "num_key_value_heads": 8, "head_dim": 128, "vocab_size": 320, "rms_norm_eps": 1e-6,
                                    "rope_theta": 10000.0, "tie_word_embeddings": True, "max_position_embeddings": 4096})
    return write_model_folder(tmp_path_factory.mktemp("wide") / "wide", config, 5, std=0.04, gain_std=0.1)


def tokens_of(lengths, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 320, (n,), generator=g).tolist() for n in lengths]


@pytest.mark.parametrize("n,length,tail,longer,single", [(24, 1024, 5, True, True), (24, 1024, 200, False, True), (3, 128, 5, False, False)])
def test_generations_under_the_lines_that_ship(wide_heads, monkeypatch, n, length, tail, longer, single):
    """Prompts' ends and single tokens that read what they share once, and those that each read their own table, as the lines have it."""
    from kernel_rush_kawk_b200 import Engine
    from kernel_rush_kawk_b200.cache import prefix
    from kernel_rush_kawk_b200.csrc import cache_ops

    seen = {"longer": [], "single": []}
    for name, where in (("longer_steps_share", "longer"), ("single_tokens_share", "single")):
        line = getattr(prefix, name)
        monkeypatch.setattr(cache_ops, name, lambda *a, line=line, where=where: (seen[where].append(line(*a)), seen[where][-1])[1])
    engine = Engine(wide_heads, dtype="bfloat16", max_slots=32)
    doc = tokens_of([length], 1)[0]
    prompts = [doc + t for t in tokens_of([max(1, tail - i % 3) for i in range(n)], 2)]
    steps = list(engine.generate(prompts, 4, share_prefix=True))
    assert set(seen["longer"]) == {longer}, "the prompts' ends"
    assert set(seen["single"]) == ({True} if single else set()), "(where it does not pay the step is one like any other)"
    assert any(isinstance(key, tuple) for key in engine.stepper._graphs) == single
    cfg, w = plain.read_folder(wide_heads)
    for i in {0, n // 2, n - 1}:
        seq = list(prompts[i])
        for t, step in enumerate(steps):
            assert_greedy_token(cfg, w, seq, step[i], "bfloat16", None, f"request {i} step {t}")
            seq.append(step[i])
    engine.ops.check()


class PlainKept:
    """A plain Qwen3 decoder with bfloat16's rounding points whose heads keep the rows that it is told to (their positions), and count the weight
    that each has received."""

    def __init__(self, folder, observe):
        self.cfg, self.w = plain.read_folder(folder)
        self.observe, self.at = observe, 0
        empty = lambda: [[torch.empty((0, self.cfg.head_dim))] * 2 + [torch.empty(0), []] for _ in range(self.cfg.kv_heads)]
        self.rows = [empty() for _ in range(self.cfg.layers)]

    def keep(self, positions) -> None:
        """positions[layer][head]: those that stay."""
        for layer, heads in zip(self.rows, positions):
            for row, stay in zip(layer, heads):
                at = [row[3].index(p) for p in stay]
                row[0], row[1], row[2], row[3] = row[0][at], row[1][at], row[2][at], list(stay)

    def step(self, ids) -> torch.Tensor:
        cfg, w, r, D = self.cfg, self.w, torch.bfloat16, self.cfg.head_dim
        rt = lambda x: x.to(r).float()
        t, per = len(ids), cfg.heads // cfg.kv_heads
        cos, sin = plain.rope_tables(D, cfg.rope_theta, self.at + t, torch.float32, r)
        cos, sin = cos[self.at:], sin[self.at:]
        x = w["model.embed_tokens.weight"][torch.as_tensor(ids)]
        for i in range(cfg.layers):
            p = f"model.layers.{i}."
            h = plain.rms_norm(x, w[p + "input_layernorm.weight"], cfg.eps, r)
            q, k, v = (plain.linear(h, w[p + f"self_attn.{n}_proj.weight"], r).view(t, -1, D) for n in "qkv")
            q = plain.head_norm_rope(q, w[p + "self_attn.q_norm.weight"], cos, sin, cfg.eps, r)
            k = plain.head_norm_rope(k, w[p + "self_attn.k_norm.weight"], cos, sin, cfg.eps, r)
            a = torch.empty((t, cfg.heads, D))
            for g, row in enumerate(self.rows[i]):
                old = len(row[3])
                row[0], row[1] = torch.cat([row[0], k[:, g]]), torch.cat([row[1], v[:, g]])
                row[2], row[3] = torch.cat([row[2], torch.zeros(t)]), row[3] + list(range(self.at, self.at + t))
                seen = torch.arange(old + t)[None, :] < old + 1 + torch.arange(t)[:, None]
                for hh in range(g * per, (g + 1) * per):
                    s = (q[:, hh] @ row[0].t() / D ** 0.5).masked_fill(~seen, float("-inf"))
                    e = torch.exp(s - s.amax(dim=-1, keepdim=True))
                    total = e.sum(dim=-1, keepdim=True)
                    a[:, hh] = rt((rt(e) @ row[1]) / total)
                    row[2] += (e / total)[t - min(t, self.observe or t):].sum(dim=0)
            x = plain.residual_add(x, plain.linear(a.reshape(t, -1), w[p + "self_attn.o_proj.weight"], r), r)
            h = plain.rms_norm(x, w[p + "post_attention_layernorm.weight"], cfg.eps, r)
            x = plain.residual_add(x, plain.swiglu_mlp(h, w[p + "mlp.gate_proj.weight"], w[p + "mlp.up_proj.weight"], w[p + "mlp.down_proj.weight"], r), r)
        self.at += t
        head = w["model.embed_tokens.weight"] if cfg.tie else w["lm_head.weight"]
        return plain.rms_norm(x, w["model.norm.weight"], cfg.eps, r) @ head.t()


@pytest.mark.parametrize("name", ["tiny_a", "tiny_b"])
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("observe", [None, 5])
def test_evicting_bfloat16_steps_agree_with_plain(folders, name, graphs, observe):
    """Step by step, prompts in pieces and single tokens: which rows stay is the definition's by the engine's own sums, to the row; sums and logits are a plain decoder's that
    keeps the same rows, within what whole models of bfloat16 are held to."""
    from cache_ops_helpers import exact_evict
    from kernel_rush_kawk_b200 import KeyEviction, StepEntry

    keep, recent, every = 80, 20, 9
    engine = engine_of(folders, name, use_cuda_graphs=graphs, eviction=KeyEviction(keep=keep, recent=recent, every=every, observe=observe), max_tokens=64 * 20)
    cache, group = engine.cache, engine.cache._kv_groups[0]
    seqs = prompts_for(name, [240, 100], seed=31)
    plains = [PlainKept(folders[name], observe) for _ in seqs]
    slots = [cache.alloc() for _ in seqs]
    done, evictions = [0, 0], 0
    for to in [(150, 4), (151, 70), (215, 71)] + [(215 + i, 71 + i) for i in range(1, 25)] + [(240, 100)]:
        chosen = [i for i in (0, 1) if to[i] > done[i]]
        lengths = [cache.length[s] for s in slots]
        due = [n if n >= keep + every else min(n, keep) for n in lengths]
        _, _, _, positions = exact_evict(group.k, group.v, group.table, slots, due, group.scores, group.positions, keep, recent)
        entries, refs = [], []
        for i in chosen:
            left = keep if lengths[i] >= keep + every else lengths[i]
            plains[i].keep([[positions[line, slots[i], h, :left].tolist() for h in range(plains[i].cfg.kv_heads)] for line in range(plains[i].cfg.layers)])
            evictions += left < lengths[i]
            entries.append(StepEntry(slots[i], seqs[i][done[i]:to[i]], list(range(to[i] - done[i]))))
            refs.append(plains[i].step(seqs[i][done[i]:to[i]]))
            done[i] = to[i]
        assert_close(engine.step(entries), torch.cat(refs), "bfloat16", f"up to {to}")
        for i in chosen:
            n = cache.length[slots[i]]
            for line in range(plains[i].cfg.layers):
                view = cache.view(line)
                for h, row in enumerate(plains[i].rows[line]):
                    assert view.positions[slots[i], h, :n].tolist() == row[3], "the rows, in their places"
                    assert_close(view.scores[slots[i], h, :n][None], row[2][None], "bfloat16", f"sums, layer {line}, head {h}, up to {to}")
    assert evictions > 4
    engine.ops.check()
    cache.check()
