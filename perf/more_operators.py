"""What a server of many fine-tuned variants of one model adds to its steps, case by case.

Three operators: a shared projection with the low-rank adapters of many requests beside it, y = x W^T + s (x A^T) B^T with A, B and s
those of each row's request; the same for the gate and up projections with the activation behind them; and the maps of a step (rows,
positions, page tables, cache places, adapters) made on the device from its requests' lengths. ``run`` computes them from elementary
torch operations, or, where ``own`` is true, by the calls that a program makes of this library. ``exact`` restates the products in 64
bits.

Sizes are the configurations' own: hidden 2,560, 4,096 and 5,120, queries beside keys and values, feed-forwards of 9,728, 12,288 and 17,408,
pages of 64 positions; ranks are those that adapters are trained with.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # one user's next token with a variant of the model: queries, keys and values; the smallest product
        {"name": "linear_token_1", "kind": "linear", "dtype": "bfloat16", "inputs": 2560, "outs": "4096,1024,1024", "batch": 1, "tokens": 1,
         "adapters": 1, "rank": 16, "none": 0},
        # a small server: eight users, five variants, one user of the model as it is; the output projection
        {"name": "linear_tokens_8", "kind": "linear", "dtype": "bfloat16", "inputs": 4096, "outs": "2560", "batch": 8, "tokens": 1,
         "adapters": 5, "rank": 16, "none": 7},
        # a full server whose users all bring a variant of their own
        {"name": "linear_tokens_64", "kind": "linear", "dtype": "bfloat16", "inputs": 2560, "outs": "4096,1024,1024", "batch": 64, "tokens": 1,
         "adapters": 60, "rank": 32, "none": 16},
        # one long prompt of one variant
        {"name": "linear_prompt_1", "kind": "linear", "dtype": "bfloat16", "inputs": 4096, "outs": "4096,1024,1024", "batch": 1, "tokens": 2001,
         "adapters": 1, "rank": 16, "none": 0},
        # unequal prompts of several variants in one step, the second feed-forward product
        {"name": "linear_prompts_9", "kind": "linear", "dtype": "bfloat16", "inputs": 9728, "outs": "2560", "batch": 9, "tokens": 300,
         "adapters": 6, "rank": 64, "none": 4},
        # the 32-bit path
        {"name": "linear_float32_6", "kind": "linear", "dtype": "float32", "inputs": 2560, "outs": "4096,1024,1024", "batch": 6, "tokens": 1,
         "adapters": 4, "rank": 8, "none": 0},
        # the feed-forward's first half at decode
        {"name": "gate_up_tokens_16", "kind": "gate_up", "dtype": "bfloat16", "inputs": 2560, "outs": "9728,9728", "batch": 16, "tokens": 1,
         "adapters": 9, "rank": 16, "none": 0},
        # and over a step full of prompts: the largest
        {"name": "gate_up_prompts_7", "kind": "gate_up", "dtype": "bfloat16", "inputs": 2560, "outs": "9728,9728", "batch": 7, "tokens": 720,
         "adapters": 4, "rank": 32, "none": 6},
        # the next token of 64 sequences, some of which need a new page
        {"name": "maps_tokens_64", "kind": "maps", "batch": 64, "tokens": 1, "low": 30, "high": 4000, "context": 40960, "adapters": 8},
        # sixteen prompts that come in, some 40,000 tokens
        {"name": "maps_prompts_16", "kind": "maps", "batch": 16, "tokens": 3300, "low": 0, "high": 0, "context": 40960, "adapters": 4},
        # a thousand sequences, pieces of prompts behind what they hold already
        {"name": "maps_pieces_1000", "kind": "maps", "batch": 1000, "tokens": 160, "low": 0, "high": 3000, "context": 4096, "adapters": 60},
    ]


SHAPES = [(2560, "4096,1024,1024"), (4096, "2560"), (9728, "2560"), (4096, "4096,1024,1024"), (4096, "4096"), (12288, "4096"),
          (5120, "5120,1024,1024"), (17408, "5120"), (96, "192,64,64"), (1000, "520,136,136"), (333, "77")]
GATES = [(2560, "9728,9728"), (4096, "12288,12288"), (5120, "17408,17408"), (96, "256,256"), (1000, "712,712")]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "gate_up", "gate_up", "maps"])
    if kind == "maps":
        batch = _log_int(rng, 1, 1000)
        tokens = 1 if rng.random() < 0.4 else _log_int(rng, 2, min(4000, 120000 // batch))
        low = rng.choice([0, _log_int(rng, 1, 2000)])
        return {"kind": kind, "batch": batch, "tokens": tokens, "low": low, "high": low + rng.randint(0, 500),
                "context": rng.choice([8192, 16384, 40960]) if batch <= 200 else 8192, "adapters": rng.randint(1, 64)}
    dtype = "float32" if rng.random() < 0.15 else "bfloat16"
    inputs, outs = rng.choice(SHAPES if kind == "linear" else GATES)
    width = sum(int(n) for n in outs.split(","))
    if rng.random() < 0.6:
        batch, tokens = _log_int(rng, 1, 160 if dtype == "bfloat16" else 12), 1
    else:
        batch = rng.randint(1, 12)
        most = min(4000, int(3.5e11 / (2 * inputs * width))) if dtype == "bfloat16" else 40
        tokens = _log_int(rng, 2, max(3, most // batch))
    return {"kind": kind, "dtype": dtype, "inputs": inputs, "outs": outs, "batch": batch, "tokens": tokens, "adapters": rng.randint(1, min(64, batch + 2)),
            "rank": _log_int(rng, 1, 128), "none": rng.choice([0, 0, 2, 5])}


# ---------------------------------------------------------------------------
# what follows from the case alone
# ---------------------------------------------------------------------------

def _outs(case):
    return [int(n) for n in case["outs"].split(",")]


def _lengths(case):
    """New tokens of every sequence: the case's, or from it down to half of it, in no order."""
    n, t = case["batch"], case["tokens"]
    if t == 1:
        return [1] * n
    return [max(1, t - (t * ((5 * i + 2) % n)) // (2 * n)) for i in range(n)]


def _held(case):
    n = case["batch"]
    return [case["low"] + (case["high"] - case["low"]) * ((7 * i + 3) % n) // max(n - 1, 1) for i in range(n)]


def _adapter_of(case):
    """The adapter of every sequence, -1 for none."""
    none = case.get("none", 3)
    return [-1 if none and i % none == none - 1 else (3 * i + 1) % case["adapters"] for i in range(case["batch"])]


def _rank_of(case, adapter, part):
    """Adapters were trained with different ranks, and some leave a projection as it is."""
    if len(_outs(case)) == 3 and part == 1 and adapter % 4 == 2:
        return 0
    return max(1, case["rank"] // 2) if adapter % 3 == 1 else case["rank"]


def work(case):
    lengths = _lengths(case)
    rows = sum(lengths)
    if case["kind"] == "maps":
        need = [(-(-(h + t) // PAGE), -(-h // PAGE)) for h, t in zip(_held(case), lengths)]
        pages = sum(a - b for a, b in need)
        # lengths, slots and adapters in; the first rows out; for every row its sequence, position, adapter and place; the new pages read and
        # written; the page of every row's position read once a page
        touched = sum(a - h // PAGE for (a, _), h in zip(need, _held(case)))
        return {"bytes": case["batch"] * 20 + rows * (4 + 4 + 4 + 8) + pages * 8 + touched * 4, "flops": 0}
    size = 2 if case["dtype"] == "bfloat16" else 4
    K, outs = case["inputs"], _outs(case)
    N = sum(outs)
    width = outs[0] if case["kind"] == "gate_up" else N
    used = sorted({a for a in _adapter_of(case) if a >= 0})
    elements = rows * K + N * K + rows * width
    elements += sum(_rank_of(case, a, p) * (K + n) for a in used for p, n in enumerate(outs))
    flops = 2 * rows * K * N
    flops += sum(2 * t * _rank_of(case, a, p) * (K + n) for a, t in zip(_adapter_of(case), lengths) if a >= 0 for p, n in enumerate(outs))
    return {"bytes": elements * size, "flops": flops}


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------

def _normal(g, shape, dtype, std):
    return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(0.0, std, generator=g).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    lengths = _lengths(case)
    rows = sum(lengths)
    if case["kind"] == "maps":
        host = random.Random(seed)
        n, held = case["batch"], _held(case)
        width = case["context"] // PAGE
        have = [-(-h // PAGE) for h in held]
        need = [-(-(h + t) // PAGE) for h, t in zip(held, lengths)]
        pool = list(range(sum(need)))
        host.shuffle(pool)
        slots = list(range(n))
        host.shuffle(slots)
        table = torch.zeros((n, width), dtype=torch.int32)
        at = 0
        for slot, m in zip(slots, have):
            table[slot, :m] = torch.tensor(pool[at:at + m], dtype=torch.int32)
            at += m
        as_ints = lambda values: torch.tensor(values, dtype=torch.int32, device=DEVICE)
        return dict(case=case, rows=rows, table=table.to(DEVICE), slots=as_ints(slots), held=as_ints(held), lengths=as_ints(lengths),
                    pages=as_ints(pool[at:]), adapter=as_ints(_adapter_of(case)))
    dtype, K, outs = DTYPES[case["dtype"]], case["inputs"], _outs(case)
    x = _normal(g, (rows, K), dtype, 1.0)
    w = _normal(g, (sum(outs), K), dtype, 0.02 if K > 500 else 0.08)
    # the first factor as it is drawn for training, the second of the size that training brings it to
    weights = []
    for a in range(case["adapters"]):
        ranks = [_rank_of(case, a, p) for p in range(len(outs))]
        weights.append(([_normal(g, (r, K), dtype, 1 / math.sqrt(K)) for r in ranks], [_normal(g, (n, r), dtype, 0.02) for r, n in zip(ranks, outs)],
                        [16.0 / r if r else 0.0 for r in ranks]))
    adapter = _adapter_of(case)
    first = [sum(lengths[:i]) for i in range(len(lengths))]
    rows_of = {}  # adapter -> its rows
    for a, at, t in zip(adapter, first, lengths):
        rows_of.setdefault(a, []).extend(range(at, at + t))
    rows_of = {a: torch.tensor(r, device=DEVICE) for a, r in rows_of.items()}
    return dict(case=case, x=x, w=w, outs=outs, weights=weights, rows_of=rows_of)


def prepare(case, seed):
    state = _inputs(case, seed)
    if not own:
        return state
    from kernel_rush_kawk_b200.csrc import load_kernels

    ops = state["ops"] = load_kernels()
    if case["kind"] == "maps":
        return state
    from kernel_rush_kawk_b200.parts.adapters import AdapterBank

    # the adapters in the place that the server keeps them in, and which row of the step is whose
    bank = state["bank"] = AdapterBank(case["inputs"], state["outs"], case["adapters"], case["rank"], DTYPES[case["dtype"]], DEVICE)
    for index, (down, up, scales) in enumerate(state.pop("weights")):
        for part, (a, b, s) in enumerate(zip(down, up, scales)):
            if a.shape[0]:
                bank.put(index, part, a, b, s)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)
    none = torch.zeros_like(lengths)
    adapter = torch.tensor(_adapter_of(case), dtype=torch.int32, device=DEVICE)
    state["adapters"] = ops.step_maps(none, none, lengths, sum(_lengths(case)), adapters=adapter).adapters
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        ops = state["ops"]
        if case["kind"] == "maps":
            maps = ops.step_maps(state["slots"], state["held"], state["lengths"], state["rows"], table=state["table"], pages=state["pages"],
                                 adapters=state["adapter"])
            return maps.cu_q, maps.row_seq, maps.row_pos, maps.row_place, maps.adapters.row_adapter, state["table"]
        if case["kind"] == "gate_up":
            return ops.adapted_gate_up_swiglu(state["x"], state["w"], state["outs"][0], state["bank"], state["adapters"])
        return ops.adapted_linear(state["x"], state["w"], state["bank"], state["adapters"])
    if case["kind"] == "maps":
        return _plain_maps(state)
    y = torch.matmul(state["x"].float(), state["w"].float().t())
    for a, rows in state["rows_of"].items():
        if a < 0:
            continue
        mine, at = state["x"][rows].float(), 0
        down, up, scales = state["weights"][a]
        parts = []
        for A, B, s in zip(down, up, scales):
            parts.append(s * torch.matmul(torch.matmul(mine, A.float().t()), B.float().t()))
        y[rows] += torch.cat(parts, dim=1)
    if case["kind"] == "gate_up":
        gate, up = y.split(state["outs"], dim=1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(state["x"].dtype)


def _plain_maps(state):
    n, rows = state["case"]["batch"], state["rows"]
    held, lengths, slots, table = state["held"], state["lengths"], state["slots"], state["table"]
    cu = torch.zeros(n + 1, dtype=torch.int32, device=held.device)
    cu[1:] = torch.cumsum(lengths, 0)
    row_seq = torch.repeat_interleave(torch.arange(n, dtype=torch.int32, device=held.device), lengths, output_size=rows)
    of = row_seq.long()
    row_pos = torch.arange(rows, dtype=torch.int32, device=held.device) - cu[of] + held[of]
    # the new pages, in the order of the sequences
    have, need = (held + PAGE - 1) // PAGE, (held + lengths + PAGE - 1) // PAGE
    new = need - have
    fresh = state["pages"].shape[0]
    seq = torch.repeat_interleave(torch.arange(n, device=held.device), new, output_size=fresh)
    logical = torch.arange(fresh, device=held.device) - (torch.cumsum(new, 0) - new)[seq] + have[seq]
    table[slots[seq].long(), logical] = state["pages"]
    place = table[slots[of].long(), (row_pos // PAGE).long()].long() * PAGE + row_pos % PAGE
    return cu, row_seq, row_pos, place, state["adapter"][of], table


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "maps":
        return None  # whole numbers
    state = _inputs(case, seed)
    outs, x = state["outs"], state["x"].double()
    out = torch.empty((x.shape[0], sum(outs)), dtype=torch.float64, device=DEVICE)
    base = state["w"].double()
    for a, rows in state["rows_of"].items():
        weight = base.clone()  # the variant's own projection, as if it had been merged
        at = 0
        for part, n in enumerate(outs):
            if a >= 0:
                down, up, scales = state["weights"][a]
                weight[at:at + n] += scales[part] * torch.einsum("nr,rk->nk", up[part].double(), down[part].double())
            at += n
        out[rows] = torch.einsum("mk,nk->mn", x[rows], weight)
    if case["kind"] == "gate_up":
        half = outs[0]
        out = out[:, :half] * torch.sigmoid(out[:, :half]) * out[:, half:]
    return out
