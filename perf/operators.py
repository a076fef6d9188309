"""The cache's operators that serving long and shared contexts lives by, case by case.

Three of them: attention for sequences that share a prefix (its keys and values read once for all of them), attention that adds up
the weight which each cached key receives, and the eviction of the keys that received least. ``run`` computes them from
elementary torch operations, or, where ``own`` is true, by the calls that a program makes of this library. ``exact`` restates
them in 64 bits.

Head counts and sizes are the configurations' own (32 or 40 query heads over 8, 12 or 16 over 4, of 128 or 64 elements), pages have 64
positions and lie anywhere in the pool.
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
        # eight chats behind one system prompt, the next token of each: where latency counts
        {"name": "prefix_chat_8", "kind": "prefix", "dtype": "bfloat16", "heads": 32, "kv": 8, "dim": 128, "groups": 1, "batch": 8,
         "prefix": 1024, "low": 40, "high": 400, "tokens": 1},
        # a full server whose requests all carry the same long document, one token each: the largest
        {"name": "prefix_server_64", "kind": "prefix", "dtype": "bfloat16", "heads": 32, "kv": 8, "dim": 128, "groups": 1, "batch": 64,
         "prefix": 8192, "low": 30, "high": 500, "tokens": 1},
        # several answers drawn for each of four prompts of unequal lengths
        {"name": "prefix_samples_4x9", "kind": "prefix", "dtype": "bfloat16", "heads": 40, "kv": 8, "dim": 128, "groups": 4, "batch": 36,
         "prefix": 2112, "low": 1, "high": 300, "tokens": 1},
        # the questions themselves: sixteen ragged prompts behind one document, in one step
        {"name": "prefix_questions_16", "kind": "prefix", "dtype": "bfloat16", "heads": 32, "kv": 8, "dim": 128, "groups": 1, "batch": 16,
         "prefix": 4096, "low": 0, "high": 0, "tokens": 90},
        # the 32-bit path
        {"name": "prefix_float32_6", "kind": "prefix", "dtype": "float32", "heads": 16, "kv": 4, "dim": 64, "groups": 1, "batch": 6,
         "prefix": 960, "low": 5, "high": 150, "tokens": 1},
        # one user's next token while the cache keeps count: the smallest call
        {"name": "scored_token_1", "kind": "scored", "dtype": "bfloat16", "heads": 32, "kv": 8, "dim": 128, "batch": 1, "tokens": 1,
         "low": 1087, "high": 1087, "observe": 0},
        # a server whose sequences hold some thousands of keys each
        {"name": "scored_tokens_32", "kind": "scored", "dtype": "bfloat16", "heads": 32, "kv": 8, "dim": 128, "batch": 32, "tokens": 1,
         "low": 2000, "high": 4500, "observe": 0},
        # a long prompt of which the last 64 queries decide what is kept
        {"name": "scored_prompt_last_64", "kind": "scored", "dtype": "bfloat16", "heads": 32, "kv": 8, "dim": 128, "batch": 1, "tokens": 4001,
         "low": 0, "high": 0, "observe": 64},
        # three unequal prompts, every query counted
        {"name": "scored_prompts_3", "kind": "scored", "dtype": "bfloat16", "heads": 12, "kv": 4, "dim": 128, "batch": 3, "tokens": 1500,
         "low": 0, "high": 0, "observe": 0},
        # the 32-bit path
        {"name": "scored_float32_3", "kind": "scored", "dtype": "float32", "heads": 16, "kv": 4, "dim": 64, "batch": 3, "tokens": 1,
         "low": 300, "high": 700, "observe": 0},
        # every 64 tokens of a running server: 64 keys of each head go, in eight layers at once
        {"name": "evict_steady_16", "kind": "evict", "dtype": "bfloat16", "kv": 8, "dim": 128, "batch": 16, "layers": 8, "rows": 1088,
         "keep": 1024, "recent": 128, "fresh": 64},
        # after a long prompt: one key in eight stays
        {"name": "evict_prompt_1", "kind": "evict", "dtype": "bfloat16", "kv": 8, "dim": 128, "batch": 1, "layers": 8, "rows": 16300,
         "keep": 2048, "recent": 256, "fresh": 16300},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["prefix", "prefix", "prefix", "scored", "scored", "evict"])
    heads, kv, dim = rng.choice([(32, 8, 128), (32, 8, 128), (40, 8, 128), (12, 4, 128), (16, 4, 64), (8, 8, 64)])
    dtype = "float32" if rng.random() < 0.15 else "bfloat16"
    if kind == "prefix":
        one = rng.random() < 0.65
        batch = _log_int(rng, 1, 64 if one else 16)
        if dtype == "float32":
            batch = min(batch, 8)
        low = _log_int(rng, 1, 400) if one else 0
        return {"kind": "prefix", "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "groups": rng.randint(1, min(4, batch)), "batch": batch,
                "prefix": PAGE * _log_int(rng, 1, 128 if dtype == "bfloat16" else 32), "low": low, "high": low + (rng.randint(0, 100) if one else 0),
                "tokens": 1 if one else _log_int(rng, 2, 1440 // batch)}
    if kind == "scored":
        one = rng.random() < 0.6
        if dtype == "float32":
            heads, kv, dim = 16, 4, 64
        batch = _log_int(rng, 1, 32 if dtype == "bfloat16" else 8) if one else rng.randint(1, 3)
        low = _log_int(rng, 1, 4000 if dtype == "bfloat16" else 900) if one else rng.choice([0, 0, rng.randint(1, 700)])
        return {"kind": "scored", "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "batch": batch,
                "tokens": 1 if one else _log_int(rng, 2, (4000 if dtype == "bfloat16" else 600) // batch),
                "low": low, "high": low + (rng.randint(0, 500) if one else 0), "observe": rng.choice([0, rng.randint(1, 100)])}
    keep = _log_int(rng, 16, 2048)
    rows = keep + _log_int(rng, 1, 14000)
    return {"kind": "evict", "dtype": dtype, "kv": kv, "dim": dim, "batch": _log_int(rng, 1, max(1, min(16, 17000 // rows))), "layers": rng.randint(1, 8),
            "rows": rows, "keep": keep, "recent": rng.randint(0, keep), "fresh": rng.choice([rows, rows - keep])}


# ---------------------------------------------------------------------------
# lengths, which follow from the case alone
# ---------------------------------------------------------------------------

def _spread(low, high, n):
    """n numbers from low to high, in no order."""
    return [low + (high - low) * ((7 * i + 3) % n) // max(n - 1, 1) for i in range(n)]


def _sequences(case):
    """Per sequence: rows held before the step, tokens brought; for a shared prefix also the groups' sizes and lengths."""
    n, t = case["batch"], case["tokens"]
    brings = [1] * n if t == 1 else [max(1, t - (t * i) // (2 * n)) for i in range(n)]
    held = _spread(case["low"], case["high"], n)
    if case["kind"] == "scored":
        return held, brings, None, None
    g = case["groups"]
    sizes = [n // g + (1 if i < n % g else 0) for i in range(g)]
    lengths = [max(PAGE, case["prefix"] - PAGE * (i % 3)) for i in range(g)]
    held = [h + p for h, p in zip(held, [p for s, p in zip(sizes, lengths) for _ in range(s)])]
    return held, brings, sizes, lengths


def _evict_rows(case):
    """Rows held per sequence: all of the case's, a few less for every other one."""
    return [case["rows"] - (min(5, case["rows"] - case["keep"]) if i % 2 else 0) for i in range(case["batch"])]


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    kv, dim = case["kv"], case["dim"]
    if case["kind"] == "evict":
        moved = rows = 0.0
        for length in _evict_rows(case):
            beyond = length - case["keep"]
            last = min(case["recent"], beyond)  # of the newest keys, those beyond the rows that stay
            rest = beyond - last
            moved += last + (rest * (case["keep"] - case["recent"]) / (length - case["recent"]) if rest else 0.0)
            rows += length
        heads = kv * case["layers"]
        # scores and positions read and the kept ones written; keys and values of the moved rows read and written
        return {"bytes": int(heads * (rows * 8 + case["batch"] * case["keep"] * 8 + moved * 2 * 2 * dim * size)), "flops": 0}
    held, brings, sizes, lengths = _sequences(case)
    heads = case["heads"]
    pairs = sum(t * h + t * (t + 1) // 2 for h, t in zip(held, brings))  # (query, key)
    if case["kind"] == "prefix":
        keys = sum(lengths) + sum(h + t for h, t in zip(held, brings)) - sum(s * p for s, p in zip(sizes, lengths))
        table = 0
        flops = 4 * dim * heads * pairs
    else:
        keys = sum(h + t for h, t in zip(held, brings))
        table = kv * (8 * keys)  # the sums read and written
        flops = 4 * dim * heads * pairs
        if case["tokens"] > 1:  # the statistics come first: the observed queries' scores are computed once more
            seen = [min(t, case["observe"] or t) for t in brings]
            flops += 2 * dim * heads * sum(o * (h + t) - o * (o - 1) // 2 for h, t, o in zip(held, brings, seen))
    return {"bytes": int(keys * kv * dim * 2 * size + sum(brings) * heads * dim * 2 * size + table), "flops": int(flops)}


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------

def _normal(g, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(0.0, std, generator=g).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(DEVICE).manual_seed(seed)
    host = random.Random(seed)
    dtype = DTYPES[case["dtype"]]
    kv, dim, n = case["kv"], case["dim"], case["batch"]
    if case["kind"] == "evict":
        rows, layers = _evict_rows(case), case["layers"]
        width = -(-case["rows"] // PAGE)
        pages = list(range(n * width))
        host.shuffle(pages)
        table = torch.tensor(pages, dtype=torch.int32, device=DEVICE).view(n, width)
        k = _normal(g, (layers, n * width, kv, PAGE, dim), dtype)
        v = _normal(g, (layers, n * width, kv, PAGE, dim), dtype)
        # a few keys take most of the weight; what little the others received is often the same
        scores = torch.exp(_normal(g, (layers, n, kv, width * PAGE), torch.float32, 1.5))
        scores = torch.where(scores < 0.5, (scores * 64).round() / 64, scores)
        positions = torch.arange(width * PAGE, dtype=torch.int32, device=DEVICE).expand(layers, n, kv, -1).clone()
        old = case["rows"] - case["fresh"]
        if old > 0:  # the rows that earlier evictions left hold earlier positions, in no order, the newest rows the last ones
            order = torch.argsort(torch.rand((layers, n, kv, old), generator=g, device=DEVICE), dim=-1)
            positions[..., :old] = 3 * order.int()
            positions[..., old:] += 2 * old
        return dict(case=case, k=k, v=v, table=table, slots=list(range(n)), rows=rows, scores=scores, positions=positions,
                    new_scores=torch.zeros_like(scores), new_positions=torch.zeros_like(positions))
    held, brings, sizes, lengths = _sequences(case)
    need = [-(-(h + t) // PAGE) for h, t in zip(held, brings)]
    width = max(need)
    group_of = [i for i, s in enumerate(sizes) for _ in range(s)] if sizes else list(range(n))
    # a group's first sequence has pages for all that it holds, the others for what they hold of their own
    used = sum(need) - (sum((size - 1) * (p // PAGE) for size, p in zip(sizes, lengths)) if sizes else 0)
    pages = list(range(used))
    host.shuffle(pages)
    slots = list(range(n))
    host.shuffle(slots)
    table = torch.zeros((n, width), dtype=torch.int32)
    at = 0
    first = {}  # group -> its first sequence's pages
    for s in range(n):
        shared = first.get(group_of[s], [])
        mine = shared + pages[at:at + need[s] - len(shared)]
        at += need[s] - len(shared)
        if sizes and group_of[s] not in first:
            first[group_of[s]] = mine[:lengths[group_of[s]] // PAGE]
        table[slots[s], :need[s]] = torch.tensor(mine, dtype=torch.int32)
    table = table.to(DEVICE)
    heads = case["heads"]
    rows = sum(brings)
    qkv = _normal(g, (rows, (heads + 2 * kv) * dim), dtype)
    qkv[:, :heads * dim] *= 2  # what a trained model's normalised queries come to: a few keys stand out
    k = _normal(g, (used, kv, PAGE, dim), dtype)
    v = _normal(g, (used, kv, PAGE, dim), dtype)
    state = dict(case=case, qkv=qkv, k=k, v=v, table=table, slots=slots, held=held, brings=brings, sizes=sizes, lengths=lengths,
                 scale=1.0 / math.sqrt(dim))
    if case["kind"] == "scored":
        scores = torch.rand((n, kv, width * PAGE), generator=g, device=DEVICE) * 3
        state.update(scores=scores, new_scores=torch.zeros_like(scores),
                     positions=torch.zeros((n, kv, width * PAGE), dtype=torch.int32, device=DEVICE))
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if not own:
        return state
    from kernel_rush_kawk_b200.cache.store import KVView
    from kernel_rush_kawk_b200.csrc import load_kernels
    from kernel_rush_kawk_b200.engine.step import BatchMeta

    state["ops"] = load_kernels((case["dim"],))
    if case["kind"] == "evict":
        return state
    table = state["table"]
    state["cache"] = KVView(state["k"], state["v"], table, table.shape[1], None, case["kv"], case["dim"])
    n = case["batch"]
    batch = state["batch"] = BatchMeta(sum(state["brings"]), n, n, DEVICE)
    ends = [sum(state["brings"][:i + 1]) - 1 for i in range(n)]
    batch.fill(state["slots"], state["held"], [[0] * t for t in state["brings"]], ends)
    if case["kind"] == "prefix":
        from kernel_rush_kawk_b200.cache.prefix import PrefixGroups
        state["prefix"] = PrefixGroups(state["sizes"], state["lengths"], DEVICE)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        ops = state["ops"]
        if case["kind"] == "prefix":
            return ops.shared_prefix_attention(state["qkv"], case["heads"], case["kv"], case["dim"], state["batch"], state["cache"],
                                               state["scale"], state["prefix"])
        if case["kind"] == "scored":
            out = ops.scored_attention(state["qkv"], case["heads"], case["kv"], case["dim"], state["batch"], state["cache"], state["scale"],
                                       state["scores"], positions=state["positions"], observe=case["observe"] or None,
                                       out_scores=state["new_scores"])
            return out, state["new_scores"], state["positions"]
        ops.evict_keys(state["k"], state["v"], state["table"], state["slots"], state["rows"], state["scores"], state["positions"],
                       case["keep"], case["recent"], out_scores=state["new_scores"], out_positions=state["new_positions"])
        return state["k"], state["v"], state["new_scores"], state["new_positions"]
    if case["kind"] == "evict":
        return _plain_evict(state)
    return _plain_attention(state)


def _rows_of(pool, table_row, length):
    """[kv, length, dim] of one sequence's pages."""
    pages = pool[table_row[:-(-length // PAGE)].long()]
    return pages.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :length]


def _plain_attention(state):
    case = state["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    qkv = state["qkv"]
    out = torch.empty((qkv.shape[0], heads * dim), dtype=qkv.dtype, device=qkv.device)
    at = 0
    for slot, held, t in zip(state["slots"], state["held"], state["brings"]):
        total = held + t
        q = qkv[at:at + t, :heads * dim].float().view(t, kv, heads // kv, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)
        keys = _rows_of(state["k"], state["table"][slot], total).float()
        values = _rows_of(state["v"], state["table"][slot], total).float()
        s = torch.matmul(q, keys.transpose(1, 2)).view(kv, heads // kv, t, total) * state["scale"]
        if t > 1:
            seen = torch.arange(total, device=qkv.device)[None, :] <= held + torch.arange(t, device=qkv.device)[:, None]
            s = s.masked_fill(~seen, float("-inf"))
        p = torch.exp(s - s.amax(dim=-1, keepdim=True))
        p = p / p.sum(dim=-1, keepdim=True)
        o = torch.matmul(p.view(kv, -1, total), values).view(kv, heads // kv, t, dim)
        out[at:at + t] = o.permute(2, 0, 1, 3).reshape(t, heads * dim).to(out.dtype)
        if case["kind"] == "scored":
            seen_by = min(t, case["observe"] or t)
            got = p[:, :, t - seen_by:].sum(dim=(1, 2))
            got[:, :held] += state["scores"][slot, :, :held]
            state["new_scores"][slot, :, :total] = got
            state["positions"][slot, :, held:total] = torch.arange(held, total, dtype=torch.int32, device=qkv.device)
        at += t
    if case["kind"] == "scored":
        return out, state["new_scores"], state["positions"]
    return out


def _plain_evict(state):
    case = state["case"]
    keep, recent = case["keep"], case["recent"]
    k, v, table = state["k"], state["v"], state["table"]
    layers, kv = case["layers"], case["kv"]
    for slot, length in zip(state["slots"], state["rows"]):
        scores, positions = state["scores"][:, slot, :, :length], state["positions"][:, slot, :, :length]
        if length <= keep:
            state["new_scores"][:, slot, :, :length] = scores
            state["new_positions"][:, slot, :, :length] = positions
            continue
        rank = scores.clone()
        if recent:  # the newest keys before all others
            newest = positions.argsort(dim=-1, descending=True)[..., :recent]
            rank.scatter_(-1, newest, float("inf"))
        kept = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
        stays = torch.zeros_like(scores, dtype=torch.bool).scatter_(-1, kept, True)
        # (layer, head, row) in ascending order: as many free rows below ``keep`` as kept rows beyond it, head by head
        layer, head, to = torch.nonzero(~stays[..., :keep], as_tuple=True)
        source = torch.nonzero(stays[..., keep:], as_tuple=True)[2] + keep
        page = table[slot].long()
        for pool in (k, v):
            pool[layer, page[to // PAGE], head, to % PAGE] = pool[layer, page[source // PAGE], head, source % PAGE]
        for old, new in ((scores, state["new_scores"]), (positions, state["new_positions"])):
            line = old[..., :keep].clone()
            line[layer, head, to] = old[layer, head, source]
            new[:, slot, :, :keep] = line
    return k, v, state["new_scores"], state["new_positions"]


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "evict":
        return None  # rows and scores are moved, none is computed
    state = _inputs(case, seed)
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    per = heads // kv
    out = torch.zeros((state["qkv"].shape[0], heads, dim), dtype=torch.float64, device=DEVICE)
    sums = state["new_scores"].double() if case["kind"] == "scored" else None
    row = 0
    for i in range(case["batch"]):
        slot, held, t = state["slots"][i], state["held"][i], state["brings"][i]
        where = torch.arange(held + t, device=DEVICE)
        page, place = state["table"][slot].long()[where // PAGE], where % PAGE
        for h in range(kv):
            keys, values = state["k"][page, h, place].double(), state["v"][page, h, place].double()
            for j in range(per):
                q = state["qkv"][row:row + t, (h * per + j) * dim:(h * per + j + 1) * dim].double()
                logits = torch.einsum("td,kd->tk", q, keys) / math.sqrt(dim)
                logits = torch.where(where[None, :] - held <= torch.arange(t, device=DEVICE)[:, None], logits, -math.inf)
                log_sum = torch.logsumexp(logits, dim=1, keepdim=True)
                weights = torch.exp(logits - log_sum)
                out[row:row + t, h * per + j] = torch.einsum("tk,kd->td", weights, values)
                if sums is not None:
                    sums[slot, h, :held + t] += weights[-(case["observe"] or t):].sum(dim=0)
            if sums is not None:
                sums[slot, h, :held] += state["scores"][slot, h, :held].double()
        row += t
    out = out.view(-1, heads * dim)
    return out if sums is None else (out, sums, None)
