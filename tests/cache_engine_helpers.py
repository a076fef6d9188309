"""Shared by the tests of shared prefixes and eviction in the engine: a stand-in for the kernels on the CPU, and a plain
decoder that keeps its cache by the eviction's definition."""

from __future__ import annotations

import math

import torch

import plain_qwen3 as plain
from cache_ops_helpers import exact_attention, exact_evict
from torch_ops import TorchOps


class CacheTorchOps(TorchOps):
    """TorchOps with the operators that share and thin out the cache."""

    def __init__(self, dtype=torch.float32):
        super().__init__(dtype)
        self.calls = {"shared": 0, "scored": 0, "evict": 0}

    def qk_norm_rope_write(self, qkv, heads, kv_in_row, head_dim, q_gain, k_gain, eps, cos, sin, batch, cache):
        shift = getattr(batch, "seq_shift", None)
        if shift is None or cos is None:
            return super().qk_norm_rope_write(qkv, heads, kv_in_row, head_dim, q_gain, k_gain, eps, cos, sin, batch, cache)
        # the rows' angles lie further on than their places: tables that begin there, sequence by sequence
        for s in range(batch.n_seqs):
            rows = slice(int(batch.cu_q[s]), int(batch.cu_q[s + 1]))
            one = type("Rows", (), dict(row_pos=batch.row_pos[rows], row_seq=batch.row_seq[rows], seq_slot=batch.seq_slot))
            at = int(shift[s])
            part = qkv[rows].contiguous()
            super().qk_norm_rope_write(part, heads, kv_in_row, head_dim, q_gain, k_gain, eps, cos[at:], sin[at:], one, cache)
            qkv[rows] = part

    def shared_prefix_attention(self, qkv, heads, kv_in_row, head_dim, batch, cache, scale, prefix):
        self.calls["shared"] += 1
        prefix.check(batch, cache)
        at = 0
        for size, length in zip(prefix.sizes, prefix.lengths):  # neighbours do hold the same pages
            pages = [cache.table[s, :length // 64].tolist() for s in batch.slots[at:at + size]]
            assert all(p == pages[0] for p in pages)
            at += size
        return self.attention(qkv, heads, kv_in_row, head_dim, batch, cache, scale, None)

    def scored_attention(self, qkv, heads, kv_in_row, head_dim, batch, cache, scale, scores, positions=None, observe=None, out_scores=None):
        self.calls["scored"] += 1
        _, _, weights, _ = exact_attention(qkv, heads, kv_in_row, head_dim, batch, cache, scale, observe)
        for i, (slot, start, t) in enumerate(zip(batch.slots, batch.starts, batch.q_lens)):
            got = weights[i].float()
            got[:, :start] += scores[slot, :, :start]
            scores[slot, :, :start + t] = got
            positions[slot, :, start:start + t] = torch.arange(start, start + t, dtype=torch.int32) + int(batch.seq_shift[i])
        return self.attention(qkv, heads, kv_in_row, head_dim, batch, cache, scale, None)

    def evict_keys(self, k, v, table, slots, lengths, scores, positions, keep, recent, out_scores=None, out_positions=None, batch=None):
        self.calls["evict"] += 1
        for t, new in zip((k, v, scores, positions), exact_evict(k, v, table, slots, lengths, scores, positions, keep, recent)):
            t.copy_(new)


class PlainEvicting:
    """A Qwen3 decoder in 64 bits whose every kv head keeps a list of (key, value, weight received, position) and gives keys up by the
    definition: all but ``keep`` when ``keep + every`` or more are held before a step."""

    def __init__(self, folder, keep, recent, every, observe=None):
        self.cfg, w = plain.read_folder(folder)
        self.w = {k: t.double() for k, t in w.items()}
        self.keep, self.recent, self.every, self.observe = keep, recent, every, observe
        self.rows = [[[] for _ in range(self.cfg.kv_heads)] for _ in range(self.cfg.layers)]
        self.at = 0

    def held(self, layer=0, head=0):
        return [r[3] for r in self.rows[layer][head]]

    def step(self, ids) -> torch.Tensor:
        cfg, w, per = self.cfg, self.w, self.cfg.heads // self.cfg.kv_heads
        t, D = len(ids), cfg.head_dim
        cos, sin = plain.rope_tables(D, cfg.rope_theta, self.at + t, torch.float64)
        cos, sin = cos[self.at:], sin[self.at:]
        x = w["model.embed_tokens.weight"][torch.as_tensor(ids)]
        for i in range(cfg.layers):
            p = f"model.layers.{i}."
            h = plain.rms_norm(x, w[p + "input_layernorm.weight"], cfg.eps)
            q, k, v = (plain.linear(h, w[p + f"self_attn.{n}_proj.weight"]).view(t, -1, D) for n in "qkv")
            q = plain.head_norm_rope(q, w[p + "self_attn.q_norm.weight"], cos, sin, cfg.eps)
            k = plain.head_norm_rope(k, w[p + "self_attn.k_norm.weight"], cos, sin, cfg.eps)
            a = torch.empty((t, cfg.heads, D), dtype=torch.float64)
            for g in range(cfg.kv_heads):
                rows = self.rows[i][g]
                if len(rows) >= self.keep + self.every:
                    newest = sorted(rows, key=lambda r: -r[3])[:self.recent]
                    rest = [r for r in rows if all(r is not n for n in newest)]
                    rows = newest + sorted(rest, key=lambda r: -r[2])[:self.keep - self.recent]
                old = len(rows)
                rows = rows + [[k[j, g], v[j, g], 0.0, self.at + j] for j in range(t)]
                keys, values = torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows])
                seen = torch.arange(len(rows))[None, :] < old + 1 + torch.arange(t)[:, None]
                first = t - min(t, self.observe or t)
                for hh in range(g * per, (g + 1) * per):
                    s = (q[:, hh] @ keys.t() / math.sqrt(D)).masked_fill(~seen, -math.inf)
                    weights = torch.softmax(s, dim=-1)
                    a[:, hh] = weights @ values
                    for r, add in zip(rows, weights[first:].sum(dim=0).tolist()):
                        r[2] += add
                self.rows[i][g] = rows
            x = x + plain.linear(a.reshape(t, -1), w[p + "self_attn.o_proj.weight"])
            h = plain.rms_norm(x, w[p + "post_attention_layernorm.weight"], cfg.eps)
            x = x + plain.swiglu_mlp(h, w[p + "mlp.gate_proj.weight"], w[p + "mlp.up_proj.weight"], w[p + "mlp.down_proj.weight"])
        self.at += t
        head = w["model.embed_tokens.weight"] if cfg.tie else w["lm_head.weight"]
        return plain.rms_norm(x, w["model.norm.weight"], cfg.eps) @ head.t()
