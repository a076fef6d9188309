"""Shared by the tests of adapters and maps: inputs, the operators in 64 bits with bounds on their error, the maps by hand.

The bounds, derived before any run. A product of K terms held in float32 on the tensor cores adds 16 terms at a time and cuts off
what lies behind 2^-22 of the running sum: (K / 16 + 16) * 2^-22 of the sum of the terms' absolute values; in float32 multiply-adds one after the
other at most K * 2^-24 of it. The first factor's sums may be rounded to bfloat16 on their way to the second (half a step, 2^-8 of each), the result is
rounded once (2^-8, or 2^-24 in float32). silu has a slope of at most 1.1; its exponential and quotient are good to 2^-20 together.
"""

from __future__ import annotations

import torch

from kernel_rush_kawk_b200.parts.adapters import AdapterBank


def make_adapters(g, count, inputs, outs, rank, dtype, device, skip=()):
    """[adapter][part] -> (a, b, scale) or None. Ranks differ; ``skip``: (adapter, part) pairs that are left out."""
    out = []
    for i in range(count):
        parts = []
        for p, n in enumerate(outs):
            r = max(1, rank - (3 * i + p) % (rank // 2 + 1))
            a = torch.randn((r, inputs), generator=g) / inputs ** 0.5
            b = torch.randn((n, r), generator=g) * 0.1
            parts.append(None if (i, p) in skip else (a.to(device, dtype), b.to(device, dtype), 0.5 + 0.25 * i))
        out.append(parts)
    return out


def make_bank(adapters, inputs, outs, rank, dtype, device, capacity=None):
    bank = AdapterBank(inputs, outs, capacity or len(adapters), rank, dtype, device)
    for i, parts in enumerate(adapters):
        for p, part in enumerate(parts):
            if part is not None:
                bank.put(i, p, *part)
    return bank


def product64(x, w, adapters, outs, adapter_of_row, rounded_t):
    """(y in 64 bits, the bound on its error before the last rounding)."""
    x64, w64 = x.double(), w.double()
    K = x.shape[1]
    eps = (K / 16 + 16) * 2.0 ** -22 if x.dtype == torch.bfloat16 else (K + 32) * 2.0 ** -24
    y = x64 @ w64.T
    bound = eps * (x64.abs() @ w64.abs().T)
    for a, parts in enumerate(adapters):
        rows = [r for r, b in enumerate(adapter_of_row) if b == a]
        if not rows:
            continue
        at = 0
        for n, part in zip(outs, parts):
            if part is not None:
                A, B, s = part[0].double(), part[1].double(), part[2]
                t = s * (x64[rows] @ A.T)
                dt = eps * abs(s) * (x64[rows].abs() @ A.abs().T) + (2.0 ** -8 if rounded_t else 2.0 ** -22) * t.abs()
                y[rows, at:at + n] += t @ B.T
                bound[rows, at:at + n] += dt @ B.abs().T + (A.shape[0] + 16) * 2.0 ** -22 * (t.abs() @ B.abs().T)
            at += n
    return y, bound


def gated64(y, bound):
    half = y.shape[1] // 2
    g, u, dg, du = y[:, :half], y[:, half:], bound[:, :half], bound[:, half:]
    z = g * torch.sigmoid(g)
    return z * u, 1.1 * dg * u.abs() + z.abs() * du + 1.1 * dg * du + 2.0 ** -20 * (z * u).abs()


def assert_within(got, ref, bound, what=""):
    step = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    room = bound + step * (ref.abs() + bound) + 1e-30
    over = ((got.double() - ref).abs() / room).nan_to_num(nan=1e9)
    assert over.max().item() <= 1.0, f"{what}: off by {over.max().item():.2f} times the bound at {tuple(torch.unravel_index(over.argmax(), over.shape))}"


def per_row(lengths, of_sequence):
    return [a for a, n in zip(of_sequence, lengths) for _ in range(n)]


def rows_of_step(ops, lengths, of_sequence, device):
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    zeros = torch.zeros_like(n)
    return ops.step_maps(zeros, zeros, n, sum(lengths), adapters=torch.tensor(of_sequence, dtype=torch.int32, device=device)).adapters


def maps_by_hand(slots, starts, lengths, table, pages, adapters):
    """(cu_q, row_seq, row_pos, row_place, row_adapter) as lists; ``table`` (a list of lists) is filled."""
    cu, seq, pos, place, of = [0], [], [], [], []
    fresh = iter(pages or ())
    for s, (slot, start, n) in enumerate(zip(slots, starts, lengths)):
        cu.append(cu[-1] + n)
        if table is not None:
            for logical in range(-(-start // 64), -(-(start + n) // 64)):
                table[slot][logical] = next(fresh)
        for p in range(start, start + n):
            seq.append(s)
            pos.append(p)
            of.append(adapters[s] if adapters is not None else None)
            place.append(table[slot][p // 64] * 64 + p % 64 if table is not None else None)
    return cu, seq, pos, place, of


# -- engines ------------------------------------------------------------------------------------------------------------

def random_factors(cfg, w, seed, rank, keys=("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"), layers=None, std=0.25):
    """{checkpoint name: (a, b, scale)} for the named projections of a plain model's layers, large enough to move the logits."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, t in w.items():
        if t.dim() == 2 and name.split(".")[-2] in keys and (layers is None or int(name.split(".")[2]) in layers):
            r = max(1, rank - len(out) % 3)
            out[name] = (torch.randn((r, t.shape[1]), generator=g) / t.shape[1] ** 0.5, torch.randn((t.shape[0], r), generator=g) * std / r ** 0.5, 0.75 + 0.25 * (seed % 3))
    return out


def merged(w, factors):
    """The plain model's weights with an adapter's products added (None: as they are)."""
    if factors is None:
        return w
    return {name: t if name not in factors else (t.double() + factors[name][2] * factors[name][1].double() @ factors[name][0].double()).to(t.dtype)
            for name, t in w.items()}


def write_adapter(folder, factors, alpha=8.0, prefix="base_model.model.", **config):
    """An adapter's folder; the scales are alpha / r."""
    import json

    from safetensors.torch import save_file

    folder.mkdir(parents=True)
    (folder / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": alpha, **config}))
    tensors = {}
    for name, (a, b, _) in factors.items():
        module = prefix + name.removesuffix(".weight")
        tensors[module + ".lora_A.weight"], tensors[module + ".lora_B.weight"] = a.contiguous(), b.contiguous()
    save_file(tensors, str(folder / "adapter_model.safetensors"))
    return folder
