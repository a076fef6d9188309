"""Low-rank adapters from files, by the names of the weights that they stand beside.

A folder holds ``adapter_config.json`` (``r`` and ``lora_alpha``: the scale is alpha / r, or alpha / sqrt(r) with
``use_rslora``) and safetensors with two tensors for each weight: ``<module>.lora_A.weight`` [r, inputs] and
``<module>.lora_B.weight`` [outputs, r], where ``<module>.weight`` is the weight's name in the checkpoint (a leading
``base_model.model.`` is dropped). Adapters that are more than these products, or beside weights changed for them, are refused. An adapter's tensors may have ranks of their own; the scale then goes by each one's.
"""

from __future__ import annotations

import json
import math
from pathlib import Path

import torch

from ..parts.adapters import AdapterError


def read_adapter(folder) -> dict[str, tuple[torch.Tensor, torch.Tensor, float]]:
    """Checkpoint name of a weight -> (a, b, scale), on the host."""
    from safetensors import safe_open

    folder = Path(folder)
    try:
        config = json.loads((folder / "adapter_config.json").read_text())
        alpha = float(config["lora_alpha"])
    except (OSError, ValueError, KeyError, TypeError) as e:
        raise AdapterError(f"{folder}: adapter_config.json with a lora_alpha is asked for ({e})") from e
    for key in ("alpha_pattern", "modules_to_save", "use_dora", "fan_in_fan_out", "use_qalora", "alora_invocation_tokens", "layer_replication", "lora_bias",
                "trainable_token_indices"):
        if config.get(key):
            raise AdapterError(f"{folder}: adapters with {key} are not taken")
    if config.get("peft_type", "LORA") != "LORA":
        raise AdapterError(f"{folder}: adapters of the type {config['peft_type']} are not taken")
    # beginnings that leave the weights as they are; others take a product out of them, and the factors then belong to what is left
    if config.get("init_lora_weights") not in (None, True, False, "gaussian", "eva", "orthogonal"):
        raise AdapterError(f"{folder}: adapters that began with '{config['init_lora_weights']}' belong to changed weights and are not taken")
    if config.get("bias", "none") != "none":
        raise AdapterError(f"{folder}: adapters with biases are not taken")
    shards = sorted(folder.glob("*.safetensors"))
    if not shards:
        raise AdapterError(f"no *.safetensors under {folder}")
    found: dict[str, dict[str, torch.Tensor]] = {}
    for shard in shards:
        try:
            with safe_open(str(shard), framework="pt", device="cpu") as f:
                for name in f.keys():
                    module, _, which = name.removeprefix("base_model.model.").partition(".lora_")
                    if which not in ("A.weight", "B.weight"):
                        raise AdapterError(f"{folder}: {name} is no factor of a low-rank adapter")
                    if found.setdefault(module + ".weight", {}).setdefault(which[0], tensor := f.get_tensor(name)) is not tensor:
                        raise AdapterError(f"{folder}: {name} comes twice")
        except AdapterError:
            raise
        except Exception as e:  # a truncated or corrupt shard
            raise AdapterError(f"{shard} cannot be read: {e}") from e
    out = {}
    for name, factors in sorted(found.items()):
        if set(factors) != {"A", "B"}:
            raise AdapterError(f"{folder}: one factor beside {name} is missing")
        a, b = factors["A"], factors["B"]
        if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1] or a.shape[0] == 0:
            raise AdapterError(f"{folder}: factors beside {name} are [rank, inputs] and [outputs, rank], got {list(a.shape)} and {list(b.shape)}")
        r = a.shape[0]
        out[name] = (a, b, alpha / (math.sqrt(r) if config.get("use_rslora") else r))
    return out
