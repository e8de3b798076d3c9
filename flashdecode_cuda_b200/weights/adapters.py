"""Low-rank adapters on disk: ``adapter_config.json`` (rank, ``lora_alpha``, the modules) and ``adapter_model.safetensors`` with
two matrices per adapted projection, ``<module>.lora_A.weight`` [r, in] and ``<module>.lora_B.weight`` [out, r]; the projection's
output gets scale * B (A x) added, scale = alpha / r (alpha / sqrt(r) with ``use_rslora``).  davidjoyme/flashdecode-cuda has no
adapters."""

from __future__ import annotations

import json
import math
from pathlib import Path
from typing import Dict, Tuple

import torch

from .safetensors_io import read_file, write_file


class AdapterError(ValueError):
    """The files or tensors are not those of a low-rank adapter that can be added here."""


_PREFIX = "base_model.model."
Adapter = Dict[str, Tuple[torch.Tensor, torch.Tensor]]         # module -> (A [r, in], B [out, r])


def pair_up(tensors: Dict[str, torch.Tensor]) -> Adapter:
    """(A, B) by module name from tensors by name; the modules' names with or without the writer's prefix."""
    halves: Dict[str, dict] = {}
    for name, t in tensors.items():
        short = name[len(_PREFIX):] if name.startswith(_PREFIX) else name
        for half in ("lora_A", "lora_B"):
            for tail in (f".{half}.weight", f".{half}.default.weight"):
                if short.endswith(tail):
                    halves.setdefault(short[:-len(tail)], {})[half] = t
                    break
            else:
                continue
            break
        else:
            raise AdapterError(f"{name}: not a tensor of a low-rank adapter (<module>.lora_A.weight or .lora_B.weight)")
    out: Adapter = {}
    for module, ab in halves.items():
        if len(ab) != 2:
            raise AdapterError(f"{module}: lora_A and lora_B come together")
        a, b = ab["lora_A"], ab["lora_B"]
        if a.dim() != 2 or b.dim() != 2 or a.shape[0] != b.shape[1]:
            raise AdapterError(f"{module}: lora_A {tuple(a.shape)} and lora_B {tuple(b.shape)} are not [r, in] and [out, r]")
        out[module] = (a, b)
    if not out:
        raise AdapterError("an adapter without a tensor")
    return out


def read_adapter(folder) -> Tuple[Adapter, float]:
    """(matrices by module, scale) of an adapter folder."""
    folder = Path(folder)
    config = json.loads((folder / "adapter_config.json").read_text())
    for key, plain in (("bias", "none"), ("use_dora", False), ("modules_to_save", None), ("fan_in_fan_out", False),
                       ("rank_pattern", {}), ("alpha_pattern", {})):
        if config.get(key, plain) not in (plain, None, [], {}):
            raise AdapterError(f"{folder}: adapters with {key} = {config[key]!r} are not taken")
    rank, alpha = config.get("r"), config.get("lora_alpha")
    if not isinstance(rank, int) or rank < 1 or not isinstance(alpha, (int, float)):
        raise AdapterError(f"{folder}: adapter_config.json needs r and lora_alpha")
    pairs = pair_up(read_file(folder / "adapter_model.safetensors"))
    for module, (a, _) in pairs.items():
        if a.shape[0] != rank:
            raise AdapterError(f"{folder}: {module} has rank {a.shape[0]}, the configuration says {rank}")
    return pairs, alpha / math.sqrt(rank) if config.get("use_rslora") else alpha / rank


def write_adapter(folder, pairs: Adapter, alpha: float) -> Path:
    folder = Path(folder)
    folder.mkdir(parents=True, exist_ok=True)
    ranks = {a.shape[0] for a, _ in pairs.values()}
    if len(ranks) != 1:
        raise AdapterError(f"an adapter folder has one rank, not {sorted(ranks)}")
    (folder / "adapter_config.json").write_text(json.dumps(
        {"peft_type": "LORA", "r": ranks.pop(), "lora_alpha": alpha, "target_modules": sorted({m.rsplit(".", 1)[-1] for m in pairs})}, indent=1))
    tensors = {}
    for module, (a, b) in pairs.items():
        tensors[f"{_PREFIX}{module}.lora_A.weight"], tensors[f"{_PREFIX}{module}.lora_B.weight"] = a, b
    write_file(folder / "adapter_model.safetensors", tensors)
    return folder
