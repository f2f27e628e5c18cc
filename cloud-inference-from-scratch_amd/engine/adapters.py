"""Low-rank adapters of a running engine: reading a folder, names, slots."""

from __future__ import annotations

import json
import math
from collections.abc import Iterable, Mapping
from dataclasses import dataclass
from pathlib import Path
from typing import Any

import torch

from ..parts.adapters import AdapterError, AdapterRoom

_PREFIX = "base_model.model."


def read_config(folder: str | Path) -> tuple[int, float]:
    """(rank, scale) of a folder's ``adapter_config.json`` (``r``, ``lora_alpha``, ``use_rslora``).  What would change the formula
    and is not built is refused."""
    with open(Path(folder) / "adapter_config.json", encoding="utf-8") as handle:
        raw = json.load(handle)
    if not isinstance(raw, dict):
        raise AdapterError("adapter_config.json holds no object")
    faults = []
    if str(raw.get("peft_type", "LORA")).upper() != "LORA":
        faults.append(f"peft_type {raw['peft_type']!r}")
    if raw.get("bias", "none") != "none":
        faults.append(f"bias {raw['bias']!r}")
    faults += [f"{name} {raw[name]!r}" for name in ("use_dora", "fan_in_fan_out", "modules_to_save", "rank_pattern", "alpha_pattern",
                                                    "lora_bias", "layer_replication", "alora_invocation_tokens", "use_qalora",
                                                    "use_bdlora", "arrow_config")
               if raw.get(name)]
    # (any other start also takes something out of the weights that the matrices were trained beside)
    if isinstance(raw.get("init_lora_weights"), str) and raw["init_lora_weights"] not in ("gaussian", "eva", "orthogonal"):
        faults.append(f"init_lora_weights {raw['init_lora_weights']!r}")
    rank, alpha = raw.get("r"), raw.get("lora_alpha")
    if not (isinstance(rank, int) and rank > 0 and isinstance(alpha, (int, float)) and math.isfinite(alpha)):
        faults.append(f"r {rank!r} and lora_alpha {alpha!r}")
    if faults:
        raise AdapterError("an adapter of this kind is not run: " + "; ".join(faults))
    return rank, alpha / (math.sqrt(rank) if raw.get("use_rslora") else rank)


def read_adapter(folder: str | Path) -> tuple[dict[str, torch.Tensor], float]:
    """(tensors by the model's own names, scale) of a folder with ``adapter_config.json`` and ``adapter_model.safetensors``."""
    import safetensors.torch

    folder = Path(folder)
    rank, scale = read_config(folder)
    stored = safetensors.torch.load_file(str(folder / "adapter_model.safetensors"))
    tensors: dict[str, torch.Tensor] = {}
    for stored_name, tensor in stored.items():
        name = stored_name[len(_PREFIX):] if stored_name.startswith(_PREFIX) else stored_name
        name = name.replace(".lora_A.default.weight", ".lora_A.weight").replace(".lora_B.default.weight", ".lora_B.weight")
        if name in tensors:
            raise AdapterError(f"the adapter has {name} under two names")
        tensors[name] = tensor
    others = sorted({int(t.shape[0]) for name, t in tensors.items() if name.endswith(".lora_A.weight") and t.dim() == 2} - {rank})
    if others:
        raise AdapterError(f"the adapter's r is {rank}, and it has matrices of rank {others}: their scale is not told")
    return tensors, scale


@dataclass(frozen=True)
class Loaded:
    slot: int
    serial: int  # of all that were ever loaded: what one of them left in the prefix index is no other's


class Adapters:
    """The adapters of an engine by name."""

    def __init__(self, room: AdapterRoom) -> None:
        self.room = room
        self.loaded: dict[str, Loaded] = {}
        self._serial = 0

    def load(self, name: str, tensors: Mapping[str, torch.Tensor], scale: float) -> Loaded:
        if not name:
            raise ValueError("an adapter needs a name")
        if name in self.loaded:
            raise ValueError(f"an adapter {name!r} is loaded already: unload it first")
        if not abs(scale) <= torch.finfo(torch.float32).max:  # (the room holds it in 32 bits)
            raise ValueError(f"an adapter's scale must be a finite number of 32 bits, not {scale}")
        taken = {known.slot for known in self.loaded.values()}
        slot = next((s for s in range(self.room.count) if s not in taken), None)
        if slot is None:
            raise ValueError(f"all {self.room.count} adapter slots are taken (max_adapters)")
        self.room.load(slot, tensors, scale)
        self._serial += 1
        self.loaded[name] = Loaded(slot, self._serial)
        return self.loaded[name]

    def unload(self, name: str, requests: Iterable[Any]) -> None:
        known = self.find(name)
        if any(request.adapter == known for request in requests):
            raise ValueError(f"requests that are not finished have the adapter {name!r}")
        del self.loaded[name]

    def find(self, name: str) -> Loaded:
        if name not in self.loaded:
            raise ValueError(f"no adapter {name!r} is loaded; loaded: {sorted(self.loaded)}")
        return self.loaded[name]
