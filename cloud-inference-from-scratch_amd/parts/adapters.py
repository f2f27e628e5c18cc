"""Room for low-rank adapters beside a model's projections, so that requests of one batch can each bring their own.

An adapter gives a projection ``W`` of the checkpoint two small matrices, ``A`` [r, in] and ``B`` [out, r]: rows of a request that
has it see ``W x + s B (A x)``.  A part stacks the projections that read the same rows (q, k and v; gate and up), and its adapters are
stacked alike: a :class:`Site` holds, for every slot of the room, the A of all its projections on top of each other and their B
side by side, in the model's type, ready for ``ops.lora_add``.  Adapters of a lower rank than the room's are filled up with
zeros, and so is whatever projection an adapter leaves out.

The room's tensors are made once and only rewritten, so captured steps may hold on to them.
"""

from __future__ import annotations

from collections.abc import Callable, Mapping, Sequence
from dataclasses import dataclass
from typing import Any, Optional

import torch

from ..kernels import ops
from .base import declares


class Site:
    """The adapters of one stacked projection with ``inputs`` numbers a row and ``columns`` of each projection."""

    def __init__(self, inputs: int, columns: Sequence[int], count: int, rank: int, dtype: torch.dtype, device: Any,
                 scale: torch.Tensor) -> None:
        self.columns = tuple(columns)
        self.rank = rank
        self.down = torch.zeros((count, len(self.columns) * rank, inputs), dtype=dtype, device=device)
        self.up = torch.zeros((count, sum(self.columns), rank), dtype=dtype, device=device)
        self.scale = scale  # float32 [count], the room's

    def clear(self, slot: int) -> None:
        self.down[slot].zero_()
        self.up[slot].zero_()

    def put(self, slot: int, piece: int, a: torch.Tensor, b: torch.Tensor) -> None:
        first, rank = sum(self.columns[:piece]), a.shape[0]
        self.down[slot, piece * self.rank: piece * self.rank + rank].copy_(a)
        self.up[slot, first: first + self.columns[piece], :rank].copy_(b)

    def add(self, x: torch.Tensor, adapters: torch.Tensor, into: torch.Tensor) -> None:
        """``into`` (x's type, or the float32 stream) plus what each row's adapter makes of its row of ``x``."""
        ops.lora_add(x, self.down, self.up, self.scale, adapters, into, columns=self.columns)


def _as_is(t: torch.Tensor) -> torch.Tensor:
    return t


@dataclass
class Module:
    """One projection of the checkpoint: where its adapters go, and the shapes that their matrices have there.  ``shape_a`` and
    ``shape_b`` bring a matrix to the shape in which the part runs the projection (heads padded to a size of the kernels)."""

    site: Site
    piece: int
    inputs: int
    outputs: int
    shape_a: Callable[[torch.Tensor], torch.Tensor] = _as_is
    shape_b: Callable[[torch.Tensor], torch.Tensor] = _as_is


class AdapterError(ValueError):
    """An adapter that this model cannot take; the message lists every fault."""


class AdapterRoom:
    def __init__(self, model: Any, count: int, rank: int) -> None:
        if count < 1 or not 1 <= rank <= ops.MAX_ADAPTER_RANK:
            raise ValueError(f"room for at least one adapter of rank 1 to {ops.MAX_ADAPTER_RANK}, not {count} of {rank}")
        self.count = count
        self.rank = -(-rank // 8) * 8  # (whole 16-byte pieces)
        self.scale = torch.zeros(count, dtype=torch.float32, device=model.device)
        self.modules: dict[str, Module] = {}
        for index, block in enumerate(model.blocks):
            prefix = model.spec.layer_prefix.format(index=index)
            for role, part in block._parts() if declares(block, "takes_adapters") else ():
                if role.startswith("norm") or not part.expected_tensors(""):
                    continue
                if not declares(part, "takes_adapters"):
                    raise AdapterError(f"layer {index}: a {role} of this kind takes no adapters")
                for name, module in part.make_sites(self.count, self.rank, self.scale).items():
                    self.modules[f"{prefix}{block.spec.name_of(role)}.{name}"] = module
            if not declares(block, "takes_adapters"):
                raise AdapterError(f"layer {index}: layers of this arrangement take no adapters")

        model.adapter_room = self

    @property
    def sites(self) -> list[Site]:
        return list({id(module.site): module.site for module in self.modules.values()}.values())

    def load(self, slot: int, tensors: Mapping[str, torch.Tensor], scale: float) -> None:
        """Put an adapter into ``slot``: ``tensors`` holds ``<projection>.lora_A.weight`` [r, in] and ``<projection>.lora_B.weight``
        [out, r] for some of the model's projections.  Everything is checked before anything is written."""
        if not 0 <= slot < self.count:
            raise ValueError(f"slot {slot} of {self.count}")
        pairs: dict[str, dict[str, torch.Tensor]] = {}
        faults: list[str] = []
        for name, tensor in tensors.items():
            side = next((s for s in ("A", "B") if name.endswith(f".lora_{s}.weight")), None)
            module = name[: -len(".lora_A.weight")] if side else name
            if side is None or module not in self.modules:
                faults.append(f"{name} belongs to no projection of this model")
            else:
                pairs.setdefault(module, {})[side] = tensor
        for module, pair in pairs.items():
            known = self.modules[module]
            if set(pair) != {"A", "B"}:
                faults.append(f"{module} has no lora_{'B' if 'A' in pair else 'A'}")
                continue
            a, b = pair["A"], pair["B"]
            if not (a.dim() == b.dim() == 2 and a.is_floating_point() and b.is_floating_point() and a.shape[1] == known.inputs
                    and b.shape[0] == known.outputs and a.shape[0] == b.shape[1] and 1 <= a.shape[0] <= self.rank):
                faults.append(f"{module}: A {tuple(a.shape)} and B {tuple(b.shape)} instead of (r, {known.inputs}) and "
                              f"({known.outputs}, r) with r from 1 to {self.rank}")
        if not pairs and not faults:
            faults.append("it has no tensors")
        if faults:
            raise AdapterError("the adapter does not fit the model:\n  " + "\n  ".join(faults))
        for site in self.sites:
            site.clear(slot)
        for module, pair in pairs.items():
            known = self.modules[module]
            known.site.put(slot, known.piece, known.shape_a(pair["A"]), known.shape_b(pair["B"]))
        self.scale[slot: slot + 1].fill_(scale)


def rows_complete(x: Any) -> torch.Tensor:
    """The rows themselves, where a norm left them to the product that reads them."""
    complete = getattr(x, "complete", None)
    return x if complete is None else complete()


def add_behind(site: Site, rows: torch.Tensor, adapters: torch.Tensor, residual: Optional[torch.Tensor],
               product: Callable[[], Any]) -> Any:
    """A part's last product and its adapters.  Where the branch joins the float32 stream the adapters' share goes there first
    (a product that adds there itself may also leave sums of the new stream's rows), else into the product's rows."""
    if residual is not None:
        site.add(rows, adapters, residual)
        return product()
    out = product()
    site.add(rows, adapters, out)
    return out
