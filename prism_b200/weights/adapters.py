"""Low-rank adapters beside a loaded model's projections: ``W + s B A`` for the requests that name an adapter, ``W`` for the
others, in one batch (``ops.low_rank``).  andre-fu/prism has none; a model folder of its own takes their place there
(engine/weight_manager.py:45).

``AdapterSet`` has room for a number of adapters of ranks up to a limit beside every matrix that the blocks' mixers and
feed-forward layers name in ``adaptable``: one ``ops.LowRank`` each, with a slice for every file tensor that the
matrix stacks (q, k and v; gate and up).  Matrices that a block runs jointly, experts and the head have none.
"""

from __future__ import annotations

import json
import math
import os
from typing import Dict, Iterator, List, Tuple

import torch

from .. import ops

CONFIG, TENSORS = "adapter_config.json", "adapter_model.safetensors"
# settings that, where they are on, change the formula: other scales, ranks or layers, more parameters, tokens that the adapter leaves alone
OTHER_FORMULAS = ("use_dora", "rank_pattern", "alpha_pattern", "modules_to_save", "fan_in_fan_out", "layer_replication", "lora_bias", "trainable_token_indices",
                  "alora_invocation_tokens", "arrow_config", "use_qalora", "use_bdlora")
# of the named ways to begin training those that leave W as it is; others take their product out of W, or round it
PLAIN_BEGINNINGS = ("gaussian", "eva", "orthogonal")


class AdapterError(ValueError):
    """An adapter that does not fit the model or the room for it; says everything that is wrong with it."""


def check_adapter_room(max_adapters, max_rank) -> None:
    if int(max_adapters) != max_adapters or max_adapters < 0:
        raise ValueError(f"max_adapters {max_adapters!r}: a number of adapters, or 0 for none")
    if int(max_rank) != max_rank or not 1 <= max_rank <= ops.low_rank_limits()[0]:
        raise ValueError(f"max_adapter_rank {max_rank!r}: from 1 to {ops.low_rank_limits()[0]}")


def adaptable_params(model) -> Iterator[Tuple[str, object, object]]:
    """``(qualified name, part, ParamSpec with the file tensors' full names)`` of every matrix that may have adapters."""
    specs = dict(model.named_params())
    for i, block in enumerate(model.layers):
        for child in ("mixer", "feed_forward"):
            part = block.children.get(child)
            own = {p.name for p in part.params()} if part is not None else ()
            for name in part.adaptable if part is not None else ():
                q = f"layers.{i}.{child}.{name}"
                if name in own and specs[q].axis == 0 and len(specs[q].sources) <= ops.low_rank_limits()[1]:
                    yield q, part, specs[q]


def read_adapter_config(folder: str) -> Tuple[int, float]:
    """``(rank, scale)`` of an adapter folder.  What would change the formula beyond ``W + scale B A`` is refused."""
    path = os.path.join(folder, CONFIG)
    if not os.path.isfile(path):
        raise AdapterError(f"no {CONFIG} in {folder}")
    try:
        with open(path) as f:
            raw = json.load(f)
    except ValueError as e:                          # no text, or no JSON
        raise AdapterError(f"{path}: {e}") from None
    if not isinstance(raw, dict):
        raise AdapterError(f"{path}: an object with the adapter's settings is needed, got {type(raw).__name__}")
    bad = [k for k in OTHER_FORMULAS if raw.get(k)]
    begin = raw.get("init_lora_weights")
    if isinstance(begin, str) and begin.lower() not in PLAIN_BEGINNINGS:
        bad.append("init_lora_weights")
    if raw.get("bias", "none") != "none":
        bad.append("bias")
    if raw.get("peft_type", "LORA") != "LORA":
        bad.append("peft_type")
    if bad:
        raise AdapterError(f"{path}: not supported: {', '.join(f'{k}={raw[k]!r}' for k in bad)}")
    r, alpha = raw.get("r"), raw.get("lora_alpha")
    if not isinstance(r, int) or isinstance(r, bool) or r < 1 or not isinstance(alpha, (int, float)) or not math.isfinite(alpha):
        raise AdapterError(f"{path}: r {r!r} and lora_alpha {alpha!r} must be a positive whole number and a number")
    return r, float(alpha) / (math.sqrt(r) if raw.get("use_rslora") else r)


def read_adapter_folder(folder: str) -> Tuple[Dict[str, Tuple[torch.Tensor, torch.Tensor]], float]:
    """``({module: (A [rank, in], B [out, rank])}, scale)`` of a folder with ``adapter_config.json`` (``r``, ``lora_alpha``) and
    ``adapter_model.safetensors`` (``[base_model.model.]<module>.lora_A.weight`` and ``.lora_B.weight`` for the model file's tensor
    ``<module>.weight``, or ``<module>`` in a design whose tensors are named without that ending)."""
    from safetensors import SafetensorError, safe_open
    rank, scale = read_adapter_config(folder)
    path = os.path.join(folder, TENSORS)
    if not os.path.isfile(path):
        raise AdapterError(f"no {TENSORS} in {folder}")
    halves: Dict[str, Dict[str, torch.Tensor]] = {}
    wrong: List[str] = []
    try:
        with safe_open(path, framework="pt", device="cpu") as f:
            tensors = {name: f.get_tensor(name) for name in f.keys()}
    except SafetensorError as e:
        raise AdapterError(f"{path}: {e}") from None
    for name, t in tensors.items():
        module, _, half = name.rpartition(".lora_")
        if half not in ("A.weight", "B.weight") or not module:
            wrong.append(f"unexpected tensor {name}")
            continue
        module = module[len("base_model.model."):] if module.startswith("base_model.model.") else module
        if t.dim() != 2 or t.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            wrong.append(f"{name}: a matrix in float32, float16 or bfloat16 is needed, got {t.dtype} {tuple(t.shape)}")
        if half[0] in halves.setdefault(module, {}):
            wrong.append(f"{name}: {module} is named twice")
        halves[module][half[0]] = t
    for name, ab in halves.items():
        if len(ab) != 2:
            wrong.append(f"{name}: only its {next(iter(ab))} is there")
        elif ab["A"].dim() == 2 and ab["A"].shape[0] != rank:
            wrong.append(f"{name}: rank {ab['A'].shape[0]}, the configuration says {rank}")
    if wrong or not halves:
        raise AdapterError(f"{path}: " + ("; ".join(wrong) or "no tensors"))
    return {n: (ab["A"], ab["B"]) for n, ab in halves.items()}, scale


class AdapterSet:
    """``model`` is bound to its matrices with room for adapters beside them; ``step`` is what a step's runner tells them."""

    def __init__(self, model, count: int, max_rank: int, device, dtype: torch.dtype):
        check_adapter_room(count, max_rank)
        self.count, self.max_rank = int(count), int(max_rank)
        self.step = ops.AdapterStep()
        self.places: Dict[str, Tuple[ops.LowRank, int]] = {}             # file tensor -> its projection's adapters, its slice
        self.stacks: List[ops.LowRank] = []
        self.names: Dict[str, int] = {}
        for q, part, spec in adaptable_params(model):
            name, w = q.rsplit(".", 1)[-1], part.w[q.rsplit(".", 1)[-1]]
            if w is None:
                continue
            low = ops.LowRank.empty(self.count, self.max_rank, [s.shape[0] for s in spec.sources], spec.shape[1], dtype, device)
            part.w[name] = ops.Adapted(w, low, self.step)
            self.stacks.append(low)
            for i, s in enumerate(spec.sources):
                self.places[s.name] = (low, i)
        if not self.places:
            raise AdapterError("no matrix of this model may have adapters beside it")

    @property
    def nbytes(self) -> int:
        return sum(low.nbytes for low in self.stacks)

    def number(self, name: str) -> int:
        try:
            return self.names[name]
        except KeyError:
            raise AdapterError(f"no adapter {name!r} is loaded; there are: {sorted(self.names)}") from None

    def load(self, name: str, folder: str) -> int:
        return self.add(name, *read_adapter_folder(folder))

    def add(self, name: str, tensors: Dict[str, Tuple[torch.Tensor, torch.Tensor]], scale: float) -> int:
        """Adapter ``name`` with ``(A, B)`` for some of the model's file tensors (by their names, with or without ``.weight``); the others stay as
        they are.  Returns its number."""
        if name in self.names:
            raise AdapterError(f"adapter {name!r} is loaded already")
        free = sorted(set(range(self.count)) - set(self.names.values()))
        if not free:
            raise AdapterError(f"no room for adapter {name!r}: all {self.count} places are taken by {sorted(self.names)}")
        wrong, named = [], {t if t in self.places else t + ".weight": ab for t, ab in tensors.items()}
        if len(named) != len(tensors):
            wrong.append("a matrix is named twice")
        for t, (a, b) in named.items():
            if t not in self.places:
                wrong.append(f"{t} is not a matrix of this model that may have an adapter")
                continue
            low, i = self.places[t]
            if a.shape[0] > self.max_rank or a.shape[1] != low.k or b.shape != (low.rows[i], a.shape[0]):
                wrong.append(f"{t}: A {tuple(a.shape)} and B {tuple(b.shape)} for a matrix [{low.rows[i]}, {low.k}] and ranks up to {self.max_rank}")
        if wrong:
            raise AdapterError(f"adapter {name!r}: " + "; ".join(wrong))
        per_stack: Dict[int, list] = {id(low): [None] * len(low.rows) for low in self.stacks}
        for t, ab in named.items():
            low, i = self.places[t]
            per_stack[id(low)][i] = ab
        for low in self.stacks:
            low.put(free[0], per_stack[id(low)], scale)
        self.names[name] = free[0]
        return free[0]

    def remove(self, name: str) -> None:
        del self.names[name]
