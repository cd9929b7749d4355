"""A loaded model's matrices in microscaled 4-bit floating point (``ops.Mxfp4``).

andre-fu/prism keeps every tensor as the file has it (engine/weight_pool.py:46-70).  Here
``EngineConfig.weight_format = "mxfp4"`` brings those matrices to 4 bits that their parts name in
``four_bit`` - the projections of attention and of the feed-forward layers, the experts among them: 17/32
of a byte a weight instead of two.  Embedding, head, router, norms and biases stay as they are, and so do the
matrices of parts that name none and those that a block has taken over from its parts to run them jointly.
"""

from __future__ import annotations

from math import prod
from typing import Dict, Iterator, Tuple

import torch

from .pool import StaticWeightPool

FORMATS = ("mxfp4",)


def check_weight_format(weight_format, act_bits: int, dtype: str = "bfloat16") -> None:
    if weight_format is not None and weight_format not in FORMATS:
        raise ValueError(f"weight_format {weight_format!r}: None (as the model file has them) or one of {FORMATS}")
    if act_bits not in (16, 4):
        raise ValueError(f"act_bits {act_bits!r}: products with 4-bit weights take activations of 16 or 4 bits")
    if weight_format is None and act_bits != 16:
        raise ValueError("act_bits 4 needs weights in 4 bits: weight_format='mxfp4'")
    if weight_format is not None and dtype != "bfloat16":
        raise ValueError(f"weight_format {weight_format!r} is for engines in bfloat16, this one computes in {dtype}")


def four_bit_params(part, path: str = "") -> Iterator[Tuple[str, object]]:
    """``(qualified name, part)`` of every parameter below ``part`` that may be kept in 4 bits."""
    own = {p.name for p in part.params()}
    for name in part.four_bit:
        if name in own:
            yield path + name, part
    for cname, child in part.children.items():
        yield from four_bit_params(child, f"{path}{cname}.")


def four_bit_share(model) -> float:
    """The share of ``model``'s parameters that may be kept in 4 bits: from nine tenths of a dense design to a twentieth of one
    whose blocks run their matrices jointly."""
    count = {q: prod(spec.shape) for q, spec in model.named_params() if not spec.alias_of}
    return sum(count[q] for q, _ in four_bit_params(model)) / sum(count.values())


def written_out_bytes(part) -> int:
    """The most that any part below ``part`` writes out of its matrices in 4 bits at once."""
    return max([part.written_out_bytes()] + [written_out_bytes(child) for child in part.children.values()])


def to_four_bits(model, pool: StaticWeightPool, device, dtype: torch.dtype, act_bits: int = 16) -> StaticWeightPool:
    """Bind ``model`` to a new pool with those matrices in 4 bits and everything else copied; ``pool`` may be dropped.  ``act_bits``:
    of the products with single matrices; layers of experts take activations of 16 bits in any case."""
    chosen: Dict[str, object] = {q: part for q, part in four_bit_params(model) if pool.tensors.get(q) is not None}
    # an absent parameter keeps its name without memory of its own (an alias or nothing), one filled with zeros is float32
    plan = [(q, spec, None if pool.tensors[q] is None or (spec.alias_of and pool.tensors[q] is pool.tensors.get(spec.alias_of))
             else pool.tensors[q].dtype) for q, spec in pool.specs.items() if q not in chosen]
    kept = StaticWeightPool(plan, device)
    for q, _, dt in plan:
        if dt is not None:
            kept.tensors[q].copy_(pool.tensors[q])
    for q, part in chosen.items():
        kept.specs[q] = pool.specs[q]
        kept.tensors[q] = part.in_four_bits(q.rsplit(".", 1)[-1], pool.tensors[q])
        for w in kept.tensors[q] if isinstance(kept.tensors[q], tuple) else (kept.tensors[q],):
            if w.dim() == 2:                     # a stack's products (ops.mxfp4_moe) take activations as they are
                w.act_bits = act_bits
            kept.total_bytes += w.nbytes
    model.bind(kept.tensors, torch.device(device), dtype)
    return kept
