"""Adapter folders for the tests' tiny models, and model folders with an adapter written into the weights."""

import json
import os
import shutil
import tempfile

import torch
from safetensors.torch import load_file, save_file


def targets(folder):
    """``{file tensor: shape}`` of the matrices of the model in ``folder`` that may have adapters."""
    from prism_b200.weights.adapters import adaptable_params
    from prism_b200.weights.loader import find_shards, read_config_json, read_safetensors_header
    from prism_b200.model_registry import build_model
    shapes = {}
    for p in find_shards(folder):
        shapes.update({n: m[0] for n, m in read_safetensors_header(p).items()})
    _, model = build_model(read_config_json(folder), shapes)
    return {s.name: tuple(s.shape) for _, _, spec in adaptable_params(model) for s in spec.sources}


def adapter_folder(folder, rank, alpha, seed, only=None, strength=1.0, dtype=torch.float32):
    """A random adapter for the model in ``folder``: for every matrix that may have one, or those whose name ``only`` accepts."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, (n, k) in sorted(targets(folder).items()):
        if only is not None and not only(name):
            continue
        module = name.removesuffix(".weight")
        out[f"base_model.model.{module}.lora_A.weight"] = (torch.randn(rank, k, generator=g) * k ** -0.5).to(dtype)
        out[f"base_model.model.{module}.lora_B.weight"] = (torch.randn(n, rank, generator=g) * strength * rank ** -0.5).to(dtype)
    d = tempfile.mkdtemp(prefix="prism_adapter_")
    save_file(out, os.path.join(d, "adapter_model.safetensors"))
    with open(os.path.join(d, "adapter_config.json"), "w") as f:
        json.dump(dict(peft_type="LORA", r=rank, lora_alpha=alpha, bias="none", target_modules=[]), f)
    return d


def merged_folder(folder, adapter):
    """The model of ``folder`` with ``W + scale B A`` in the place of W, in float32."""
    from prism_b200.weights.adapters import read_adapter_folder
    tensors, scale = read_adapter_folder(adapter)
    d = tempfile.mkdtemp(prefix="prism_merged_")
    for f in os.listdir(folder):
        if f.endswith(".safetensors"):
            t = {n: v.float() if v.is_floating_point() else v for n, v in load_file(os.path.join(folder, f)).items()}
            for n, (a, b) in tensors.items():
                n = n if n in t else n + ".weight"
                if n in t:
                    t[n] = (t[n].double() + scale * b.double() @ a.double()).float()
            save_file(t, os.path.join(d, f))
        else:
            shutil.copy(os.path.join(folder, f), d)
    return d
