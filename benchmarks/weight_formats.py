"""Decode steps and prompts of one engine with its weights as they are and in 4 bits (with activations of 16 and 4 bits): random
weights, a dense model and one of experts.

    python benchmarks/weight_formats.py [dense] [experts]

A line per format: gigabytes of weights, the share of the parameters in 4 bits, milliseconds a decode step of 1, 16 and 64
requests behind prompts of 256 tokens (the difference of two generations of different length, by the host's clock; all weights are
read every step and are larger than L2), and of a prompt of 65, 512 and 2,048 tokens.
"""

import gc
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from prism_b200 import Engine, EngineConfig, SamplingParams, SchedulerConfig  # noqa: E402
from prism_b200.weights.four_bit import four_bit_share  # noqa: E402

from bench import BASE, SHAPES  # noqa: E402

FORMATS = ((None, 16), ("mxfp4", 16), ("mxfp4", 4))


def experts_config(width=2048, layers=8, ff=1024, experts=64, top=8):
    attention = dict(type="attention", mixer=dict(heads=16, kv_heads=4, dim=128, scale=128 ** -0.5, rot=dict(base=10000.0, dims=128)),
                     mlp=dict(kind="moe", expert=dict(ff=ff), router=dict(experts=experts, top=top)))
    return dict(architecture="Zuvulorn", vocab=32768, width=width, norm=dict(eps=1e-6), layers=[attention] * layers)


def best(f, times):
    out = []
    for _ in range(times):
        torch.cuda.synchronize()
        t = time.perf_counter()
        f()
        torch.cuda.synchronize()
        out.append(time.perf_counter() - t)
    return min(out) * 1e3


def measure(name, config):
    for fmt, bits in FORMATS:
        ec = EngineConfig(kv_page_size=64, num_pages=64 * 10, graph_batch_sizes=(1, 16, 64), max_seq_len=4096, weight_format=fmt, act_bits=bits,
                          scheduler=SchedulerConfig(8192, 64, 2048))
        eng = Engine(None, ec, dtype="bfloat16", config=config, random_seed=0)
        vocab, g = eng.model.spec.vocab_size, torch.Generator().manual_seed(1)

        def prompts(count, length):
            return [torch.randint(0, vocab, (length,), generator=g).tolist() for _ in range(count)]

        def generate(ps, n):
            eng.generate(ps, SamplingParams(max_new_tokens=n, ignore_eos=True))
        line = [f"{name} {'16-bit weights' if fmt is None else f'4-bit weights, {bits}-bit activations'}: {eng.pool.total_gb:.2f} GB"]
        if fmt is not None:
            line.append(f"{four_bit_share(eng.model):.0%} of the parameters in 4 bits")
        for batch in (1, 16, 64):
            ps = prompts(batch, 256)
            generate(ps, 8)
            step = (best(lambda: generate(ps, 84), 2) - best(lambda: generate(ps, 20), 2)) / 64
            line.append(f"decode {batch} {step:.3f} ms")
        for length in (65, 512, 2048):
            ps = prompts(1, length)
            generate(ps, 1)
            line.append(f"prompt {length} {best(lambda: generate(ps, 1), 5):.2f} ms")
        print(", ".join(line), flush=True)
        del eng
        gc.collect()
        torch.cuda.empty_cache()


if __name__ == "__main__":
    which = sys.argv[1:] or ["dense", "experts"]
    if "dense" in which:
        measure("dense", dict(BASE, **SHAPES["7b"]))
    if "experts" in which:
        measure("experts", experts_config())
