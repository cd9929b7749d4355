"""Decode steps and prompts of the 7B shape with random weights: requests alike, with a low-rank adapter each, and with filtered draws.

    python benchmarks/request_settings.py [rank]

Milliseconds a decode step of 1, 16 and 64 requests behind prompts of 256 tokens (the difference of two generations of different length, by
the host's clock) and of a prompt of 2,048 tokens; adapters (of ``rank``, 16 if it is not given) beside every matrix that may have one.
"""

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from prism_b200 import Engine, EngineConfig, SamplingParams, SchedulerConfig  # noqa: E402

from bench import BASE, SHAPES  # noqa: E402
from benchmarks.weight_formats import best  # noqa: E402

FILTERS = dict(temperature=0.8, top_k=50, top_p=0.95)


def main(rank=16, count=64):
    ec = EngineConfig(kv_page_size=64, num_pages=64 * 10, graph_batch_sizes=(1, 16, 64), max_seq_len=4096, max_adapters=count, max_adapter_rank=rank,
                      scheduler=SchedulerConfig(8192, 64, 2048))
    eng = Engine(None, ec, dtype="bfloat16", config=dict(BASE, **SHAPES["7b"]), random_seed=0)
    g, on_device = torch.Generator().manual_seed(1), torch.Generator(device=eng.device).manual_seed(2)
    for i in range(count):
        eng.adapters.add(f"a{i}", {n: (torch.randn(rank, low.k, generator=on_device, device=eng.device) * low.k ** -0.5,
                                       torch.randn(low.rows[s], rank, generator=on_device, device=eng.device) * 0.02)
                                   for n, (low, s) in eng.adapters.places.items()}, 1.0)
    print(f"{eng.pool.total_gb:.2f} GB of weights, {eng.adapters.nbytes / 1e9:.2f} GB for {count} adapters of rank {rank}", flush=True)
    for name, settings, adapted in (("greedy", {}, False), ("an adapter each", {}, True), ("top-k and top-p", FILTERS, False),
                                    ("logprobs, top-p 0.95 alone", dict(temperature=0.8, top_p=0.95, logprobs=True), False), ("all of it", FILTERS, True)):
        def generate(ps, n):
            eng.generate(ps, SamplingParams(max_new_tokens=n, ignore_eos=True, **settings), [f"a{i % count}" for i in range(len(ps))] if adapted else None)
        line = []
        for batch in (1, 16, 64):
            ps = [torch.randint(0, eng.model.spec.vocab_size, (256,), generator=g).tolist() for _ in range(batch)]
            generate(ps, 8)
            line.append(f"decode {batch} {(best(lambda: generate(ps, 84), 2) - best(lambda: generate(ps, 20), 2)) / 64:.3f} ms")
        ps = [torch.randint(0, eng.model.spec.vocab_size, (2048,), generator=g).tolist()]
        generate(ps, 1)
        line.append(f"prompt 2048 {best(lambda: generate(ps, 1), 5):.2f} ms")
        print(f"{name}: " + ", ".join(line), flush=True)


if __name__ == "__main__":
    main(*(int(a) for a in sys.argv[1:]))
