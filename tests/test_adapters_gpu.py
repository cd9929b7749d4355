"""Engines with adapters and filters (GPU): against the same model with the adapter written into its weights, in every way of running a
step, and draws against the definition.

Tolerances.  In float32 the two engines differ by roundings: sums of K products in another order, K 2^-24 relative each and a few of them a
layer, taken as 2^-13 of the logits' largest for these models of 2 to 4 layers with K up to 300.  In bfloat16 both round every
activation to 2^-8 of itself, but not the same values: 2^-3 of the logits' largest, and the mean a tenth of it."""

import importlib

import pytest
import torch

import adapter_helpers as H
import helpers

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def engine(folder, ps=16, dtype="float32", adapters=0, rank=16, graph=False, **kw):
    from prism_b200 import Engine, EngineConfig
    return Engine(folder, EngineConfig(kv_page_size=ps, num_pages=96, graph_batch_sizes=(1, 2, 4, 8), use_cuda_graph=graph, max_adapters=adapters,
                                       max_adapter_rank=rank, **kw), dtype=dtype)


def logits_of(eng, prompt, adapter=-1, cut=None):
    """Logits at every place of a prompt, fed whole or in portions of ``cut`` tokens."""
    from prism_b200.engine.batch import Segment
    rid = object()
    eng.runner.begin_request(rid)
    out, at = [], 0
    while at < len(prompt):
        n = min(cut or len(prompt), len(prompt) - at)
        out.append(eng.runner.step([Segment(rid, prompt[at:at + n], range(n), adapter)]).clone())
        at += n
    eng.runner.end_request(rid)
    eng.runner.check_errors()
    return torch.cat(out)


def prompt_of(eng, n, seed):
    return torch.randint(0, eng.model.spec.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def close(a, b, share):
    worst = b.abs().max()
    assert (a - b).abs().max() <= share * worst, ((a - b).abs().max() / worst).item()


FAMILIES = [("helpers", "A"), ("helpers", "B"), ("helpers", "C"), ("helpers", "D"), ("tagelorn_helpers", "Ex"), ("nivotar_helpers", "B"), ("zuvulorn_helpers", "Fx"),
            ("limatar_helpers", "B")]


@pytest.mark.parametrize("family,name", FAMILIES)
def test_an_adapter_is_what_it_is_in_the_weights(family, name):
    mod = importlib.import_module(family)
    folder = mod.model_folder(name)
    ps = (mod.TINY if family == "helpers" else mod.CONFIGS)[name][2]
    if not H.targets(folder):
        from prism_b200.weights.adapters import AdapterError
        with pytest.raises(AdapterError):
            engine(folder, ps, adapters=1)
        return
    one, two = H.adapter_folder(folder, 6, 9, 11), H.adapter_folder(folder, 16, 16, 12, only=lambda n: n.count("o") % 2 == 0, strength=2.0)
    eng = engine(folder, ps, adapters=3)
    plain = engine(folder, ps)
    p = prompt_of(eng, 40, 3)
    before = logits_of(eng, p)
    assert torch.equal(before, logits_of(plain, p))                # room for adapters changes nothing
    eng.load_adapter("one", one)
    eng.load_adapter("two", two)
    assert torch.equal(before, logits_of(eng, p))
    want1, want2 = (logits_of(engine(H.merged_folder(folder, d), ps), p) for d in (one, two))
    assert (want1 - before).abs().max() > 0.05 * before.abs().max()            # the adapter matters
    for cut in (None, 7, 1):
        close(logits_of(eng, p, 0, cut), want1, 2.0 ** -13)
        close(logits_of(eng, p, 1, cut), want2, 2.0 ** -13)


@pytest.mark.parametrize("name", ["A", "B", "D"])
def test_in_bfloat16(name):
    folder, ps = helpers.model_folder(name), helpers.TINY[name][2]
    d = H.adapter_folder(folder, 8, 8, 21, strength=0.5)
    eng = engine(folder, ps, "bfloat16", adapters=2)
    eng.load_adapter("none", H.adapter_folder(folder, 8, 8, 22, strength=0.0))
    eng.load_adapter("d", d)
    p = prompt_of(eng, 90, 5)
    want = logits_of(engine(H.merged_folder(folder, d), ps), p)
    base = logits_of(engine(folder, ps), p)
    for cut in (None, 33, 1):
        got = logits_of(eng, p, 1, cut)
        close(got, want, 2.0 ** -3)
        assert (got - want).abs().mean() <= 2.0 ** -3 / 10 * want.abs().max()
        assert (got - want).norm() < 0.5 * (got - base).norm()     # nearer to its own model than to the shared one
        close(logits_of(eng, p, 0, cut), base, 2.0 ** -3)


@pytest.mark.parametrize("weight_format", [None, "mxfp4"])
def test_beside_matrices_of_either_format(weight_format):
    """The adapters' part does not care how the shared product is made: over its own base it changes the logits as it does over the 4-bit one."""
    folder, ps = helpers.model_folder("D"), helpers.TINY["D"][2]
    d = H.adapter_folder(folder, 8, 8, 21, strength=0.5)
    eng = engine(folder, ps, "bfloat16", adapters=1, weight_format=weight_format)
    eng.load_adapter("d", d)
    p = prompt_of(eng, 50, 5)
    base, got = logits_of(eng, p), logits_of(eng, p, 0)
    change = logits_of(engine(H.merged_folder(folder, d), ps), p) - logits_of(engine(folder, ps), p)
    cos = torch.nn.functional.cosine_similarity((got - base).flatten(), change.flatten(), dim=0)
    assert cos > (0.97 if weight_format is None else 0.7), cos


@pytest.mark.parametrize("dtype,graph", [("float32", False), ("float32", True), ("bfloat16", True)])
def test_a_batch_of_requests_with_their_own(dtype, graph):
    """Continuous batching with portions, decode steps (graphs too) and several adapters: the same tokens as alone."""
    from prism_b200 import SamplingParams, SchedulerConfig
    folder = helpers.model_folder("B")
    folders = [H.adapter_folder(folder, r, 8, 30 + r, strength=1.5) for r in (2, 5, 16)]
    eng = engine(folder, 8, dtype, adapters=3, graph=graph, scheduler=SchedulerConfig(max_batch_tokens=40, max_num_seqs=6, prefill_chunk=24))
    for i, d in enumerate(folders):
        eng.load_adapter(f"a{i}", d)
    if graph:
        eng.warmup((1, 2))
    prompts = [prompt_of(eng, n, 40 + n) for n in (3, 50, 17, 30, 1, 24, 9)]
    names = ["a0", None, "a1", "a2", None, "a0", "a2"]
    sp = SamplingParams(max_new_tokens=12, ignore_eos=True)
    together = [r.token_ids for r in eng.generate(prompts, sp, names)]
    if dtype == "float32":
        for p, n, got in zip(prompts, names, together):
            merged = engine(folder if n is None else H.merged_folder(folder, folders[int(n[1])]), 8)
            # a near tie may fall either way: compare up to the first place where the two largest logits are close
            seq = list(p)
            for t in got:
                top = logits_of(merged, seq)[-1].topk(2)
                if top.values[0] - top.values[1] < 2.0 ** -9 * top.values[0].abs():
                    break
                assert t == top.indices[0].item()
                seq.append(t)
    assert [r.token_ids for r in eng.generate(prompts, sp, names)] == together
    with pytest.raises(ValueError, match="1 adapters for 2"):
        eng.generate(prompts[:2], sp, ["a0"])
    with pytest.raises(ValueError, match="no adapter 'zz'"):
        eng.generate(prompts[:1], sp, "zz")


def test_loading_and_unloading():
    from prism_b200 import SamplingParams
    folder = helpers.model_folder("A")
    eng = engine(folder, adapters=1)
    d1, d2 = H.adapter_folder(folder, 4, 8, 51, strength=2.0), H.adapter_folder(folder, 4, 8, 52, strength=2.0, only=lambda n: "q_proj" in n)
    eng.load_adapter("x", d1)
    with pytest.raises(ValueError, match="no room"):
        eng.load_adapter("y", d2)
    p = prompt_of(eng, 20, 1)
    first = logits_of(eng, p, 0)
    eng.scheduler.add_request(p, SamplingParams(max_new_tokens=2), 0)
    with pytest.raises(ValueError, match="in use"):
        eng.unload_adapter("x")
    eng.scheduler.run_to_completion()
    eng.unload_adapter("x")
    with pytest.raises(ValueError, match="no adapter"):
        eng.generate([p], adapters="x")
    eng.load_adapter("y", d2)                                      # in x's place, and nothing of x is left
    close(logits_of(eng, p, 0), logits_of(engine(H.merged_folder(folder, d2)), p), 2.0 ** -13)
    assert (logits_of(eng, p, 0) - first).abs().max() > 0.01
    plain = engine(folder)
    with pytest.raises(ValueError, match="no room for adapters"):
        plain.load_adapter("x", d1)
    with pytest.raises(ValueError, match="no room for adapters"):
        plain.generate([p], adapters="x")
    from prism_b200.engine.batch import Segment
    with pytest.raises(ValueError, match="beyond the 1"):
        eng.runner.begin_request("r")
        eng.runner.step([Segment("r", [1], [0], 1)])


# ---- filtered draws in an engine ------------------------------------------------------------------------------------------

def test_draws_by_filters_and_their_probabilities():
    """A request's tokens are the definition's at its own uniform numbers, whatever it shares its steps with, adapters among it."""
    from prism_b200 import SamplingParams
    from prism_b200.sampling.rng import uniform
    from test_sample_filtered_gpu import plain_row
    import numpy as np
    folder = helpers.model_folder("B")
    eng = engine(folder, 8, adapters=2, graph=True)
    eng.load_adapter("a", H.adapter_folder(folder, 4, 8, 61, strength=1.5))
    sps = [SamplingParams(max_new_tokens=9, temperature=0.9, seed=3, top_k=12, top_p=0.8, logprobs=True, ignore_eos=True),
           SamplingParams(max_new_tokens=12, temperature=0.7, seed=4, ignore_eos=True),
           SamplingParams(max_new_tokens=10, ignore_eos=True, logprobs=True),
           SamplingParams(max_new_tokens=11, temperature=1.3, seed=5, min_p=0.2, logprobs=True, ignore_eos=True),
           SamplingParams(max_new_tokens=6, ignore_eos=True)]
    prompts, names = [prompt_of(eng, n, 70 + n) for n in (5, 20, 9, 14, 3)], ["a", None, None, "a", None]
    first = eng.scheduler._next_id
    out = eng.generate(prompts, sps, names)
    for i, (p, sp, name, r) in enumerate(zip(prompts, sps, names, out)):
        assert len(r.token_ids) == sp.max_new_tokens and (r.logprobs is not None) == sp.logprobs
        if not sp.by_filters:
            continue
        seq = list(p)
        for j, t in enumerate(r.token_ids):
            row = logits_of(eng, seq, 0 if name else -1)[-1].cpu().numpy()
            u = np.float32(uniform(sp.seed or 0, first + i, j))
            tok, _, lp = plain_row(row, np.float32(sp.temperature), u, sp.top_k, np.float32(sp.top_p), np.float32(sp.min_p))
            assert t == tok and abs(r.logprobs[j] - lp) < 1e-3
            seq.append(t)
    # without filters a request draws as it does in an engine that has never heard of them
    eng2 = engine(folder, 8, graph=True)
    eng2.scheduler._next_id = first
    again = eng2.generate([prompts[0], prompts[1], prompts[2], prompts[3], prompts[4]], [SamplingParams(max_new_tokens=1)] + [sps[1]] + [SamplingParams(max_new_tokens=1)] * 3)
    assert again[1].token_ids == out[1].token_ids
