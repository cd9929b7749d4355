"""Models in 4 bits whose parts mix formats: what a part hands to another (CPU), and whole models against the same models
with the 4-bit values written out (GPU)."""

import pytest
import torch

import helpers
import limatar_helpers as LH
from test_four_bit_engine import engine, folder_of, logits, page_size, rms, write_out


def four_bits(N, K):
    from prism_b200 import ops
    return ops.Mxfp4(torch.zeros(N, -(-K // 128) * 64, dtype=torch.uint8), torch.zeros(-(-N // 128), -(-K // 128), 512, dtype=torch.uint8), K)


def test_a_shared_expert_in_four_bits_runs_on_its_own(monkeypatch):
    """Experts that stay in bfloat16 run their shared expert with them only where it has stayed in bfloat16 too."""
    from prism_b200 import ops
    from prism_b200.parts.base import PartSpec, build_part
    H, I, E = 64, 32, 300
    part = build_part("feed_forward", PartSpec("moe", dict(hidden_size=H, intermediate_size=I, experts=E, top=2, shared=PartSpec(
        "swiglu", dict(hidden_size=H, intermediate_size=I)))))
    assert part.four_bit == () and part.shared.four_bit
    part.w = {"router_w": torch.zeros(E, H), "gate_up_w": torch.zeros(E * 2 * I, H), "down_w": torch.zeros(E * H, I)}
    part.choice = None
    calls = []
    monkeypatch.setattr(ops, "linear", lambda x, w, *a, **k: torch.zeros(x.shape[0], w.shape[0]))
    monkeypatch.setattr(ops, "moe_feed_forward", lambda ctx, x, z, gu, dn, top, *a, extra_planes=0, shared=None, **k: calls.append(
        (extra_planes, shared)) or torch.zeros(top + extra_planes + (shared is not None), x.shape[0], H))
    monkeypatch.setattr(part.shared, "forward_to", lambda ctx, x, out: calls.append(out.shape))
    x = torch.zeros(3, H)
    part.shared.w = {"gate_up_w": torch.zeros(2 * I, H), "down_w": torch.zeros(H, I)}
    assert part.forward(None, x).shape == (3, 3, H) and calls[0][0] == 0 and calls[0][1] is not None and len(calls) == 1
    calls.clear()
    part.shared.w = {"gate_up_w": four_bits(2 * I, H), "down_w": four_bits(H, I)}
    assert part.forward(None, x).shape == (3, 3, H)
    assert calls == [(1, None), (3, H)]


def fake_pool(model, dtype=torch.bfloat16):
    from prism_b200.weights.pool import StaticWeightPool
    return StaticWeightPool([(q, spec, dtype) for q, spec in model.named_params()], "cpu")


def quantise_on_the_cpu(x):
    from prism_b200 import ops
    q = four_bits(x.shape[-2], x.shape[-1])
    return q if x.dim() == 2 else ops.Mxfp4(torch.stack([q.codes] * x.shape[0]), torch.stack([q.scales] * x.shape[0]), x.shape[-1])


def test_experts_keep_sixteen_bit_activations(monkeypatch):
    """``act_bits`` 4 is for products with a matrix; a layer of experts takes its activations as they are, and its stacks say so."""
    from prism_b200 import ops
    from prism_b200.cli import build_parser
    from prism_b200.model_registry import build_model
    from prism_b200.weights import four_bit

    monkeypatch.setattr(ops, "mxfp4_quantize", quantise_on_the_cpu)
    _, model = build_model(LH.CONFIGS["B"][0])
    pool = four_bit.to_four_bits(model, fake_pool(model), "cpu", torch.bfloat16, 4)
    seen = set()
    for w in pool.tensors.values():
        for q in w if isinstance(w, tuple) else (w,):
            if isinstance(q, ops.Mxfp4):
                seen.add((q.dim(), q.act_bits))
    assert seen == {(2, 4), (3, 16)}
    assert "experts" in " ".join(a.help or "" for a in build_parser()._actions if "--act-bits" in a.option_strings)


@pytest.mark.parametrize("module,name,low,high", [("helpers", "D", 0.9, 1.0), ("limatar_helpers", "B", 0.5, 0.6), ("dolezen_helpers", "Y", 0.0, 0.1)])
def test_the_share_in_four_bits_is_known(module, name, low, high):
    """Part of some designs' parameters is never taken; how much is for the user to see."""
    import importlib
    from prism_b200.model_registry import build_model
    from prism_b200.weights.four_bit import four_bit_params, four_bit_share
    mod = importlib.import_module(module)
    _, model = build_model((mod.TINY if module == "helpers" else mod.CONFIGS)[name][0])
    share = four_bit_share(model)
    count = {q: torch.Size(spec.shape).numel() for q, spec in model.named_params() if not spec.alias_of}
    assert low < share < high and share == sum(count[q] for q, _ in four_bit_params(model)) / sum(count.values())


def test_the_cache_s_budget_leaves_room_for_experts_written_out(monkeypatch):
    """A step of more than 64 tokens writes a layer's experts out in bfloat16; the largest layer's are no room for keys."""
    from types import SimpleNamespace
    from prism_b200 import EngineConfig, ops
    from prism_b200.engine import llm
    from prism_b200.model_registry import build_model
    from prism_b200.weights import four_bit
    budgets = []
    monkeypatch.setattr(llm, "pool_sizes", lambda *a: budgets.append(a[-1]))
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (10 ** 9, 2 * 10 ** 9))
    monkeypatch.setattr(ops, "mxfp4_quantize", quantise_on_the_cpu)
    _, model = build_model(LH.CONFIGS["B"][0])
    pool = fake_pool(model)
    model.bind(pool.tensors, "cpu", torch.bfloat16)
    self = SimpleNamespace(model=model, device="cpu", dtype=torch.bfloat16)
    llm.Engine._pages_per_group(self, EngineConfig(), 128)
    four_bit.to_four_bits(model, pool, "cpu", torch.bfloat16)
    llm.Engine._pages_per_group(self, EngineConfig(), 128)
    written_out = 2 * 8 * 3 * 128 * 64                            # the larger of the two layers: 8 experts of 3 x 64 x 128
    assert budgets == [0.7 * 10 ** 9, 0.7 * (10 ** 9 - written_out)]


# ---- whole models ----------------------------------------------------------------------------------------------------

MANY = LH.model(120, 64, [
    LH.layer("latent", LH.latent(2, 16, 8, 16, 24, 32), LH.moe(16, 260, 260, shared=16)),
    LH.layer("retention", LH.retain(2, 16, 16, (0.9, 0.98)), LH.moe(16, 258, 258, shared=24)),
])


def compare(family, name, **kw):
    """As ``test_a_model_in_four_bits_is_the_model_with_those_values``: twice the bfloat16 engine's error and 2^-8 of the logits."""
    folder, ps = folder_of(family, name), page_size(family, name)
    four, b16, f32 = engine(folder, ps, weight_format="mxfp4", **kw), engine(folder, ps), engine(folder, ps, "float32")
    vocab = four.model.spec.vocab_size
    seqs = {"a": helpers.random_tokens(vocab, 73, 5), "b": helpers.random_tokens(vocab, 11, 6)}
    n = write_out(four, b16)
    assert n == write_out(four, f32) > 0
    cuts = (0, 1, 1, 2)
    want = logits(f32, seqs, cuts)
    own, ref = rms(logits(four, seqs, cuts) - want), rms(logits(b16, seqs, cuts) - want)
    assert own <= 2 * ref + 2 ** -8 * rms(want), (own, ref, rms(want))
    return four


@pytest.mark.gpu
def test_a_model_of_many_experts_with_shared_ones(monkeypatch):
    monkeypatch.setitem(LH.CONFIGS, "many", (MANY, 21, 16))
    four = compare("limatar_helpers", "many")
    from prism_b200 import ops
    kept = [isinstance(w, (ops.Mxfp4, tuple)) for q, w in four.pool.tensors.items() if q.endswith("gate_up_w")]
    assert sorted(kept) == [False, False, True, True]            # the experts', the shared ones'


@pytest.mark.gpu
def test_the_matrices_of_the_file_are_given_back_before_the_cache_is_sized(monkeypatch):
    """What the 16-bit weights held is the device's again, not torch's, when the cache's share of the free memory is taken."""
    import gc
    from prism_b200 import Engine, EngineConfig
    raw = dict(helpers.TINY_B, hidden_size=1024, head_dim=64, intermediate_size=8192, num_hidden_layers=8)
    held = []
    sized = Engine._pages_per_group
    monkeypatch.setattr(Engine, "_pages_per_group", lambda self, *a: held.append(torch.cuda.memory_reserved()) or sized(self, *a))
    gc.collect()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_reserved()
    four = Engine(None, EngineConfig(kv_page_size=16, num_pages=8, use_cuda_graph=False, weight_format="mxfp4"), config=raw, random_seed=1)
    matrices = 8 * 2 * 3 * 1024 * 8192                            # bytes of the feed-forwards' in bfloat16
    assert four.pool.total_bytes < matrices // 2 and held[0] - before < matrices // 2


@pytest.mark.gpu
@pytest.mark.parametrize("family,name", [("dolezen_helpers", "X"), ("dolezen_helpers", "Y"), ("pofazen_helpers", "P"), ("pofazen_helpers", "Q")])
def test_the_other_families(family, name):
    compare(family, name)


@pytest.mark.gpu
def test_a_model_with_experts_and_four_bit_activations():
    """``act_bits`` 4 in a model of both: the products of single matrices take it and the layers of experts do not, so the
    logits are those of the same engine whose dense products are written out with activations brought to 4 bits."""
    from prism_b200 import ops
    four = engine(folder_of("limatar_helpers", "Bx"), page_size("limatar_helpers", "Bx"), weight_format="mxfp4", act_bits=4)
    seqs = {"a": helpers.random_tokens(four.model.spec.vocab_size, 40, 5), "b": helpers.random_tokens(four.model.spec.vocab_size, 11, 6)}
    got = logits(four, seqs, (0, 1, 1, 2))
    for k in seqs:
        four.runner.end_request(k)
    dense, layers, exact, moe = [], [], ops.mxfp4_linear, ops.mxfp4_moe

    def product(x, w, bias=None, out=None, out_dtype=None, act_bits=16):
        dense.append(act_bits)
        return exact(ops.mxfp4_quantize(x).dequantize(), w, bias, out, out_dtype, 16)

    with pytest.MonkeyPatch.context() as m:
        m.setattr(ops, "mxfp4_linear", product)
        m.setattr(ops, "mxfp4_moe", lambda *a, **k: layers.append(1) or moe(*a, **k))
        want = logits(four, seqs, (0, 1, 1, 2))
    assert set(dense) == {4} and layers
    assert rms(got - want) <= 0.03 * rms(want)
