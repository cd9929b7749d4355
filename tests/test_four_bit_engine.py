"""Models whose layers' matrices are kept in 4 bits: what is chosen, what is refused (CPU), and whole models against
the same models with the 4-bit values written out (GPU)."""

import importlib

import pytest
import torch

import helpers

FAMILIES = [("helpers", "D"), ("tagelorn_helpers", "Ex"), ("zuvulorn_helpers", "Fx"), ("nivotar_helpers", "B"), ("limatar_helpers", "B")]


def folder_of(family, name):
    return importlib.import_module(family).model_folder(name)


def page_size(family, name):
    mod = importlib.import_module(family)
    return (mod.TINY if family == "helpers" else mod.CONFIGS)[name][2]


# ---- what is chosen and refused --------------------------------------------------------------------------------------

def test_a_dense_model_s_layers_are_chosen_and_nothing_else():
    from prism_b200.model_registry import build_model
    from prism_b200.weights.four_bit import four_bit_params
    _, model = build_model(helpers.TINY_B)
    chosen = {q for q, _ in four_bit_params(model)}
    every = dict(model.named_params())
    assert chosen <= set(every)
    last = {}
    for q in every:
        last.setdefault(q.rsplit(".", 1)[-1], []).append(q)
    assert chosen == set(last["qkv_w"] + last["o_w"] + last["gate_up_w"] + last["down_w"])
    assert len(chosen) == 4 * helpers.TINY_B["num_hidden_layers"]


def test_experts_that_the_layer_does_not_take_are_left_alone():
    from prism_b200.parts.base import PartSpec, build_part

    def moe(**kw):
        args = dict(hidden_size=64, intermediate_size=32, experts=8, top=2)
        args.update(kw)
        return build_part("feed_forward", PartSpec("moe", args))
    assert moe().four_bit == ("gate_up_w", "down_w")
    assert moe(gated=False, activation="relu2").four_bit == ()
    assert moe(identity=2, scale_input=False).four_bit == ()
    assert moe(experts=512).four_bit == ()
    assert moe(experts=64, top=17).four_bit == ()


@pytest.mark.parametrize("kw", [dict(weight_format="int4"), dict(act_bits=4), dict(weight_format="mxfp4", act_bits=8), dict(act_bits=0)])
def test_configurations_that_make_no_sense_are_refused(kw):
    from prism_b200 import EngineConfig
    with pytest.raises(ValueError):
        EngineConfig(**kw)


def test_an_engine_in_float32_is_refused():
    from prism_b200 import Engine, EngineConfig
    with pytest.raises(ValueError, match="bfloat16"):
        Engine("nowhere", EngineConfig(weight_format="mxfp4"), dtype="float32")


def test_the_command_takes_the_format():
    from prism_b200.cli import build_parser
    args = build_parser().parse_args(["--model", "x", "--weight-format", "mxfp4", "--act-bits", "4"])
    assert args.weight_format == "mxfp4" and args.act_bits == 4
    assert build_parser().parse_args([]).weight_format is None


# ---- whole models ----------------------------------------------------------------------------------------------------

def engine(folder, ps, dtype="bfloat16", **kw):
    from prism_b200 import Engine, EngineConfig
    return Engine(folder, EngineConfig(kv_page_size=ps, num_pages=64, graph_batch_sizes=(1, 2, 4), use_cuda_graph=kw.pop("graph", False), **kw),
                  dtype=dtype)


def write_out(four, other):
    """The 4-bit values of ``four``'s matrices into the same parameters of ``other``; how many."""
    from prism_b200 import ops
    n = 0
    for q, w in four.pool.tensors.items():
        place = other.pool.tensors[q]
        if isinstance(w, tuple):
            E, I, H = w[0].shape
            place = place.view(E, 2, I, H)
            for i in range(2):
                place[:, i].copy_(w[i].dequantize(torch.float32))
        elif isinstance(w, ops.Mxfp4):
            place.view(w.shape).copy_(w.dequantize(torch.float32))
        else:
            continue
        n += 1
    return n


def logits(eng, seqs, cuts):
    """Logits of every position: each sequence's first tokens in one step, then pieces of ``cuts`` tokens."""
    from prism_b200.engine.batch import Segment
    at, rows = {k: 0 for k in seqs}, {k: [] for k in seqs}
    for k in seqs:
        eng.runner.begin_request(k)
    for cut in cuts:
        segs = []
        for k, seq in seqs.items():
            part = seq[at[k]:at[k] + (cut if cut else len(seq) - 4)]
            if part:
                segs.append(Segment(k, part, list(range(len(part)))))
                at[k] += len(part)
        out = eng.runner.step(segs)
        i = 0
        for s in segs:
            rows[s.req_id].append(out[i:i + len(s.tokens)].clone())
            i += len(s.tokens)
    eng.runner.check_errors()
    assert all(at[k] == len(seqs[k]) for k in seqs)
    return torch.cat([r for k in seqs for r in rows[k]]).double()


def rms(t):
    return float(t.pow(2).mean().sqrt())


@pytest.mark.gpu
@pytest.mark.parametrize("family,name", FAMILIES)
def test_a_model_in_four_bits_is_the_model_with_those_values(family, name):
    """Against a float32 engine with the 4-bit values written out: 16-bit activations are rounded where a bfloat16 engine
    with those values rounds them, and a product's two 8-bit terms hold them to about one rounding more, so the error may be
    twice that engine's (and 2^-8 of the logits, where that engine has next to none)."""
    folder, ps = folder_of(family, name), page_size(family, name)
    four, b16, f32 = engine(folder, ps, weight_format="mxfp4"), engine(folder, ps), engine(folder, ps, "float32")
    vocab = four.model.spec.vocab_size
    seqs = {"a": helpers.random_tokens(vocab, 73, 5), "b": helpers.random_tokens(vocab, 11, 6)}
    n = write_out(four, b16)
    assert n == write_out(four, f32) > 0
    cuts = (0, 1, 1, 2)
    want = logits(f32, seqs, cuts)
    own, ref = rms(logits(four, seqs, cuts) - want), rms(logits(b16, seqs, cuts) - want)
    assert own <= 2 * ref + 2 ** -8 * rms(want), (own, ref, rms(want))


@pytest.mark.gpu
def test_four_bit_activations_in_a_model(monkeypatch):
    """``act_bits`` 4, against the same engine with its products written out (x to 4 bits and back, float64 sums): results
    differ by a rounding to bfloat16 here and there, each worth at most one step of a 4-bit activation."""
    from prism_b200 import ops
    folder, ps = folder_of("helpers", "D"), page_size("helpers", "D")
    four = engine(folder, ps, weight_format="mxfp4", act_bits=4)
    seqs = {"a": helpers.random_tokens(four.model.spec.vocab_size, 73, 5), "b": helpers.random_tokens(four.model.spec.vocab_size, 11, 6)}
    got = logits(four, seqs, (0, 1, 1, 2))
    calls = []

    def plain(x, w, bias=None, out=None, out_dtype=None, act_bits=16):
        calls.append(act_bits)
        y = ops.mxfp4_quantize(x).dequantize(torch.float32).double() @ w.dequantize(torch.float32).double().t()
        y = (y if bias is None else y + bias.double()).to(out_dtype or (x.dtype if out is None else out.dtype))
        return y if out is None else out.copy_(y)
    monkeypatch.setattr(ops, "mxfp4_linear", plain)
    for k in seqs:
        four.runner.end_request(k)
    want = logits(four, seqs, (0, 1, 1, 2))
    assert set(calls) == {4} and len(calls) == 4 * 4 * len(four.model.layers)
    assert rms(got - want) <= 0.03 * rms(want)


@pytest.mark.gpu
@pytest.mark.parametrize("family,name", [("helpers", "D"), ("tagelorn_helpers", "Ex")])
def test_generation_replays_and_repeats(family, name):
    """Tokens of an engine with decode graphs are those of one without, and come again; the pool has shrunk."""
    from prism_b200 import SamplingParams
    folder, ps = folder_of(family, name), page_size(family, name)
    eager, graphs = engine(folder, ps, weight_format="mxfp4"), engine(folder, ps, weight_format="mxfp4", graph=True)
    prompts = [helpers.random_tokens(eager.model.spec.vocab_size, n, 70 + n) for n in (1, 9, 40)]
    sp = SamplingParams(max_new_tokens=9, ignore_eos=True)
    a = [r.token_ids for r in eager.generate(prompts, sp)]
    assert [r.token_ids for r in graphs.generate(prompts, sp)] == a and graphs.runner.graph_kernel_launches > 0
    assert [r.token_ids for r in graphs.generate(prompts, sp)] == a
    assert eager.pool.total_bytes < engine(folder, ps).pool.total_bytes


@pytest.mark.gpu
def test_values_of_a_stack_into_a_place_of_their_own():
    from prism_b200 import ops
    x = torch.randn(3, 130, 264, device="cuda").bfloat16()
    w = ops.mxfp4_quantize(x)
    place = torch.full((3, 2, 130, 264), 7.0, dtype=torch.bfloat16, device="cuda")
    assert w.dequantize(out=place[:, 1]).data_ptr() == place[:, 1].data_ptr()
    assert torch.equal(place[:, 1], w.dequantize()) and bool((place[:, 0] == 7).all())
    for bad in (place[:, :, :, :200], place[:, 1].transpose(1, 2), place[:2, 1], place[:, 1].half()):
        with pytest.raises(ops.KernelError):
            w.dequantize(out=bad)
