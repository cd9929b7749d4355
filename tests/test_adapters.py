"""Adapters and filtered sampling on the host: what is chosen, read, refused, and carried along (CPU)."""

import json
import os

import pytest
import torch
from safetensors.torch import load_file, save_file

import adapter_helpers as H
import helpers
from prism_b200 import EngineConfig, SamplingParams, ops
from prism_b200.engine.batch import BatchLayout, Segment, StepContext, pack_batch
from prism_b200.weights import adapters as A


def bound_model(name="B"):
    """A tiny model whose matrices are zeros on the CPU."""
    from prism_b200.model_registry import build_model
    _, model = build_model(helpers.TINY[name][0])
    model.bind({q: torch.zeros(s.shape) for q, s in model.named_params()}, torch.device("cpu"), torch.float32)
    return model


def test_a_dense_model_s_projections_may_have_adapters():
    t = H.targets(helpers.model_folder("B"))
    layers = helpers.TINY_B["num_hidden_layers"]
    kinds = {n.split(".")[-2] for n in t}
    assert kinds == {"q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"} and len(t) == 7 * layers


def test_experts_shared_or_not_have_none():
    import zuvulorn_helpers
    for name in H.targets(zuvulorn_helpers.model_folder("Fx")):
        assert "expert" not in name and ".e0." not in name


@pytest.mark.parametrize("kw", [dict(max_adapters=-1), dict(max_adapters=1.5), dict(max_adapters=1, max_adapter_rank=0), dict(max_adapter_rank=129)])
def test_room_that_makes_no_sense_is_refused(kw):
    with pytest.raises(ValueError):
        EngineConfig(**kw)


@pytest.mark.parametrize("kw", [dict(top_k=-1), dict(top_k=1.5), dict(top_p=0.0), dict(top_p=1.5), dict(top_p=-0.1), dict(top_p=float("nan")), dict(min_p=-0.1),
                                dict(min_p=1.1), dict(min_p=float("nan")), dict(top_k=2 ** 31)])
def test_filters_that_make_no_sense_are_refused(kw):
    with pytest.raises(ValueError):
        SamplingParams(temperature=1.0, **kw)


def test_which_rows_go_by_filters():
    S = SamplingParams
    assert not S().by_filters and not S(temperature=1.0).by_filters and not S(top_k=5).by_filters and not S(top_p=0.5, min_p=0.1).by_filters
    assert S(temperature=1.0, top_k=5).by_filters and S(temperature=1.0, top_p=0.9).by_filters and S(temperature=1.0, min_p=0.1).by_filters
    assert S(logprobs=True).by_filters


def test_the_command_takes_them():
    from prism_b200.cli import build_parser
    args = build_parser().parse_args(["--model", "x", "--top-k", "4", "--top-p", "0.9", "--min-p", "0.05", "--adapter", "d"])
    assert (args.top_k, args.top_p, args.min_p, args.adapter) == (4, 0.9, 0.05, "d")
    args = build_parser().parse_args([])
    assert (args.top_k, args.top_p, args.min_p, args.adapter) == (0, 1.0, 0.0, None)


# ---- folders ---------------------------------------------------------------------------------------------------------

def test_an_adapter_folder_is_read():
    folder = helpers.model_folder("B")
    d = H.adapter_folder(folder, 3, 12, 1, dtype=torch.bfloat16)
    assert A.read_adapter_config(d) == (3, 4.0)
    tensors, scale = A.read_adapter_folder(d)
    assert scale == 4.0 and {n + ".weight" for n in tensors} == set(H.targets(folder))
    for name, (a, b) in tensors.items():
        n, k = H.targets(folder)[name + ".weight"]
        assert a.shape == (3, k) and b.shape == (n, 3)
    cfg = json.load(open(os.path.join(d, "adapter_config.json")))
    json.dump(dict(cfg, use_rslora=True, r=4), open(os.path.join(d, "adapter_config.json"), "w"))
    assert A.read_adapter_config(d) == (4, 6.0)
    with pytest.raises(A.AdapterError, match="rank 3"):
        A.read_adapter_folder(d)


@pytest.mark.parametrize("change", [dict(use_dora=True), dict(bias="all"), dict(rank_pattern={"q_proj": 4}), dict(modules_to_save=["lm_head"]), dict(r=0), dict(r=None),
                                    dict(lora_alpha=None), dict(lora_alpha=float("inf")), dict(peft_type="IA3"), dict(r=True)])
def test_a_folder_with_another_formula_is_refused(change):
    d = H.adapter_folder(helpers.model_folder("B"), 3, 12, 1)
    path = os.path.join(d, "adapter_config.json")
    cfg = json.load(open(path))
    json.dump(dict(cfg, **change), open(path, "w"))
    with pytest.raises(A.AdapterError):
        A.read_adapter_config(d)


def test_broken_folders_are_refused():
    with pytest.raises(A.AdapterError, match="adapter_config"):
        A.read_adapter_folder("/nonexistent")
    d = H.adapter_folder(helpers.model_folder("B"), 3, 12, 1)
    path = os.path.join(d, "adapter_model.safetensors")
    t = {n: v.clone() for n, v in load_file(path).items()}          # the file is written over
    half = sorted(t)[0]
    for broken, say in (({k: v for k, v in t.items() if k != half}, "only its"), (dict(t, **{"x.bias": torch.zeros(3)}), "unexpected"), ({}, "no tensors"),
                        (dict(t, **{half: t[half].int()}), "float32"), (dict(t, **{half: t[half][0].contiguous()}), "matrix")):
        save_file(broken, path)
        with pytest.raises(A.AdapterError, match=say):
            A.read_adapter_folder(d)
    os.remove(path)
    with pytest.raises(A.AdapterError, match="adapter_model"):
        A.read_adapter_folder(d)


# ---- the set ----------------------------------------------------------------------------------------------------------

def test_adapters_find_their_places():
    model = bound_model()
    s = A.AdapterSet(model, 2, 5, "cpu", torch.float32)
    folder = helpers.model_folder("B")
    d = H.adapter_folder(folder, 5, 10, 3, only=lambda n: "k_proj" in n or "down_proj" in n)
    tensors, scale = A.read_adapter_folder(d)
    assert s.load("one", d) == 0 and s.number("one") == 0
    w = model.layers[1].mixer.w["qkv_w"]
    assert type(w) is ops.Adapted and w.shape == w.base.shape and ops.in_use(w) is w.base
    a, b = tensors["model.layers.1.self_attn.k_proj"]
    q = w.low.rows[0]
    assert torch.equal(w.low.a[0, 1, :5, :w.low.k], a) and torch.equal(w.low.b[0, q:q + w.low.rows[1], :5], b) and w.low.scale.tolist() == [2.0, 0.0]
    assert w.low.a[0, 0].count_nonzero() == 0 and w.low.a[0, 2].count_nonzero() == 0 and w.low.b[1].count_nonzero() == 0
    assert model.layers[0].mixer.w["o_w"].low.a.count_nonzero() == 0 and s.nbytes > 0
    s.add("two", {}, 1.0)
    with pytest.raises(A.AdapterError, match="no room"):
        s.add("three", {}, 1.0)
    with pytest.raises(A.AdapterError, match="loaded already"):
        s.add("two", {}, 1.0)
    s.remove("one")
    with pytest.raises(A.AdapterError, match="no adapter"):
        s.number("one")
    assert s.add("three", {}, 1.0) == 0 and w.low.a[0].count_nonzero() == 0
    s.step.ids = torch.zeros(1, dtype=torch.int32)
    assert ops.in_use(w) is w


def test_what_does_not_fit_is_refused_and_leaves_nothing():
    s = A.AdapterSet(bound_model(), 1, 4, "cpu", torch.float32)
    folder = helpers.model_folder("B")
    with pytest.raises(A.AdapterError, match="ranks up to 4"):
        s.load("a", H.adapter_folder(folder, 5, 10, 3))
    with pytest.raises(A.AdapterError, match="not a matrix"):
        s.add("a", {"lm_head.weight": (torch.zeros(2, 96), torch.zeros(320, 2))}, 1.0)
    two = torch.zeros(2, 96), torch.zeros(96, 2)
    with pytest.raises(A.AdapterError, match="twice"):
        s.add("a", {"model.layers.0.self_attn.o_proj": two, "model.layers.0.self_attn.o_proj.weight": two}, 1.0)
    with pytest.raises(A.AdapterError, match="for a matrix"):
        s.load("a", H.adapter_folder(helpers.model_folder("A"), 2, 10, 3))
    assert s.names == {} and all(low.a.count_nonzero() == 0 for low in s.stacks)


# ---- what a step carries -----------------------------------------------------------------------------------------------

def test_the_descriptor_carries_adapters_only_where_there_are_any():
    plain, lay = BatchLayout(4, 2, 2, 4, [0]), BatchLayout(4, 2, 2, 4, [0], None, True)
    assert "adapter_ids" not in plain.off and set(lay.off) == set(plain.off) | {"adapter_ids"}
    args = ([1, 2, 3, 4], [0, 1, 2, 3], [0, 1, 1, 1], [0, 1, 4], [9, 4], [1, 3], [0, 1], [0, 3], {0: [[1], [2]]}, {0: 9}, None)
    host = pack_batch(lay, *args, adapter_ids=[1, -1, -1, -1])
    ctx = StepContext(lay, host, torch.float32, "cpu", None, 64, None, 3, 10)
    assert ctx.adapter_ids.tolist() == [1, -1, -1, -1] and ctx.logit_rows.tolist() == [0, 3] and ctx.block_tables[0].tolist() == [[1, 9, 9, 9], [2, 9, 9, 9]]
    host = pack_batch(plain, *args, adapter_ids=[1, -1, -1, -1])
    assert StepContext(plain, host, torch.float32, "cpu", None, 64, None, 3, 10).adapter_ids is None


class _Handle:
    def __init__(self, tokens, n):
        self.tokens, self.host_logprobs, self.device_tokens = tokens, torch.arange(n) * -0.5, None


class _Sampler:
    """Knows which rows' settings it was given."""

    def __init__(self):
        self.seen = []

    def sample(self, logits, temps, us):
        self.seen.append(None)
        return [int(r.argmax()) for r in logits]

    def sample_async(self, logits, temps, us, params=None):
        self.seen.append(params)
        return _Handle([int(r.argmax()) for r in logits], len(logits))

    def read(self, h):
        return h.tokens


@pytest.mark.parametrize("pipelined", [False, True])
def test_the_scheduler_hands_adapters_and_filters_on(pipelined):
    from test_scheduler import FakeRunner
    from prism_b200.config.engine_config import SchedulerConfig
    from prism_b200.engine.scheduler import Scheduler

    class Runner(FakeRunner):
        adapters_seen = set()

        def can_run(self, segments):
            return True

        def step(self, segments, token_source=None):
            self.adapters_seen |= {(s.req_id, s.adapter) for s in segments}
            if token_source is not None or any(s.tokens == [0] for s in segments):
                segments = [Segment(s.req_id, [self.last[s.req_id]] if s.tokens == [0] else s.tokens, s.want, s.adapter) for s in segments]
            out = super().step(segments)
            if out is not None:
                for s, row in zip([s for s in segments if s.want], out):
                    self.last[s.req_id] = int(row.argmax())
            return out

    runner, sampler = Runner(64), _Sampler()
    runner.last = {}
    sched = Scheduler(runner, sampler, SchedulerConfig(async_decode=pipelined))
    plain = sched.add_request([1, 2, 3], SamplingParams(max_new_tokens=4))
    sched.run_to_completion()
    assert all(p is None for p in sampler.seen) and plain.logprobs == []
    reqs = [sched.add_request([4, 5], SamplingParams(max_new_tokens=5, temperature=1.0, top_k=3, logprobs=True), 2),
            sched.add_request([6], SamplingParams(max_new_tokens=3)), sched.add_request([7, 8], SamplingParams(max_new_tokens=4, temperature=0.5), 0)]
    sched.run_to_completion()
    assert {(r.id, r.adapter) for r in reqs} <= runner.adapters_seen and [r.adapter for r in reqs] == [2, -1, 0]
    assert len(reqs[0].logprobs) == len(reqs[0].generated_tokens) == 5 and reqs[1].logprobs == [] == reqs[2].logprobs
    given = [p for p in sampler.seen if p is not None]
    assert given and all(any(q.top_k == 3 for q in p) for p in given)
