"""Adapter folders whose configuration says that W + scale B A is not the formula, and how the command answers (CPU)."""

import json
import os

import pytest
from safetensors.torch import load_file, save_file

import adapter_helpers as H
import helpers
from prism_b200.weights import adapters as A


def folder_with(**change):
    d = H.adapter_folder(helpers.model_folder("B"), change.pop("rank", 3), 12, 1)
    path = os.path.join(d, "adapter_config.json")
    with open(path) as f:
        cfg = json.load(f)
    with open(path, "w") as f:
        json.dump(dict(cfg, **change), f)
    return d


@pytest.mark.parametrize("how", ["pissa", "pissa_niter_16", "PiSSA", "olora", "corda", "loftq", "lora_ga", "something new"])
def test_an_adapter_beside_a_changed_matrix_is_refused(how):
    """Such a beginning takes its product out of W (or rounds W): the adapter belongs to the matrix that is left."""
    with pytest.raises(A.AdapterError, match="init_lora_weights"):
        A.read_adapter_config(folder_with(init_lora_weights=how))


@pytest.mark.parametrize("how", [True, False, None, "gaussian", "eva", "orthogonal"])
def test_a_beginning_that_leaves_the_matrix_is_taken(how):
    assert A.read_adapter_config(folder_with(init_lora_weights=how)) == (3, 4.0)


@pytest.mark.parametrize("change", [dict(alora_invocation_tokens=[5, 6]), dict(arrow_config={"top_k": 2}), dict(use_qalora=True), dict(use_bdlora={"nblocks": 2}),
                                    dict(lora_bias=True), dict(trainable_token_indices=[1])])
def test_what_applies_to_some_tokens_or_adds_more_is_refused(change):
    with pytest.raises(A.AdapterError, match=next(iter(change))):
        A.read_adapter_config(folder_with(**change))


def test_settings_that_are_off_are_taken():
    assert A.read_adapter_config(folder_with(alora_invocation_tokens=None, arrow_config=None, use_qalora=False, lora_bias=False, trainable_token_indices=None)) == (3, 4.0)


@pytest.mark.parametrize("make,say", [(lambda: folder_with(r=129), "129"), (lambda: folder_with(use_dora=True), "use_dora"), (lambda: "/nonexistent", "adapter_config")])
def test_the_command_says_what_is_wrong_with_an_adapter(make, say, capsys):
    """Before it loads a model, in a line."""
    from prism_b200.cli import main
    assert main(["--model", "/nonexistent", "--adapter", make()]) == 2
    err = capsys.readouterr().err
    assert say in err and "Traceback" not in err and err.count("\n") == 1


@pytest.mark.parametrize("text", ["", "{", "[1, 2]", "3", "null", "\xff\xfe"])
def test_a_configuration_that_is_none_is_refused(text, capsys):
    from prism_b200.cli import main
    d = folder_with()
    with open(os.path.join(d, "adapter_config.json"), "w", encoding="latin-1") as f:
        f.write(text)
    with pytest.raises(A.AdapterError, match="adapter_config"):
        A.read_adapter_config(d)
    assert main(["--model", "/nonexistent", "--adapter", d]) == 2 and "adapter_config" in capsys.readouterr().err


@pytest.mark.parametrize("keep", [0, 5, 40, -16])
def test_tensors_that_are_cut_off_are_refused(keep):
    d = folder_with()
    path = os.path.join(d, "adapter_model.safetensors")
    with open(path, "rb") as f:
        data = f.read()
    with open(path, "wb") as f:
        f.write(data[:keep])
    with pytest.raises(A.AdapterError, match="adapter_model"):
        A.read_adapter_folder(d)


def test_a_matrix_that_is_named_twice_is_refused():
    d = folder_with()
    path = os.path.join(d, "adapter_model.safetensors")
    tensors = {n: v.clone() for n, v in load_file(path).items()}
    first = sorted(tensors)[0]
    save_file(dict(tensors, **{first.removeprefix("base_model.model."): tensors[first] * 2}), path)
    with pytest.raises(A.AdapterError, match="twice"):
        A.read_adapter_folder(d)
