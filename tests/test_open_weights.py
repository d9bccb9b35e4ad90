"""Weights that are made when a part asks for them.  No GPU needed."""
import gc
import weakref

import pytest
import torch

import tiny
from alofa_b200.errors import AlofaError
from alofa_b200.models.qwen2 import build_spec
from alofa_b200.parts import expected_tensors
from alofa_b200.parts.base import Runtime, stacked
from alofa_b200.parts.model import Model
from alofa_b200.weights.loader import Weights, load_state, open_weights
from alofa_b200.weights.random_init import random_state, random_weights
from alofa_b200.weights.safetensors_io import write_safetensors


def test_a_tensor_is_made_when_asked_for_and_again_when_it_is_gone():
    made = []

    def fetch(name):
        made.append(name)
        return torch.full((2,), float(len(made)))

    w = Weights({"a": (2,), "b": (2,)}, fetch)
    assert "a" in w and "c" not in w and len(w) == 2 and list(w) == ["a", "b"] and not made
    a = w["a"]
    assert w["a"] is a and made == ["a"]
    gone = weakref.ref(a)
    del a
    gc.collect()
    assert gone() is None and float(w["a"][0]) == 2 and made == ["a", "a"]
    table = w.setdefault("__table__", {})
    assert w.setdefault("__table__", {}) is table and w["__table__"] is table and list(w) == ["a", "b", "__table__"] and len(w) == 3
    assert w.pop("b").shape == (2,) and "b" not in w and list(w) == ["a", "__table__"]
    for missing in ("b", "c"):
        with pytest.raises(KeyError):
            w[missing]
        with pytest.raises(KeyError):
            del w[missing]


@pytest.mark.parametrize("name", ["A", "B"])
def test_the_same_tensors_as_the_whole_state(tmp_path, name):
    cfg, seed = tiny.CONFIGS[name]
    expected = expected_tensors(build_spec(cfg))
    folder = tiny.write(tmp_path / name, name)
    drawn = random_state(expected, seed)
    for dtype in (torch.bfloat16, torch.float32):
        whole = load_state(expected, folder, dtype, "cpu")
        for source in (folder, drawn, random_weights(expected, seed)):
            with open_weights(expected, source, dtype, "cpu") as weights:
                assert set(weights) == set(whole) and all(torch.equal(weights[n], whole[n]) and weights[n].dtype == whole[n].dtype for n in whole)


def test_a_model_holds_what_its_parts_hold(tmp_path):
    """While a layer loads, nothing of the layers before it is there but their own weights."""
    cfg, seed = tiny.CONFIGS["B"]
    model = Model(build_spec(cfg), Runtime(torch.device("cpu"), torch.bfloat16))
    drawn, alive, most = random_state(model.tensors(), seed), {}, 0

    def fetch(name):
        nonlocal most
        t = drawn[name].clone()
        alive[name] = weakref.ref(t)
        loose = [n for n, ref in alive.items() if ref() is not None and (".gate_proj." in n or ".up_proj." in n or "q_proj.w" in n or "k_proj.w" in n or "v_proj.w" in n)]
        most = max(most, len(loose))
        return t

    model.load(Weights({n: t.shape for n, t in drawn.items()}, fetch))
    assert most == 1 and len(alive) == len(drawn)
    other = Model(build_spec(cfg), Runtime(torch.device("cpu"), torch.bfloat16))
    other.load(drawn)
    assert "__rotary_tables__" not in drawn
    for a, b in zip(model.layers, other.layers):
        assert torch.equal(a.mixer.qkv.weight, b.mixer.qkv.weight) and torch.equal(a.feed_forward.gate_up.weight, b.feed_forward.gate_up.weight)
        assert torch.equal(a.mixer.qkv.bias, b.mixer.qkv.bias) and a.mixer.q_only.weight.data_ptr() == a.mixer.qkv.weight.data_ptr()


def test_what_does_not_fit_is_refused_before_anything_is_read(tmp_path):
    cfg, seed = tiny.CONFIGS["B"]
    expected = expected_tensors(build_spec(cfg))
    state = random_state(expected, seed)
    lacking = {n: t for n, t in state.items() if n != "model.norm.weight"}
    with pytest.raises(AlofaError, match="missing tensors"), open_weights(expected, lacking, torch.bfloat16, "cpu"):
        pass
    with pytest.raises(AlofaError, match="missing tensors"), open_weights(expected, Weights({n: t.shape for n, t in lacking.items()}, None), torch.bfloat16, "cpu"):
        pass
    state["model.norm.weight"] = state["model.norm.weight"].half()
    write_safetensors(tmp_path / "model.safetensors", state)
    with pytest.raises(AlofaError, match="float16.*model.norm.weight"), open_weights(expected, tmp_path, torch.bfloat16, "cpu"):
        pass


def test_stacked():
    state = {"a": torch.randn(3, 4).bfloat16(), "b": torch.randn(2, 4).bfloat16(), "c": torch.randn(1, 4)}
    assert torch.equal(stacked(state, ["a", "b"], 5), torch.cat([state["a"], state["b"]]))
    mixed = stacked(state, ["a", "c", "b"], 6)
    assert mixed.dtype == torch.float32 and torch.equal(mixed, torch.cat([state["a"], state["c"], state["b"]]))
