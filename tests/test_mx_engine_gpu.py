"""The engine with its layers' weights in 4 bits, against the plain model whose
products take weights and rows as their formats hold them."""
import json
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import plain_mx
import plain_qwen2 as plain
import replay
import tiny

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
NAMES = ["A", "B", "C"]
LENGTHS = {"A": [5, 17, 33, 70], "B": [1, 9, 64, 143], "C": [3, 40, 130]}


def loud(folder, name):
    """A tiny model whose sublayers weigh as much as the embedding does."""
    from alofa_b200.weights.safetensors_io import write_safetensors

    folder = tiny.write(folder, name)
    state = {k: torch.from_numpy(v) for k, v in plain.read_safetensors(folder / "model.safetensors").items()}
    for k in state:
        if k.endswith("_proj.weight"):
            state[k] = state[k] * 3
    write_safetensors(folder / "model.safetensors", {k: v.to(torch.bfloat16) for k, v in state.items()})
    return folder


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    base = tmp_path_factory.mktemp("loud")
    return {name: loud(base / name, name) for name in NAMES}


def held(folder):
    """(weights as 4 bits hold them, config) of a model folder."""
    wts, cfg = plain.load(folder)
    return {k: plain_mx.values(v, True) if k.endswith("_proj.weight") else v for k, v in wts.items()}, cfg


def held_forward(ids, wts, cfg):
    """The plain model; a product with a weight in 4 bits takes its rows in 8."""
    full = plain.linear
    mine = {id(v) for k, v in wts.items() if k.endswith("_proj.weight")}
    plain.linear = lambda x, w, b=None: full(plain_mx.values(x) if id(w) in mine else x, w, b)
    try:
        return plain.forward(ids, wts, cfg)
    finally:
        plain.linear = full


def runner_for(folder, block=16, pages=40, weight_format="mxfp4", graphs=True):
    from alofa_b200.engine.loading import load_model
    from alofa_b200.engine.step import StepRunner

    model, *_ = load_model(folder, "bfloat16", weight_format=weight_format)
    return StepRunner(model, block_size=block, num_pages=pages, max_requests=8, max_tokens=model.spec.max_position, max_step_tokens=512, cuda_graphs=graphs)


def requests(name):
    return {f"r{i}": tiny.tokens(name, n + 16, seed=i) for i, n in enumerate(LENGTHS[name])}, {f"r{i}": n for i, n in enumerate(LENGTHS[name])}


# bfloat16 leaves q, k, v and the attention's output off by up to 2^-9 of their size.  A number that is off by d (of a step s of
# E4M3, 2^-4 to 2^-3 of its size) before it is rounded comes out a whole step off with probability d / s, so off by sqrt(d s),
# about 1 %, in the mean square, and these loud models enlarge that: rounding those four to bfloat16 in the plain model itself moves
# its logits by 4 to 7 % (root mean square) and 20 to 36 % (the largest).  The probabilities, which are rounded too, and products
# whose q, k and v are rounded before and after they are turned, come on top: half as much again is allowed.
RMS, LARGEST = 0.1, 0.54


def far(got, want):
    size = np.sqrt((want**2).mean())
    return np.sqrt(((got - want) ** 2).mean()) / size, np.abs(got - want).max() / size


@pytest.mark.parametrize("name", NAMES)
def test_every_cut_is_the_plain_model_in_these_formats(folders, name):
    reqs, prompts = requests(name)
    wts, cfg = held(folders[name])
    vocab = tiny.CONFIGS[name][0].vocab_size
    want = {rid: held_forward(toks, wts, cfg) for rid, toks in reqs.items()}
    others = {rid: plain.forward(toks, *plain.load(folders[name])) for rid, toks in reqs.items()}
    runner = runner_for(folders[name])
    for steps in (replay.whole(reqs), replay.tail_decoded(reqs, 16), replay.portions(reqs), replay.mixed(reqs, prompts, 40 * 16, 16)):
        got = replay.collect(steps, replay.run_inprocess(runner, steps), vocab)
        for rid in reqs:
            rms, largest = far(got[rid], want[rid])
            assert rms <= RMS and largest <= LARGEST, (rid, rms, largest)
    # the formats are what is compared: the same model without them is much further away
    assert min(far(others[rid], want[rid])[0] for rid in reqs if len(reqs[rid]) > 30) > 2 * RMS


def test_steps_give_the_same_again(folders):
    """Sums are taken in a fixed order: replayed graphs, and steps that are not, give equal logits, run after run."""
    reqs, _ = requests("B")
    steps = replay.tail_decoded(reqs, 16)
    first = replay.run_inprocess(runner_for(folders["B"]), steps)
    again = runner_for(folders["B"])
    for _ in range(2):
        got = replay.run_inprocess(again, steps)
        assert all(np.array_equal(first[i], got[i]) for i in first)
    plainly = replay.run_inprocess(runner_for(folders["B"], graphs=False), steps)
    assert all(np.array_equal(first[i], plainly[i]) for i in first)


def test_generate_and_the_command_line(folders):
    from alofa_b200.engine.engine import Engine

    name = "B"
    prompts = [tiny.tokens(name, n, seed=i) for i, n in enumerate([9, 21, 40])]
    settings = dict(block_size=16, max_batch=4, token_budget=24, max_chunk=16, max_tokens=128)
    engine = Engine(str(folders[name]), weight_format="mxfp4", **settings)
    out = engine.generate(prompts, max_new_tokens=6)
    wts, cfg = held(folders[name])
    for p, o in zip(prompts, out):
        for k, token in enumerate(o):
            row = held_forward(p + o[:k], wts, cfg)[-1]
            assert row.max() - row[token] <= 2 * LARGEST * np.sqrt((row**2).mean())
    assert engine.generate(prompts, max_new_tokens=6) == out
    cmd = [sys.executable, str(ROOT / "bin" / "generate"), "--model", str(folders[name]), "--weight-format", "mxfp4", "--max-new-tokens", "6", "--block-size", "16", "--max-tokens", "128", "--token-budget",
           "24", "--max-chunk", "16", "--max-batch", "4", "--json"]
    for p in prompts:
        cmd += ["--prompt-ids", ",".join(map(str, p))]
    ran = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0, ran.stderr[-2000:]
    assert json.loads(ran.stdout.strip().splitlines()[-1])["out_ids"] == out


def test_trace_run_takes_the_format(folders, tmp_path):
    reqs, _ = requests("A")
    steps = replay.whole(reqs)
    got = replay.run_trace_program(folders["A"], "bfloat16", steps, tmp_path, 512, ["--weight-format", "mxfp4", "--block-size", "16"])
    mine = replay.run_inprocess(runner_for(folders["A"]), steps)
    assert all(np.array_equal(mine[i].reshape(-1), got[i]) for i in mine)


def test_random_weights_and_what_they_take(folders):
    from alofa_b200.engine.loading import random_model
    from alofa_b200.models.qwen2 import NAME, Qwen2Config

    cfg = Qwen2Config(2, 896, 14, 2, 64, 4864, 1000, 1e-6, 1e6, True, 512)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    model, *_ = random_model(NAME, cfg, 0, "bfloat16", None, True, "mxfp4")
    held_bytes = torch.cuda.memory_allocated() - before
    per_layer = 896 * (1152 + 896 + 3 * 4864)
    assert held_bytes < 2 * 1000 * 896 + 2 * (per_layer * 17 / 32) * 1.02 + (1 << 20)
    del model


def test_a_layer_that_reads_another_layers_cache(folders):
    """Its queries come from the same packed rows as those of a layer that writes."""
    from alofa_b200.engine.loading import random_model
    from alofa_b200.engine.step import StepRunner
    from alofa_b200.models import qwen2
    from alofa_b200.parts.base import Runtime
    from alofa_b200.parts.model import Model
    from alofa_b200.config.spec import RunEntry
    from alofa_b200.weights.loader import load_state
    from alofa_b200.weights.random_init import random_state

    cfg = tiny.CONFIGS["B"][0]
    spec = qwen2.build_spec(cfg)
    spec.run = [RunEntry(0, 0), RunEntry(1, 0), RunEntry(2, 2)]
    model = Model(spec, Runtime(torch.device("cuda"), torch.bfloat16, "mxfp4"))
    model.load(load_state(model.tensors(), random_state(model.tensors(), 3), torch.bfloat16, torch.device("cuda")))
    runner = StepRunner(model, block_size=16, num_pages=20, max_requests=4, max_tokens=128, max_step_tokens=128)
    steps = replay.tail_decoded({"a": tiny.tokens("B", 40)}, 8)
    whole = replay.whole({"a": tiny.tokens("B", 40)})
    a = replay.collect(steps, replay.run_inprocess(runner, steps), cfg.vocab_size)["a"]
    b = replay.collect(whole, replay.run_inprocess(runner, whole), cfg.vocab_size)["a"]
    rms, largest = far(a, b)
    assert np.isfinite(a).all() and rms <= RMS and largest <= LARGEST
