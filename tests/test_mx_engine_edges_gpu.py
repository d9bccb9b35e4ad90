"""The engine with weights in 4 bits beside other work."""
import threading

import pytest
import torch

import tiny
from alofa_b200 import mx
from test_mx_engine_gpu import folders  # noqa: F401 (a fixture)
from test_mx_gpu import chain, chain_operands

pytestmark = pytest.mark.gpu


def test_operators_of_another_thread_beside_a_stepping_engine(folders):  # noqa: F811
    """A thread on a stream of its own: its operators run there, behind what that stream has to do first, not on the engine's."""
    from alofa_b200.engine.engine import Engine

    prompts = [tiny.tokens("B", n, seed=i) for i, n in enumerate([9, 21, 40])]
    engine = Engine(str(folders["B"]), weight_format="mxfp4", block_size=16, max_batch=4, token_budget=24, max_chunk=16, max_tokens=128)
    alone = [engine.generate(prompts, max_new_tokens=24) for _ in range(4)][-1]  # every shape recorded by now
    h, weight, wg, wd, owed = chain_operands(20, 3)
    w1, w2 = mx.pack_weight(wg, True), mx.pack_weight(wd)
    want = [chain(h * s, weight, w1, w2, owed) for s in (1.0, 3.0, 0.01)]
    torch.cuda.synchronize()
    checked, failed = [], []

    def other():
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for i in range(200):
                x = torch.zeros_like(h)
                torch.cuda._sleep(200_000)  # what makes the operands is late
                x.add_(h * (1.0, 3.0, 0.01)[i % 3])
                got = chain(x, weight, w1, w2, owed)
                stream.synchronize()
                checked.append(i)
                if not torch.equal(got, want[i % 3]):
                    failed.append(i)

    thread = threading.Thread(target=other)
    thread.start()
    beside = []
    while thread.is_alive():
        beside.append(engine.generate(prompts, max_new_tokens=24))
    thread.join()
    assert len(checked) == 200 and not failed and beside and all(b == alone for b in beside)


def peak_of(load):
    """(bytes that a loaded model takes, the most there were on the way)."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    model, *_ = load()
    torch.cuda.synchronize()
    return torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("weight_format", ["mxfp4", None])
@pytest.mark.parametrize("where", ["folder", "random", "random on the device"])
def test_a_model_loads_a_layer_at_a_time(tmp_path, where, weight_format):
    """Beside what the loaded model takes, one layer's weights as the checkpoint has them at most."""
    from alofa_b200.engine.loading import load_model, random_model
    from alofa_b200.models.qwen2 import NAME, Qwen2Config
    from alofa_b200.weights.random_init import write_random_model

    cfg = Qwen2Config(6, 512, 8, 2, 64, 2048, 300, 1e-6, 1e6, False, 256)
    layer = 2 * 512 * (8 * 64 + 2 * 2 * 64 + 512 + 3 * 2048)
    if where == "folder":
        folder = write_random_model(tmp_path / "m", NAME, cfg, 5)
        held, peak = peak_of(lambda: load_model(folder, "bfloat16", weight_format=weight_format))
    else:
        held, peak = peak_of(lambda: random_model(NAME, cfg, 5, "bfloat16", None, where != "random", weight_format))
    # drawn on the device, numbers stand in 32 bits before they are rounded: the largest matrix twice as large beside itself
    extra = 2 * 2 * 512 * 2048 if where == "random on the device" else 0
    assert peak <= held + layer + extra + (1 << 18), (held / layer, peak / layer)


def test_what_is_loaded_is_what_it_was(folders):  # noqa: F811
    """A layer at a time, from a folder or drawn: the tensors of the whole state, tied head and tables shared as before."""
    from alofa_b200.engine.loading import load_model
    from alofa_b200.parts.base import Runtime
    from alofa_b200.parts.model import Model
    from alofa_b200.weights.loader import load_state

    for name in ("A", "B"):
        model, cfg, arch = load_model(folders[name], "bfloat16")
        other = Model(arch.build_spec(cfg), Runtime(torch.device("cuda"), torch.bfloat16))
        other.load(load_state(other.tensors(), folders[name], torch.bfloat16, "cuda"))
        for a, b in zip(model.layers, other.layers):
            for x, y in ((a.mixer.qkv, b.mixer.qkv), (a.mixer.out, b.mixer.out), (a.feed_forward.gate_up, b.feed_forward.gate_up), (a.feed_forward.down, b.feed_forward.down)):
                assert torch.equal(x.weight, y.weight) and (x.bias is None) == (y.bias is None) and (x.bias is None or torch.equal(x.bias, y.bias))
        assert torch.equal(model.head.linear.weight, other.head.linear.weight) and torch.equal(model.embedding.weight, other.embedding.weight)
        assert (model.head.linear.weight.data_ptr() == model.embedding.weight.data_ptr()) == (other.head.linear.weight.data_ptr() == other.embedding.weight.data_ptr())
        assert len({block.mixer.position.rotary_table()[0].data_ptr() for block in model.layers}) == 1
