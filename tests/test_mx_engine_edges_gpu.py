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
