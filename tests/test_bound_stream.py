"""The stream that a step binds is its own thread's: no other thread's launches go to it.  No GPU needed."""
import threading

import pytest
import torch

from alofa_b200 import mx
from alofa_b200.csrc import ops


class Stream:
    def __init__(self, handle):
        self.cuda_stream = handle


@pytest.fixture
def streams(monkeypatch):
    """A current stream for each thread, as torch has them: its handle is the thread's entry."""
    mine = {}
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(mine[threading.get_ident()]))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: mine[threading.get_ident()], raising=False)
    return mine


def handles():
    return ops._stream(), mx._stream(0)


def in_a_thread(streams, handle, call):
    """What ``call`` gives in a thread whose current stream has this handle."""
    out = []

    def run():
        streams[threading.get_ident()] = handle
        out.append(call())

    thread = threading.Thread(target=run)
    thread.start()
    thread.join()
    return out[0]


def test_a_thread_keeps_its_own_stream_while_another_is_in_a_step(streams):
    streams[threading.get_ident()] = 11
    with ops.bound_stream():
        assert handles() == (11, 11)
        assert in_a_thread(streams, 22, handles) == (22, 22)

        def step():
            with ops.bound_stream():
                return handles()

        assert in_a_thread(streams, 33, step) == (33, 33)
        assert handles() == (11, 11)  # what another thread bound and let go is not this one's
    assert handles() == (11, 11)


def test_bound_once_and_nested(streams):
    me = threading.get_ident()
    streams[me] = 11
    with ops.bound_stream():
        streams[me] = 12  # looked up on entry only
        assert handles() == (11, 11)
        with ops.bound_stream():
            assert handles() == (12, 12)
        assert handles() == (11, 11)
    assert handles() == (12, 12)
    with pytest.raises(ValueError):
        with ops.bound_stream():
            streams[me] = 13
            raise ValueError
    assert handles() == (13, 13)
