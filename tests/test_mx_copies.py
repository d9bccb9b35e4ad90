"""Copies of rows and weights of microscaled numbers have their own memory, and know where it is.  No GPU needed."""
import copy
import io
import pickle

import pytest
import torch

from alofa_b200 import mx


@pytest.fixture
def rows(monkeypatch):
    """Rows on the CPU: what looks at addresses does not mind."""
    monkeypatch.setattr(mx, "_here", lambda: -1)
    codes = torch.arange(3 * 128, dtype=torch.int32).to(torch.uint8).view(3, 128)
    return mx.MxRows(codes, torch.full((3, 4), 120, dtype=torch.uint8), 100)


def saved(v):
    room = io.BytesIO()
    torch.save(v, room)
    room.seek(0)
    return torch.load(room, weights_only=False)


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda v: pickle.loads(pickle.dumps(v)), saved])
def test_copied_rows(rows, how):
    got = how(rows)
    assert got.codes_at == got.codes.data_ptr() and got.scales_at == got.scales.data_ptr() and got.shape == (3, 100) and got.device == -1
    assert torch.equal(got.codes, rows.codes) and torch.equal(got.scales, rows.scales)
    if how is not copy.copy:
        rows.codes.zero_()
        assert got.codes.any()
