"""How a product of microscaled numbers is cut, by the device that it runs on.  No GPU needed."""
import pytest

from alofa_b200 import mx


@pytest.fixture
def device(monkeypatch):
    """What the current device is, and how many SMs each has."""
    now = {"device": 0, "sms": {0: 148, 1: 20}}
    monkeypatch.setattr(mx, "_here", lambda: now["device"])
    monkeypatch.setattr(mx, "_sms", lambda here: now["sms"][here])
    mx._plans.clear()
    yield now
    mx._plans.clear()


def test_a_plan_is_its_devices(device):
    sizes = [(t, n, k, gated) for t in (1, 8, 64, 200, 700) for n, k in ((1152, 896), (3584, 18944), (37888, 3584)) for gated in (False, True)]
    first = [mx.plan(*s) for s in sizes]
    device["device"] = 1
    other = [mx.plan(*s) for s in sizes]
    mx._plans.clear()
    assert other == [mx.plan(*s) for s in sizes] != first
    device["device"] = 0
    assert [mx.plan(*s) for s in sizes] == first


def test_runs_are_short_where_they_can_be(device):
    """No way sums more slices in one accumulator than 16 (64 where nothing is rounded to 8 bits) where more parts would have cut them."""
    for t in (1, 16, 33, 65, 96, 128, 200, 256, 400, 700, 1024):
        for n, k in ((1152, 896), (896, 4864), (1536, 8960), (3584, 18944), (37888, 3584), (300, 40000), (128, 16384), (512, 2049)):
            for gated in (False, True):
                tokens, parts = mx.plan(t, n, k, gated)
                slices = mx.padded(k) // 128
                if tokens < 256:  # pairs cut any depth
                    assert parts == 8 or -(-slices // parts) <= (16 if gated else 64) * mx.MOST_RUNS[tokens], (t, n, k, gated)


def test_accumulators_fit_the_kernels():
    """As many as the columns that a CTA may have leave room for beside its scales (two CTAs an SM, eight columns a stage)."""
    import pathlib
    import re

    text = (pathlib.Path(mx.__file__).parent / "csrc" / "kernels" / "mx_gemm.cu").read_text()
    assert tuple(map(int, re.search(r"RUN_SLICES = (\d+), RUN_SLICES_STORED = (\d+);", text).groups())) == (mx.RUN_SLICES, mx.RUN_SLICES_STORED)
    small, middle, large = (int(v) for v in re.search(r"STAGES = BN <= 32 \? (\d+) : BN == 64 \? (\d+) : (\d+);", text).groups())
    assert mx.MOST_RUNS == {bn: (256 - 8 * stages) // bn for bn, stages in ((16, small), (32, small), (64, middle), (96, large), (128, large))}
