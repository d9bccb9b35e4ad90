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
