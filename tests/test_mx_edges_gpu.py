"""Microscaled operators at their edges on the GPU: what a product does whose waits run out."""
import ctypes

import numpy as np
import pytest
import torch

from alofa_b200 import mx
from alofa_b200.csrc.build import load_library
from test_mx_gpu import host, product_operands, sum_bound

pytestmark = pytest.mark.gpu

F32 = torch.float32


# ---- waits that run out -----------------------------------------------------------------------------------------------


@pytest.fixture
def no_patience(monkeypatch):
    """The products from a library whose waits on a barrier give up at once: no slice has landed by then."""
    lib = load_library("alofa_mx_no_patience", ["kernels/mx_gemm.cu"], {"ALOFA_WAIT_LIMIT": "0u"})
    lib.alofa_mx_gemm.restype, lib.alofa_mx_gemm.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]
    patient = mx._lib.alofa_mx_gemm
    monkeypatch.setattr(mx._lib, "alofa_mx_gemm", lib.alofa_mx_gemm, raising=False)
    return patient


@pytest.mark.parametrize("t,n,k,how", [(1, 128, 128, (16, 1)), (5, 300, 500, (16, 1)), (5, 300, 2048, (16, 4)), (33, 520, 4000, (32, 8)), (70, 200, 1100, (64, 2)), (130, 384, 3000, (128, 3))])
def test_a_product_that_gives_up(no_patience, monkeypatch, t, n, k, how):
    """Its copies land, its sums are not numbers, it says so, and what runs next is right.  Depths of fewer slices than the
    ring has stages, where the copying warps never wait, and of more."""
    xr, wp, xv, wv = product_operands(t, n, k, 80)
    room = torch.full((t + 2, n), 7.0, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for _ in range(20):
        mx.linear(xr, wp, out=room[1:-1], how=how, status=status)
    torch.cuda.synchronize()
    assert int(status) == 2 and torch.isnan(room[1:-1]).all() and (room[0] == 7).all() and (room[-1] == 7).all()
    monkeypatch.setattr(mx._lib, "alofa_mx_gemm", no_patience)
    status.zero_()
    assert (np.abs(host(mx.linear(xr, wp, dtype=F32, how=how, status=status)) - xv @ wv.T) <= sum_bound(xv, wv)).all() and int(status) == 0


def test_a_gated_product_that_gives_up(no_patience):
    xr, wp, _, _ = product_operands(20, 2 * 70, 1500, 81, gated=True)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = mx.gated_linear(xr, wp, how=(32, 3), status=status)
    assert torch.isnan(rows.dequantize(F32)).all() and int(status) == 2


# ---- the gate far below zero ---------------------------------------------------------------------------------------------

#: gates as sums of numbers that weights in 4 bits have, and how large the factors beside them are
FAR = [([64, 16, 6, q], 120) for q in (0, 0.5, 1, 1.5, 2, 3)] + [([64, 16, 8, q], 122) for q in (0, 0.5, 1, 1.5, 2, 3)] + [([64, 16, 12, 0], 125), ([64, 32, 4, 0], 125), ([64, 48, 8, 0], 126), ([128, 16, 6, 0], 126), ([128, 48, 0, 0], 126),
      ([64, 16, 6, 0.5], 0), ([64, 24, 1, 0], 30), ([64, 16, 1, 0], 100), ([2**20, 0, 0, 0], 126), ([2**100, 0, 0, 0], 126)]


@pytest.mark.parametrize("how", [None, (256, 1)])
@pytest.mark.parametrize("t", [1, 5, 300])
@pytest.mark.parametrize("gate", [None, (1.0, 2.0**127), (2.0, 2.0**127)])
def test_a_gate_far_below_zero(gate, t, how):
    """silu(g) u where the logistic function is next to the smallest numbers of 32 bits and below them, and u is large: each
    feature alone in its block, so that its own size decides its scale.  Sums here are exact, so what is rounded is off by
    ROWS_SLACK of itself (the exponential, by two factors of at most 4 units each) where it is a normal number."""
    w = torch.zeros(2 * 32 * len(FAR), 160)
    g, u = np.zeros(32 * len(FAR)), np.zeros(32 * len(FAR))
    for i, (parts, power) in enumerate(FAR):
        w[32 * i, 0:128:32] = -torch.tensor(parts, dtype=F32)
        w[32 * len(FAR) + 32 * i, 128] = -1.5 * 2.0**power
        g[32 * i], u[32 * i] = -float(sum(parts)), -1.5 * 2.0**power
    x = torch.zeros(t, 160)
    x[:, ::32] = 1
    rows = mx.gated_linear(x.cuda(), mx.pack_weight(w.cuda(), True), *([] if gate is None else [gate]), how=how)
    alpha = 1.0 if gate is None else gate[0]
    with np.errstate(over="ignore"):
        want = g / (1 + np.exp(-alpha * g)) * (u if gate is None else np.maximum(u, -(2.0**127)) + 1)
    got, scales = host(rows.dequantize(F32)).astype(np.float64), host(rows.scales).astype(np.float64)
    unit = np.exp2(scales - 127).repeat(32, -1)[:, : len(g)]
    step = unit * np.exp2(np.maximum(np.frexp(np.maximum(np.abs(got), np.abs(want)) / unit)[1] - 1, -6) - 3.0)
    off = np.abs(got - want) - step / 2 - 2.0**-18 * np.abs(want)
    assert (off <= 0).all(), [(float(g[32 * i]), got[0, 32 * i], want[32 * i]) for i in range(len(FAR)) if (off[:, 32 * i] > 0).any()]
