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
