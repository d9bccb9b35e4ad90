"""Microscaled operators at their edges on the GPU: what a product does whose waits run out."""
import copy
import ctypes
import pickle

import numpy as np
import pytest
import torch

import plain_mx as plain
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


# ---- sums of deep products -----------------------------------------------------------------------------------------------


def deep_operands(t, n, k, seed):
    """Rows and weights in their codes as a model has them: most of a block's numbers well below its largest, scales over a range of 2^14."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kp = mx.padded(k)
    x = (120 * torch.randn(t, kp, generator=g, device="cuda")).clamp(-448, 448)
    x[:, k:] = 0
    xs = torch.randint(117, 121, (t, kp // 32), generator=g, device="cuda").to(torch.uint8)
    wc = torch.randint(0, 256, (n, kp // 2), generator=g, device="cuda").to(torch.uint8)
    ws = (120 + 1.5 * torch.randn(n, kp // 32, generator=g, device="cuda")).round().clamp(112, 126).to(torch.uint8)
    return mx.MxRows(x.to(torch.float8_e4m3fn).view(torch.uint8), xs, k), wc, ws


@pytest.mark.parametrize("k,how", [(k, how) for k, hows in {3584: [None, (16, 1), (32, 1), (64, 2), (96, 1), (128, 2), (256, 1)], 8960: [None, (16, 2), (64, 3), (96, 4), (256, 1)], 18944: [None, (16, 1), (16, 8), (32, 2), (64, 4), (128, 8), (256, 1)]}.items()
                                  for how in hows])
def test_deep_sums_are_as_exact_as_rounded_ones(k, how):
    """The tensor cores' additions cut off towards zero.  Measured on one accumulator over such operands, that takes 3.95e-9 off every
    sum for each slice of 128 (0.55e-7 over 14, 1.1e-7 over 28; 5.2e-9 each over 148), and the rest of what sums are off by is 1.1e-7 of them over 28
    slices and 5.5e-7 over 148; scalar additions leave no common share and 0.7e-7 at depth 3,584, 1.8e-7 at 18,944.  In runs the common share is
    that of the longest run (of 16, or 32 for prompts, or what eight parts leave), and the rest no more than that of sums which round: half as much again is allowed on each."""
    t, n = (300, 512) if how in (None, (256, 1), (128, 8), (128, 2)) else (60, 512)
    x, wc, ws = deep_operands(t, n, k, 90)
    w = mx.MxWeight.from_codes(wc, ws, k)
    want = x.dequantize(F32).double() @ w.dequantize(F32).double().T
    off = mx.linear(x, w, dtype=F32, how=how).double() - want
    share = float((off * want).sum() / (want * want).sum())
    slices, (bn, parts) = -(-k // 128), how or mx.plan(t, n, k)
    part = -(-slices // parts)
    runs = -(-part // 32) if bn == 256 else min(-(-part // 16), mx.MOST_RUNS[bn])
    assert abs(share) <= 1.5 * 3.95e-9 * -(-part // runs) and float((off - share * want).norm() / want.norm()) <= 1.5 * 1.8e-7, (share, float(off.norm() / want.norm()))


@pytest.mark.parametrize("t,n,k,parts", [(70, 200, 1100, 1), (96, 128, 3000, 3), (200, 515, 1000, 2), (97, 130, 2600, 1), (65, 129, 130, 2)])
def test_tiles_of_96_tokens(t, n, k, parts):
    xr, wp, xv, wv = product_operands(t, n, k, 82)
    want, loose = xv @ wv.T, sum_bound(xv, wv)
    assert (np.abs(host(mx.linear(xr, wp, dtype=F32, how=(96, parts))) - want) <= loose).all()
    f = n // 2
    xr, wp, xv, wv = product_operands(t, 2 * f, k, 83, gated=True)
    g, u = xv @ wv[:f].T, xv @ wv[f:].T
    want, slope = plain.silu(g) * u, 1.1 * np.abs(u) * sum_bound(xv, wv[:f]) + (np.abs(g) + 1) * sum_bound(xv, wv[f:])
    rows = mx.gated_linear(xr, wp, how=(96, parts))
    largest = np.abs(np.pad(want, ((0, 0), (0, -f % 32)))).reshape(t, -1, 32).max(-1).repeat(32, -1)[:, :f]
    # half a step of E4M3: 2^-4 of the number, or of the smallest normal number by a scale that is at most 2^-7 of the block's largest
    assert (np.abs(host(rows.dequantize(F32)).astype(np.float64) - want) <= np.maximum(2.0**-4 * np.abs(want), 2.0**-17 * largest) * (1 + 2.0**-10) + slope).all()


@pytest.mark.parametrize("t", [3, 72, 300])
def test_gated_products_of_several_runs(t):
    """Depths of two and more runs in a row, tiles behind one another: every accumulator begins anew."""
    for f, k in ((70, 2200), (9500, 2304), (40, 9000)):
        xr, wp, xv, wv = product_operands(t, 2 * f, k, 84, gated=True)
        g, u = xv @ wv[:f].T, xv @ wv[f:].T
        want, slope = plain.silu(g) * u, 1.1 * np.abs(u) * sum_bound(xv, wv[:f]) + (np.abs(g) + 1) * sum_bound(xv, wv[f:])
        largest = np.abs(np.pad(want, ((0, 0), (0, -f % 32)))).reshape(t, -1, 32).max(-1).repeat(32, -1)[:, :f]
        for how in (None, (256, 1)):
            rows = mx.gated_linear(xr, wp, how=how)
            assert (np.abs(host(rows.dequantize(F32)).astype(np.float64) - want) <= np.maximum(2.0**-4 * np.abs(want), 2.0**-17 * largest) * (1 + 2.0**-10) + slope).all()


# ---- copies --------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("gated", [False, True])
def test_a_copied_weight_has_its_own_memory(gated):
    xr, wp, _, _ = product_operands(5, 300, 500, 85, gated)
    product = (lambda w: mx.gated_linear(xr, w).dequantize()) if gated else (lambda w: mx.linear(xr, w))
    want, made = product(wp), copy.deepcopy({"w": wp, "same": wp})
    again, part = pickle.loads(pickle.dumps(wp)), None if gated else copy.deepcopy(wp.first_rows(140))
    assert made["w"] is made["same"] and copy.copy(wp) is wp
    for w in (made["w"], again):
        assert w.at == w.tiles.data_ptr() != wp.at and w.maps_at == ctypes.addressof(w.maps) != wp.maps_at and torch.equal(w.tiles, wp.tiles)
    wp.tiles.zero_()
    torch.cuda.synchronize()
    assert torch.equal(product(made["w"]), want) and torch.equal(product(again), want)
    if part is not None:
        assert torch.equal(product(part), want[:, :140].contiguous())


# ---- a weight made on another stream ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("recorded", [False, True])
def test_a_weight_packed_on_another_stream(recorded):
    """Products read their weight ahead of the kernel before them in their own stream, but not ahead of a wait for the stream
    that packed it.  The weights take one another's memory, so that a product that came too early would see the last one's."""
    w = [torch.randn(1152, 896, device="cuda") * 0.05 for _ in range(3)]
    x = mx.quantize_rows(torch.randn(8, 896, device="cuda"))
    want = [mx.linear(x, mx.pack_weight(v)).clone() for v in w]
    src = w[0].clone()
    packer, user = torch.cuda.Stream(), torch.cuda.Stream()

    def once():
        main = torch.cuda.current_stream()
        packer.wait_stream(main)
        user.wait_stream(main)
        with torch.cuda.stream(packer):
            for _ in range(3):
                v = src * 1.0  # something before it, so that it is late
            packed = mx.pack_weight(v)
        with torch.cuda.stream(user):
            before = mx.linear(x, other)  # the kernel before it, whose last CTAs are far from done when it lets the next one begin
            user.wait_stream(packer)
            out = mx.linear(x, packed)
        main.wait_stream(user)
        packed.tiles.record_stream(user)
        return out, before

    other = mx.pack_weight(w[2])
    torch.cuda.synchronize()
    if recorded:
        with torch.cuda.stream(torch.cuda.Stream()):
            once()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, before = once()
    for i in (1, 0, 2, 1, 1, 0) * 10:
        src.copy_(w[i])
        if recorded:
            graph.replay()
        else:
            out, before = once()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]) and torch.equal(before, want[2])
