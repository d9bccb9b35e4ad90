"""Microscaled weights and rows on the GPU, against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import plain_mx as plain
from alofa_b200 import mx
from alofa_b200.csrc import ops
from alofa_b200.errors import AlofaError

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
ROWS_SLACK = 2.0**-18  # what fp32 sums of a few thousand numbers and the hardware's exponential leave in a normed or gated number


def numbers(t, k, seed, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, k, generator=g) * torch.exp(2 * torch.randn(t, 1, generator=g)) * scale
    x[:, ::37] *= 30
    return x.to(dtype)


def host(t):
    return t.cpu().numpy()


def unpack(tiles, n, k, gated):
    """Codes and scales of a weight's tiles, by rows of the product."""
    tall, slices, _ = tiles.shape
    raw = host(tiles)
    c = raw[:, :, :8192].reshape(tall, slices, 128, 64).transpose(0, 2, 1, 3).reshape(tall * 128, -1)
    codes = np.stack([c & 15, c >> 4], -1).reshape(tall * 128, -1)
    s = raw[:, :, 8192:].reshape(tall, slices, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(tall * 128, -1)
    if gated:
        f = np.arange(n // 2)
        at = f // 16 * 32 + f % 16
        at = np.concatenate([at, at + 16])
    else:
        at = np.arange(n)
    rest = np.setdiff1d(np.arange(tall * 128), at)
    return codes[at], s[at], codes[rest]


# ---- rows ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,k", [(1, 1), (1, 32), (3, 33), (2, 127), (5, 128), (7, 896), (1, 1000), (33, 1537), (300, 264)])
def test_rows_are_the_nearest_codes(t, k, dtype):
    x = numbers(t, k, 1, dtype)
    rows = mx.quantize_rows(x.cuda())
    codes, scales = plain.encode(x, False)
    assert np.array_equal(host(rows.scales), scales) and np.array_equal(host(rows.codes), codes)
    want = plain.decode(codes, scales, k, False)
    assert np.array_equal(host(rows.dequantize(F32)), want)
    assert np.array_equal(host(rows.dequantize().float()), want)  # four digits: bfloat16 has them all


def test_rows_ties_borders_and_the_smallest_numbers():
    steps = np.concatenate([plain.E4M3, (plain.E4M3[1:] + plain.E4M3[:-1]) / 2])  # every code and every tie
    x = np.zeros((12, 32 * 12), np.float32)
    for r, power in enumerate([-140, -133, -127, -120, -60, -1, 0, 1, 50, 100, 110, 118]):
        block = np.concatenate([steps[:240], -steps[:144]])
        x[r] = block * 2.0**power
        x[r, ::32] = 448 * 2.0**power  # the block's largest: its scale is 2^power
    x[6, 0::32] = np.float32(448.0)
    x[6, 32] = np.nextafter(np.float32(448.0), np.float32(500))  # one step over: the next scale
    rows = mx.quantize_rows(torch.from_numpy(x).cuda())
    codes, scales = plain.encode(x, False)
    assert np.array_equal(host(rows.scales), scales) and np.array_equal(host(rows.codes), codes)


def test_rows_of_zeros_infinities_and_nan():
    x = torch.randn(4, 160)
    x[0] = 0
    x[1, 5], x[1, 40], x[2, 159], x[3, 64] = float("inf"), float("nan"), float("-inf"), 3.0e38
    rows = mx.quantize_rows(x.cuda())
    codes, scales = plain.encode(x, False)
    assert np.array_equal(host(rows.scales), scales) and np.array_equal(host(rows.codes), codes)
    got = host(rows.dequantize(F32))
    assert np.isnan(got[1, :64]).all() and np.isfinite(got[1, 64:]).all() and np.isnan(got[2, 128:]).all() and np.isfinite(got[3]).all() and (got[0] == 0).all()


def test_rows_over_memory_off_its_alignment():
    base = torch.randn(3 * 64 + 1).cuda()
    x = base[1:].view(3, 64)  # 4 bytes off
    codes, scales = plain.encode(x, False)
    rows = mx.quantize_rows(x)
    assert np.array_equal(host(rows.codes), codes) and np.array_equal(host(rows.scales), scales)


# ---- weights ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k,gated", [(1, 1, False), (128, 128, False), (130, 257, False), (2, 32, True), (66, 100, True), (1152, 896, False), (512, 1000, True)])
def test_weights_are_the_nearest_codes(n, k, gated, dtype):
    w = numbers(n, k, 2, dtype, 0.02)
    packed = mx.pack_weight(w.cuda(), gated)
    codes, scales = plain.encode(w, True)
    got_codes, got_scales, rest = unpack(packed.tiles, n, k, gated)
    assert np.array_equal(got_codes, codes) and np.array_equal(got_scales, scales) and not rest.any()
    want = plain.decode(codes, scales, k, True)
    assert np.array_equal(host(packed.dequantize(F32)), want) and np.array_equal(host(packed.dequantize().float()), want)


def test_weights_ties_and_what_is_clipped():
    v = np.array([0, 0.25, 0.26, 0.5, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 5.01, 6, 6.5, 7.99, -0.25, -0.75, -5, -7, 4, 1, 2, 3] + [0.1] * 10, np.float32)
    w = np.stack([v, v * 2.0**-20, v * 2.0**100, v * 2.0**-128])
    packed = mx.pack_weight(torch.from_numpy(w.astype(np.float32)).cuda())
    codes, scales = plain.encode(w.astype(np.float32), True)
    got_codes, got_scales, _ = unpack(packed.tiles, 4, 32, False)
    assert np.array_equal(got_codes, codes) and np.array_equal(got_scales, scales)


@pytest.mark.parametrize("n,k,gated", [(130, 257, False), (66, 100, True), (256, 256, True)])
def test_a_weight_from_codes_is_the_weight_packed(n, k, gated):
    w = numbers(n, k, 3, F32, 0.02)
    codes, scales = plain.encode(w, True)
    dirty = codes.copy()
    dirty[:, k:] = 5  # behind the depth: not read
    made = mx.MxWeight.from_codes(torch.from_numpy(plain.nibbles(dirty)).cuda(), torch.from_numpy(scales.astype(np.uint8)).cuda(), k, gated)
    assert torch.equal(made.tiles, mx.pack_weight(w.cuda(), gated).tiles)


# ---- the norm --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("t,k,planes,bias,layer", [(1, 896, 4, False, False), (3, 100, 0, True, False), (5, 1537, 2, True, True), (37, 1536, 1, False, False), (2, 9000, 3, False, True), (300, 64, 8, True, False), (1, 1, 0, False, False)])
def test_norm_rows(t, k, planes, bias, layer):
    base, weight = numbers(t, k, 4), 1 + 0.1 * torch.randn(k)
    owed = torch.randn(planes, t, k) if planes else None
    b, shift = torch.randn(k) if bias else None, torch.randn(k) if layer else None
    dev = lambda v: None if v is None else v.cuda()  # noqa: E731
    h = base.cuda()
    rows = mx.norm_rows(h, dev(weight), 1e-6, owed=dev(owed), bias=dev(b), shift=dev(shift))
    want_h = base.double() + (owed.double().sum(0) if planes else 0) + (b.double() if bias else 0)
    size = base.abs().double() + (owed.abs().double().sum(0) if planes else 0) + (b.abs().double() if bias else 0)
    assert ((h.cpu().double() - want_h).abs() <= (planes + 1) * 2.0**-24 * size).all()  # a rounding an addition
    y = plain.norm(h.cpu().double().numpy(), weight.double().numpy(), 1e-6, None if shift is None else shift.double().numpy())
    if layer and k > 1:  # a difference from the mean, and a sum with the shift, may cancel: their roundings count by what went in
        spread = np.abs(y) + np.abs(shift.double().numpy()) + 1
        got = host(rows.dequantize(F32)).astype(np.float64)
        unit = np.exp2(host(rows.scales).astype(np.float64) - 127).repeat(32, -1)[:, :k]
        step = unit * np.exp2(np.maximum(np.frexp(np.maximum(np.abs(got), np.abs(y)) / unit)[1] - 1, -6) - 3.0)
        assert (np.abs(got - y) <= step / 2 + ROWS_SLACK * spread).all()
    else:
        assert plain.near(host(rows.codes), host(rows.scales), y, ROWS_SLACK)
    # into another tensor, the base left as it is
    base_dev, h2 = base.cuda(), torch.full((t, k), float("nan"), device="cuda")
    again = mx.norm_rows(h2, dev(weight), 1e-6, base=base_dev, owed=dev(owed), bias=dev(b), shift=dev(shift))
    assert torch.equal(h2, h) and torch.equal(again.codes, rows.codes) and torch.equal(again.scales, rows.scales) and torch.equal(base_dev.cpu(), base)


# ---- attention's splits ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("t,heads,hd,splits,split_keys,window", [(1, 14, 64, 3, 256, 0), (5, 3, 48, 1, 64, 0), (8, 28, 128, 16, 128, 0), (3, 5, 16, 9, 64, 0), (4, 2, 40, 12, 64, 200)])
def test_merged_splits(t, heads, hd, splits, split_keys, window):
    g = torch.Generator().manual_seed(9)
    o, m = torch.randn(splits, t * heads, hd, generator=g), 20 * torch.randn(splits, t * heads, generator=g)
    l = 1 + 5 * torch.rand(splits, t * heads, generator=g)
    m[0, 0] = m[-1, -1] = -float("inf")  # a split that saw nothing (its sums are not read)
    o[0, 0], o[-1, -1] = float("nan"), float("nan")
    positions = torch.randint(0, splits * split_keys, (t,), generator=g)
    positions[0] = splits * split_keys - 1
    rows = mx.merge_rows(o.cuda(), torch.stack([m, l], -1).cuda(), positions.int().cuda(), heads, window, split_keys)
    want = np.zeros((t, heads * hd))
    for i in range(t):
        p = int(positions[i])
        first, last = (max(0, p - window + 1) if window else 0) // split_keys, p // split_keys
        for h in range(heads):
            r = i * heads + h
            seen = [s for s in range(first, last + 1) if m[s, r] > -float("inf")]
            top = max((float(m[s, r]) for s in seen), default=0.0)
            w = [2.0 ** (float(m[s, r]) - top) for s in seen]
            low = sum(a * float(l[s, r]) for a, s in zip(w, seen))
            want[i, h * hd : (h + 1) * hd] = sum(a * o[s, r].double().numpy() for a, s in zip(w, seen)) / low if seen else np.nan
    got = host(rows.dequantize(F32)).astype(np.float64)
    bad = np.isnan(want)
    # positions behind the splits see all of them, negative ones nothing
    ml = torch.stack([m, l], -1).cuda()
    ends = mx.merge_rows(o.cuda(), ml, torch.full((t,), splits * split_keys - 1, dtype=torch.int32, device="cuda"), heads, 0, split_keys)
    beyond = mx.merge_rows(o.cuda(), ml, torch.full((t,), 2**31 - 1, dtype=torch.int32, device="cuda"), heads, 0, split_keys)
    assert torch.equal(beyond.codes, ends.codes) and torch.equal(beyond.scales, ends.scales)
    nothing = mx.merge_rows(o.cuda(), ml, torch.full((t,), -1, dtype=torch.int32, device="cuda"), heads, 0, split_keys)
    assert torch.isnan(nothing.dequantize(F32)).all()
    if bad.any():  # a head that saw nothing: not a number, and its blocks
        assert np.isnan(got[bad]).all()
    keep = ~np.isnan(got)
    assert not bad.any() or keep.any()
    # sums over splits may cancel: what is off is off by a part of the sizes that went in, up to about 4 here
    unit = np.exp2(host(rows.scales).astype(np.float64) - 127).repeat(32, -1)[:, : heads * hd]
    step = unit * np.exp2(np.maximum(np.frexp(np.maximum(np.abs(got), np.abs(want)) / unit)[1] - 1, -6) - 3.0)
    assert (np.abs(got - want) <= step / 2 + ROWS_SLACK * 4)[keep].all()


# ---- the product -----------------------------------------------------------------------------------------------------


def product_operands(t, n, k, seed, gated=False):
    x, w = numbers(t, k, seed), numbers(n, k, seed + 1, F32, 0.05)
    xr, wp = mx.quantize_rows(x.cuda()), mx.pack_weight(w.cuda(), gated)
    return xr, wp, plain.values(x), plain.values(w, True)


def sum_bound(xv, wv):
    """Each of a sum's additions may lose a step of fp32 at most (a truncating adder), of no more than the sum of sizes."""
    k = xv.shape[1]
    return (k + 8) * 2.0**-23 * (np.abs(xv) @ np.abs(wv).T)


@pytest.mark.parametrize("t,n,k", [(1, 128, 128), (1, 1, 1), (3, 130, 257), (16, 128, 1024), (17, 300, 384), (33, 1152, 896), (64, 64, 2048), (65, 129, 640), (128, 256, 896), (200, 515, 1000), (257, 384, 512), (515, 200, 96)])
def test_linear(t, n, k):
    xr, wp, xv, wv = product_operands(t, n, k, 10)
    want, loose = xv @ wv.T, sum_bound(xv, wv)
    got = mx.linear(xr, wp, dtype=F32)
    assert got.shape == (t, n) and (np.abs(host(got) - want) <= loose).all()
    bias, add = torch.randn(n), torch.randn(t, n)
    got = mx.linear(xr, wp, bias=bias.cuda())
    assert got.dtype == BF16
    full = want + bias.double().numpy()
    assert (np.abs(host(got.float()) - full) <= loose * 1.01 + 2.0**-8 * np.abs(full) + 2.0**-22 * np.abs(bias.numpy())).all()
    h = add.cuda()
    got = mx.linear(xr, wp, bias=bias.cuda(), add=h, out=h)
    full += add.double().numpy()
    assert got is h and (np.abs(host(h) - full) <= loose + 2.0**-22 * (np.abs(want) + np.abs(bias.numpy()) + np.abs(add.numpy()))).all()


HOWS = [(bn, parts) for bn in (16, 32, 64, 128) for parts in (1, 2, 3, 5, 8)] + [(256, 1)]


@pytest.mark.parametrize("how", HOWS)
@pytest.mark.parametrize("t,n,k", [(70, 200, 1100), (300, 520, 1024), (9, 640, 2000)])
def test_every_tile_and_part(how, t, n, k):
    if how[1] > mx.padded(k) // 128:
        with pytest.raises(AlofaError):  # a part without a slice
            mx.linear(*product_operands(t, n, k, 20)[:2], how=how)
        return
    xr, wp, xv, wv = product_operands(t, n, k, 20)
    want, loose = xv @ wv.T, sum_bound(xv, wv)
    assert (np.abs(host(mx.linear(xr, wp, dtype=F32, how=how)) - want) <= loose).all()
    bias, add = torch.randn(n), torch.randn(t, n)
    full, size = want + bias.double().numpy() + add.double().numpy(), np.abs(want) + np.abs(bias.numpy()) + np.abs(add.numpy())
    got = mx.linear(xr, wp, bias=bias.cuda(), add=add.cuda(), dtype=BF16, how=how)
    assert (np.abs(host(got.float()) - full) <= 1.01 * loose + 2.0**-8 * np.abs(full) + 2.0**-22 * size).all()


@pytest.mark.parametrize("t,n,k", [(2100, 8000, 128), (1030, 10500, 384)])
def test_many_tiles_a_pair(t, n, k):
    """More tiles than pairs of CTAs: accumulators that share columns, a ring that runs on from tile to tile."""
    xr, wp, xv, wv = product_operands(t, n, k, 50)
    assert (np.abs(host(mx.linear(xr, wp, dtype=F32, how=(256, 1))) - xv @ wv.T) <= sum_bound(xv, wv)).all()
    f = n // 2
    xr, wp, xv, wv = product_operands(t, n, k, 52, gated=True)
    got = host(mx.gated_linear(xr, wp, how=(256, 1)).dequantize(F32)).astype(np.float64)
    g, u = xv @ wv[:f].T, xv @ wv[f:].T
    slope = 1.1 * np.abs(u) * sum_bound(xv, wv[:f]) + (np.abs(g) + 1) * sum_bound(xv, wv[f:])
    want = plain.silu(g) * u
    largest = np.abs(np.pad(want, ((0, 0), (0, -f % 32)))).reshape(t, -1, 32).max(-1).repeat(32, -1)[:, :f]
    # half a step of E4M3: 2^-4 of the number, or of the smallest normal number by a scale that is at most 2^-7 of the block's largest
    assert (np.abs(got - want) <= np.maximum(2.0**-4 * np.abs(want), 2.0**-17 * largest) * (1 + 2.0**-10) + slope).all()


def test_every_pair_of_codes():
    """Row t holds E4M3's code t in place t, feature f all of E2M1's codes in turn: each product stands alone in its sum."""
    codes = torch.zeros(254, 256, dtype=torch.uint8)
    every = torch.tensor([c for c in range(256) if c & 127 != 127], dtype=torch.uint8)
    codes[torch.arange(254), torch.arange(254)] = every
    scales = torch.full((254, 8), 127, dtype=torch.uint8)
    w = ((torch.arange(256)[None, :] + torch.arange(16)[:, None]) % 16).numpy()
    wp = mx.MxWeight.from_codes(torch.from_numpy(plain.nibbles(w)).cuda(), torch.full((16, 8), 127, dtype=torch.uint8).cuda(), 256)
    got = mx.linear(mx.MxRows(codes.cuda(), scales.cuda(), 256), wp, dtype=F32)
    want = plain.decode(codes, scales, 256, False) @ plain.decode(w, np.full((16, 8), 127), 256, True).T
    assert np.array_equal(host(got), want)


def test_scales_over_their_whole_range():
    """One number a block, scales from both ends: the product of the two powers is taken without a rounding."""
    codes = torch.zeros(20, 128, dtype=torch.uint8)
    codes[:, 0] = 0x38  # 1
    scales = torch.zeros(20, 4, dtype=torch.uint8)
    scales[:, 0] = torch.tensor([0, 1, 2, 30, 60, 90, 100, 110, 120, 126, 127, 128, 130, 140, 160, 180, 200, 220, 240, 250])
    ws = torch.zeros(20, 4, dtype=torch.uint8)
    ws[:, 0] = torch.tensor([127, 126, 128, 100, 200, 247, 1, 3, 10, 20, 30, 40, 50, 60, 70, 80, 90, 110, 140, 254])
    wc = np.zeros((20, 128), np.int64)
    wc[:, 0] = 2  # 1
    wp = mx.MxWeight.from_codes(torch.from_numpy(plain.nibbles(wc)).cuda(), ws.cuda(), 128)
    got = host(mx.linear(mx.MxRows(codes.cuda(), scales.cuda(), 128), wp, dtype=F32)).astype(np.float64)
    want = np.exp2(scales[:, :1].double().numpy() + ws[:, 0].double().numpy() - 254)
    normal = (want >= 2.0**-126) & (want < 2.0**128)
    assert np.array_equal(got[normal], want[normal])


@pytest.mark.parametrize("seed", range(24))
def test_any_size(seed):
    """Sizes drawn over the whole range, each the way the rule chooses."""
    rng = np.random.default_rng(seed)
    t, n, k = (int(np.exp(rng.uniform(0, np.log(most)))) for most in (1500, 3000, 4000))
    xr, wp, xv, wv = product_operands(t, n, k, 70 + seed)
    got = mx.linear(xr, wp, dtype=F32)
    assert (np.abs(host(got) - xv @ wv.T) <= sum_bound(xv, wv)).all(), (t, n, k)
    rows = mx.gated_linear(xr, mx.pack_weight(numbers(2 * n, k, 71 + seed, F32, 0.05).cuda(), True))
    wg = plain.values(numbers(2 * n, k, 71 + seed, F32, 0.05), True)
    g, u = xv @ wg[:n].T, xv @ wg[n:].T
    want, slope = plain.silu(g) * u, 1.1 * np.abs(u) * sum_bound(xv, wg[:n]) + (np.abs(g) + 1) * sum_bound(xv, wg[n:])
    largest = np.abs(np.pad(want, ((0, 0), (0, -n % 32)))).reshape(t, -1, 32).max(-1).repeat(32, -1)[:, :n]
    off = np.abs(host(rows.dequantize(F32)).astype(np.float64) - want)
    assert (off <= np.maximum(2.0**-4 * np.abs(want), 2.0**-17 * largest) * (1 + 2.0**-10) + slope).all(), (t, n, k)


def test_a_block_of_nan_reaches_its_row_only():
    xr, wp, xv, wv = product_operands(5, 140, 300, 30)
    xr.scales[2, 1] = 255  # a view of the rows' own memory
    got = host(mx.linear(xr, wp, dtype=F32))
    assert np.isnan(got[2]).all() and np.isfinite(got[[0, 1, 3, 4]]).all()


def test_rows_behind_the_last_are_left_alone():
    xr, wp, xv, wv = product_operands(5, 140, 300, 31)
    room = torch.full((20, 140), 7.0, device="cuda")
    mx.linear(xr, wp, out=room[:5])
    assert (room[5:] == 7).all() and (np.abs(host(room[:5]) - xv @ wv.T) <= sum_bound(xv, wv)).all()


@pytest.mark.parametrize("t,f,k,how", [(1, 16, 128, None), (3, 33, 100, None), (16, 4864, 896, None), (70, 200, 384, None), (300, 260, 256, None), (20, 64, 1024, (16, 8)), (33, 70, 700, (32, 3)), (40, 130, 640, (64, 2)), (130, 96, 640, (128, 5)),
                                       (7, 193, 512, (256, 1)), (513, 64, 256, (256, 1))])
@pytest.mark.parametrize("gate", [ops.SILU_GATE, (1.702, 7.0)])
def test_gated_linear(t, f, k, how, gate):
    xr, wp, xv, wv = product_operands(t, 2 * f, k, 40, gated=True)
    rows = mx.gated_linear(xr, wp, gate, how=how)
    g, u = xv @ wv[:f].T, xv @ wv[f:].T
    eg, eu = sum_bound(xv, wv[:f]), sum_bound(xv, wv[f:])
    if gate == ops.SILU_GATE:
        want, slope = plain.silu(g) * u, 1.1 * np.abs(u) * eg + (np.abs(g) + eg) * eu
    else:
        a, top = gate
        g, u = np.minimum(g, top), np.clip(u, -top, top)
        want, slope = g / (1 + np.exp(np.minimum(-a * g, 700))) * (u + 1), 1.1 * (np.abs(u) + 1) * eg + (np.abs(g) + eg) * eu
    got = host(rows.dequantize(F32)).astype(np.float64)
    assert rows.shape == (t, f) and not host(rows.codes)[:, f:].any()
    unit = np.exp2(host(rows.scales).astype(np.float64) - 127).repeat(32, -1)[:, :f]
    step = unit * np.exp2(np.maximum(np.frexp(np.maximum(np.abs(got), np.abs(want)) / unit)[1] - 1, -6) - 3.0)
    assert (np.abs(got - want) <= step / 2 + slope + ROWS_SLACK * np.abs(want)).all()
    # the scales are those of the numbers' own sizes
    full = np.zeros((t, plain.padded(f)))
    full[:, :f] = want
    pad = np.zeros_like(full)
    pad[:, :f] = slope + ROWS_SLACK * np.abs(want)
    sizes, room = np.abs(full).reshape(t, -1, 32), pad.reshape(t, -1, 32)
    scales = host(rows.scales)
    assert (scales >= plain.scale_bytes(np.maximum(sizes - room, 0).max(-1), False)).all() and (scales <= plain.scale_bytes((sizes + room).max(-1), False)).all()


@pytest.mark.parametrize("t,how", [(5, None), (40, None), (300, None), (5, (256, 1))])
@pytest.mark.parametrize("gate", [ops.SILU_GATE, (1.702, 7.0)])
def test_gated_rows_of_nan(t, how, gate):
    """Sums that are not numbers are none behind either gate, in their row only."""
    xr, wp, xv, wv = product_operands(t, 2 * 70, 300, 41, gated=True)
    xr.scales[2, 1] = 255
    got = host(mx.gated_linear(xr, wp, gate, how=how).dequantize(F32))
    assert np.isnan(got[2]).all() and np.isfinite(np.delete(got, 2, 0)).all()


def test_a_gate_near_the_largest_number():
    """silu(g) u of g = 1.75 2^127 (g log2(e) is beyond 32 bits) and u = 0.875: 1.53125 2^127, as a code 1.5 2^127."""
    x, w = torch.zeros(1, 32), torch.zeros(2, 32)
    x[0, 0], w[0, 0], w[1, 0] = 1.75 * 2.0**63, 2.0**64, 2.0**-64
    wp = mx.pack_weight(w.cuda(), True)
    for how in (None, (256, 1)):
        assert mx.gated_linear(x.cuda(), wp, how=how).dequantize(F32).item() == 1.5 * 2.0**127


def test_more_tokens_than_tiles_of_a_few():
    """So many tokens that the kernel for a few of them has no grid: they go by pairs."""
    t = 64 * mx.MOST_TILES + 3
    x = torch.zeros(t, 128, dtype=BF16, device="cuda")
    x[-1], x[-2] = 1, 2
    w = numbers(8, 128, 42)
    got, want = mx.linear(x, mx.pack_weight(w.cuda()), dtype=F32), plain.values(w.double().numpy(), True).sum(1)
    bound = 128 * 2.0**-23 * np.abs(plain.values(w.double().numpy(), True)).sum(1)
    assert (np.abs(host(got[-1]) - want) <= bound).all() and (np.abs(host(got[-2]) - 2 * want) <= 2 * bound).all() and not got[:-2].any()


# ---- as a program uses them ------------------------------------------------------------------------------------------


def chain(h, weight, w1, w2, owed):
    """A norm, a gated feed-forward and its sum into the stream: the operators one after another."""
    x = mx.norm_rows(h, weight, 1e-6, owed=owed)
    return mx.linear(mx.gated_linear(x, w1), w2, add=h)


def chain_operands(t, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    h, weight, owed = rnd(t, 384), 1 + 0.1 * rnd(384), rnd(1, t, 384)
    wg, wd = 0.05 * rnd(2 * 640, 384), 0.05 * rnd(384, 640)
    return h, weight, wg, wd, owed


@pytest.mark.parametrize("t", [1, 20, 150, 600])
def test_a_run_of_them_together(t):
    h, weight, wg, wd, owed = chain_operands(t, 1)
    h0 = h.clone()
    got = chain(h, weight, mx.pack_weight(wg, True), mx.pack_weight(wd), owed)
    f64 = lambda v: v.cpu().double().numpy()  # noqa: E731
    hh = f64(h0) + f64(owed[0])
    x = plain.values(plain.norm(hh, f64(weight), 1e-6))
    w = plain.values(wg.cpu(), True)
    g, u = x @ w[:640].T, x @ w[640:].T
    want = hh + plain.values(plain.silu(g) * u) @ plain.values(wd.cpu(), True).T
    # a number next to a border of two codes may take the other one, a step of 2^-3 of it at most: a few of them move a sum of
    # 640 products by a few times 2^-3 / sqrt(640) of its size, 0.5 % each
    size = np.sqrt((want - hh).std() ** 2)
    assert np.abs(f64(got) - want).max() <= 0.05 * size and np.sqrt(((f64(got) - want) ** 2).mean()) <= 0.003 * size
    assert (np.abs(f64(h) - hh) <= 2.0**-23 * (np.abs(f64(h0)) + np.abs(f64(owed[0])))).all()


def test_captured_and_replayed_on_new_inputs():
    t = 40
    h, weight, wg, wd, owed = chain_operands(t, 2)
    w1, w2 = mx.pack_weight(wg, True), mx.pack_weight(wd)
    want = [chain(h.clone().mul_(s), weight, w1, w2, owed).clone() for s in (1.0, 3.0, 0.01)]
    src, work = h.clone(), h.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(stream):
        work.copy_(src)
        chain(work, weight, w1, w2, owed)
        for _ in range(2):  # two graphs of the same calls: neither shares a workspace with the other
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                work.copy_(src)
                out = chain(work, weight, w1, w2, owed)
            graphs.append((graph, out))
    for scale, ref in zip((1.0, 3.0, 0.01), want):
        for graph, out in graphs:
            src.copy_(h * scale)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, ref)


def test_a_weight_packed_and_used_in_one_graph():
    """The product reads its weight ahead of the kernel before it; what packs one leaves it settled."""
    w = torch.randn(2, 1152, 896, device="cuda") * 0.05
    x = mx.quantize_rows(torch.randn(8, 896, device="cuda"))
    want = [mx.linear(x, mx.pack_weight(w[i])).clone() for i in range(2)]
    src = w[0].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        mx.linear(x, mx.pack_weight(src))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            packed = mx.pack_weight(src)
            out = mx.linear(x, packed)
    for i in (1, 0, 1, 1, 0) * 10:
        src.copy_(w[i])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


def test_two_streams_at_once():
    """The same weight and rows, other outputs, beside each other."""
    operands = [chain_operands(t, 5 + t) for t in (3, 300)]
    packed = [(mx.pack_weight(o[2], True), mx.pack_weight(o[3])) for o in operands]
    want = [chain(o[0].clone(), o[1], *p, o[4]) for o, p in zip(operands, packed)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in operands]
    got = [[] for _ in operands]
    hs = [[o[0].clone() for _ in range(20)] for o in operands]
    torch.cuda.synchronize()
    for k in range(20):
        for i, (o, p, s) in enumerate(zip(operands, packed, streams)):
            with torch.cuda.stream(s):
                got[i].append(chain(hs[i][k], o[1], *p, o[4]))
    torch.cuda.synchronize()
    for g, ref in zip(got, want):
        assert all(torch.equal(x, ref) for x in g)


def test_joined_splits_in_a_graph_on_another_stream():
    g = torch.Generator(device="cuda").manual_seed(21)
    po, ml = torch.randn(3, 4 * 5, 32, generator=g, device="cuda"), 1 + torch.rand(3, 4 * 5, 2, generator=g, device="cuda")
    at = torch.tensor([5, 64, 100, 191], dtype=torch.int32, device="cuda")
    want = mx.merge_rows(po, ml, at, 5, 0, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        aside = mx.merge_rows(po, ml, at, 5, 0, 64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mx.merge_rows(po, ml, at, 5, 0, 64)
    first = want.codes.clone()
    po.mul_(2)
    graph.replay()
    again = mx.merge_rows(po, ml, at, 5, 0, 64)
    assert torch.equal(aside.codes, first) and torch.equal(aside.scales, want.scales)
    assert torch.equal(got.codes, again.codes) and torch.equal(got.scales, again.scales) and torch.equal(again.scales[:, :5], want.scales[:, :5] + 1)  # five blocks of numbers; those behind the width are zeros, scale byte 0


def test_no_tokens():
    w, wg = mx.pack_weight(torch.randn(64, 96, device="cuda")), mx.pack_weight(torch.randn(64, 96, device="cuda"), True)
    x = mx.quantize_rows(torch.empty(0, 96, device="cuda"))
    assert x.dequantize().shape == (0, 96) and mx.linear(x, w).shape == (0, 64) and mx.gated_linear(x, wg).shape == (0, 32)
    assert mx.norm_rows(torch.empty(0, 96, device="cuda"), torch.ones(96, device="cuda"), 1e-6).shape == (0, 96)


def test_refusals():
    def refused(code, call, *args, **kw):
        with pytest.raises(AlofaError) as err:
            call(*args, **kw)
        assert err.value.code == code, err.value

    x, w = torch.randn(4, 96, device="cuda"), mx.pack_weight(torch.randn(64, 96, device="cuda"))
    wg, rows, ones = mx.pack_weight(torch.randn(64, 96, device="cuda"), True), mx.quantize_rows(x), torch.ones(96, device="cuda")
    refused("invalid_argument", mx.quantize_rows, x.half())
    refused("invalid_argument", mx.quantize_rows, x.t())
    refused("invalid_argument", mx.quantize_rows, [1.0])
    refused("invalid_argument", mx.quantize_rows, x[0])
    refused("invalid_argument", mx.quantize_rows, torch.empty(3, 0, device="cuda"))
    refused("unsupported", mx.quantize_rows, x.cpu())
    refused("invalid_argument", mx.pack_weight, torch.empty(0, 96, device="cuda"))
    refused("invalid_argument", mx.pack_weight, torch.randn(3, 96, device="cuda"), True)  # an odd number of rows
    refused("invalid_argument", mx.linear, rows, wg)
    refused("invalid_argument", mx.gated_linear, rows, w)
    refused("invalid_argument", mx.linear, rows, torch.randn(64, 96, device="cuda"))
    refused("invalid_argument", mx.linear, mx.quantize_rows(torch.randn(4, 128, device="cuda")), w)  # another depth
    refused("invalid_argument", mx.linear, rows, w, bias=torch.zeros(63, device="cuda"))
    refused("invalid_argument", mx.linear, rows, w, bias=torch.zeros(64, device="cuda").bfloat16())
    refused("invalid_argument", mx.linear, rows, w, add=torch.zeros(4, 65, device="cuda"))
    refused("invalid_argument", mx.linear, rows, w, out=torch.zeros(5, 64, device="cuda"))
    refused("unsupported", mx.linear, rows, w, dtype=torch.float16)
    refused("invalid_argument", mx.linear, rows, w, out=torch.zeros(4, 64, device="cuda"), dtype=BF16)
    refused("invalid_argument", mx.linear, rows, w, status=1)
    refused("invalid_argument", mx.gated_linear, rows, wg, (0.0, 7.0))
    refused("invalid_argument", mx.gated_linear, rows, wg, (1.702, 0.0))
    refused("unsupported", mx.linear, rows, w, how=(48, 1))
    refused("unsupported", mx.linear, rows, w, how=(16, 2))  # a part without a slice
    refused("unsupported", mx.linear, rows, w, how=(256, 2))
    refused("unsupported", rows.dequantize, torch.float16)
    refused("unsupported", w.dequantize, torch.float16)
    refused("invalid_argument", mx.norm_rows, x.bfloat16(), ones, 1e-6)
    refused("invalid_argument", mx.norm_rows, x, ones[:95], 1e-6)
    refused("invalid_argument", mx.norm_rows, x, ones, 1e-6, owed=torch.zeros(4, 96, device="cuda"))
    refused("invalid_argument", mx.norm_rows, x, ones, 1e-6, base=x[:3])
    refused("invalid_argument", mx.norm_rows, x, ones, 1e-6, shift=ones.double())
    refused("unsupported", mx.norm_rows, torch.zeros(1, mx.MOST_WIDTH + 128, device="cuda"), torch.ones(mx.MOST_WIDTH + 128, device="cuda"), 1e-6)
    refused("invalid_argument", mx.MxRows, rows.codes[:, :64].contiguous(), rows.scales, 96)
    refused("invalid_argument", mx.MxRows, rows.codes, rows.scales[:3], 96)
    refused("unsupported", mx.MxRows, torch.zeros(4 * 128 + 1, dtype=torch.uint8, device="cuda")[1:].view(4, 128), rows.scales, 96)  # off its alignment
    refused("invalid_argument", mx.MxWeight.from_codes, rows.codes, rows.scales, 300)
    refused("invalid_argument", w.first_rows, 65)
    po, ml, at = torch.zeros(2, 6, 16, device="cuda"), torch.zeros(2, 6, 2, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    mx.merge_rows(po, ml, at, 3, 0, 64)
    refused("invalid_argument", mx.merge_rows, po, ml, at, 4, 0, 64)
    refused("invalid_argument", mx.merge_rows, po[..., :12].contiguous(), ml, at, 3, 0, 64)
    refused("invalid_argument", mx.merge_rows, po, ml[:1], at, 3, 0, 64)
    refused("invalid_argument", mx.merge_rows, po, ml, at.long(), 3, 0, 64)
    refused("invalid_argument", mx.merge_rows, po, ml, at, 3, 0, 0)
    refused("invalid_argument", wg.first_rows, 3)


def test_rows_given_by_their_codes():
    x = numbers(9, 300, 60)
    made = mx.quantize_rows(x.cuda())
    again = mx.MxRows(made.codes.clone(), made.scales.clone(), 300)
    w = mx.pack_weight(numbers(130, 300, 61).cuda())
    assert torch.equal(mx.linear(made, w), mx.linear(again, w)) and torch.equal(made.dequantize(), again.dequantize())
    assert torch.equal(mx.linear(x.cuda(), w), mx.linear(made, w))  # a tensor of numbers is made rows first


def test_first_rows_of_a_weight():
    xr, wp, xv, wv = product_operands(5, 300, 256, 62)
    part = wp.first_rows(140)
    assert torch.equal(part.dequantize(), wp.dequantize()[:140].contiguous()) and torch.equal(mx.linear(xr, part), mx.linear(xr, wp)[:, :140].contiguous())


def test_the_widest_norm_and_a_deep_product():
    k = mx.MOST_WIDTH
    h, weight = numbers(2, k, 63), 1 + 0.1 * torch.randn(k)
    rows = mx.norm_rows(h.cuda(), weight.cuda(), 1e-6)
    assert plain.near(host(rows.codes), host(rows.scales), plain.norm(h.double().numpy(), weight.double().numpy(), 1e-6), ROWS_SLACK)
    xr, wp, xv, wv = product_operands(3, 128, 40000, 64)
    assert (np.abs(host(mx.linear(xr, wp, dtype=F32)) - xv @ wv.T) <= sum_bound(xv, wv)).all()


def test_status_is_left_alone():
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for t in (4, 300):
        xr, wp, _, _ = product_operands(t, 300, 256, 65)
        mx.linear(xr, wp, status=status)
    assert int(status) == 0


def test_launches_are_counted():
    from alofa_b200.csrc import ops

    x, w = torch.randn(4, 96, device="cuda"), torch.randn(64, 96, device="cuda")
    for call, launches in ((lambda: mx.pack_weight(w), 2), (lambda: mx.quantize_rows(x), 1), (lambda: mx.quantize_rows(x).dequantize(), 2), (lambda: mx.norm_rows(x, torch.ones(96, device="cuda"), 1e-6), 1)):
        before = ops.launch_count()
        call()
        assert ops.launch_count() - before == launches
