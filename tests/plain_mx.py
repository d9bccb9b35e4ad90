"""Microscaled numbers from their definition, in 64 bits: every code's value in
a table, the nearest found among all of them."""
import numpy as np
import torch

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m / 512 for m in range(8)] + [(8 + m) / 8 * 2.0**e for e in range(-6, 9) for m in range(8)][:-1])


def padded(k):
    return -(-k // 128) * 128


def scale_bytes(largest, weights):
    """The scale of a block by its largest magnitude (float64): 255 where that is no number."""
    out = np.zeros(largest.shape, np.int64)
    bad = ~np.isfinite(largest)
    ok = ~bad & (largest > 0)
    m, e = np.frexp(largest[ok])  # largest = m 2^e, m in [1/2, 1)
    power = e - 1 - 2 if weights else e - 9 + (m > 0.875)  # 448 = 0.875 * 2^9
    out[ok] = np.maximum(power + 127, 0)
    out[bad] = 255
    return out


def encode(x, weights):
    """(codes, scale bytes) of rows x [T, K]: int64 [T, Kp], [T, Kp / 32]."""
    x = np.asarray(x.double().cpu()) if isinstance(x, torch.Tensor) else np.asarray(x, np.float64)
    t, k = x.shape
    b = np.zeros((t, padded(k)))
    b[:, :k] = x
    b = b.reshape(t, -1, 32)
    scales = scale_bytes(np.abs(b).max(-1), weights)  # a NaN comes out of max as itself
    table = E2M1 if weights else E4M3
    with np.errstate(invalid="ignore", over="ignore"):
        v = np.where((scales == 255)[..., None], 0.0, b * np.exp2(127.0 - scales)[..., None])
    size = np.minimum(np.abs(v), table[-1])
    above = np.minimum(np.searchsorted(table, size), len(table) - 1)
    below = np.maximum(above - 1, 0)
    up, down = table[above] - size, size - table[below]
    code = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    code = code + np.where(np.signbit(v), 8 if weights else 128, 0)
    return code.reshape(t, -1), scales


def decode(codes, scales, k, weights):
    """The numbers that codes [T, Kp] with scale bytes stand for, float64 [T, k]."""
    codes, scales = np.asarray(codes, np.int64), np.asarray(scales, np.int64)
    sign = 8 if weights else 128
    table = E2M1 if weights else np.append(E4M3, np.nan)
    v = table[codes & (sign - 1)] * np.where(codes & sign, -1.0, 1.0)
    power = np.where(scales == 255, np.nan, np.exp2(scales - 127.0))
    return (v.reshape(v.shape[0], -1, 32) * power[..., None]).reshape(v.shape[0], -1)[:, :k]


def values(x, weights=False):
    codes, scales = encode(x, weights)
    return decode(codes, scales, x.shape[1], weights)


def nibbles(codes):
    """Two codes a byte, the first in the low half."""
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def norm(h, weight, eps, shift=None):
    mean = h.mean(-1, keepdims=True) if shift is not None else 0.0
    y = (h - mean) / np.sqrt(((h - mean) ** 2).mean(-1, keepdims=True) + eps) * weight
    return y if shift is None else y + shift


def silu(g):
    return g / (1 + np.exp(-np.maximum(g, -700)))  # below it is zero in 64 bits too


def near(codes, scales, y, slack):
    """Whether rows in 8 bits are y [T, K] rounded, where what was rounded may be off y by ``slack`` of its size (and of the
    block's largest for nothing): each scale is one that a largest number within that slack has, each number within half a
    step of E4M3 by that scale."""
    codes, scales = np.asarray(codes, np.int64), np.asarray(scales, np.int64)
    t, k = y.shape
    kp = padded(k)
    full = np.zeros((t, kp))
    full[:, :k] = y
    largest = np.abs(full.reshape(t, -1, 32)).max(-1)
    low, high = scale_bytes(largest * (1 - slack), False), scale_bytes(largest * (1 + slack), False)
    if not ((scales >= low) & (scales <= high)).all():
        return False
    got = decode(codes, scales, kp, False)
    unit = np.exp2(scales - 127.0).repeat(32, -1).reshape(t, kp)
    e = np.maximum(np.frexp(np.abs(got) / unit)[1] - 1, -6)  # the step above a number; half of it is the most a rounding is off by
    return bool((np.abs(got - full) <= unit * np.exp2(e - 3.0) / 2 + slack * np.abs(full)).all())
