"""Microscaled numbers: weights in 4 bits, rows in 8 bits, and their product.

Numbers along the depth stand in blocks of 32 that share a power of two, kept
as a byte ``s`` that means ``2^(s - 127)`` (255: the block is not a number).
Rows are E4M3 with the smallest scale that clips nothing, weights E2M1 with the
scale ``2^(floor(log2(largest)) - 2)``, what is over 6 by it becoming 6; both
round to nearest, ties to the even code.  A weight so takes 4.25 bits a number.

    w = mx.pack_weight(weight)                     # [N, K] bfloat16 or float32, once
    x = mx.norm_rows(h, norm_weight, 1e-6)         # h [T, K] float32: its RMSNorm in 8 bits
    y = mx.linear(x, w, bias=b)                    # [T, N] bfloat16

:func:`quantize_rows` makes rows of any tensor, :func:`gated_linear` takes rows
through a gate and an up projection (``pack_weight(..., gated=True)``) and gives
rows again.  Everything runs on the current stream of the device that the
tensors are on, which has to be the current one; what is returned belongs to
that stream.  The engine uses these operators where it is given
``weight_format="mxfp4"``."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .csrc import ops
from .errors import AlofaError

TOKEN_TILES = (16, 32, 64, 128, 256)  # tokens a CTA of the product may take


def _check(t, name: str, dims: int, dtypes: tuple) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.dim() != dims or t.dtype not in dtypes:
        got = f"{t.dtype} {tuple(t.shape)}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise AlofaError("invalid_argument", f"{name} must be a tensor of {dims} dimensions", f"got {got}, want one of {[str(d) for d in dtypes]}")
    if not t.is_cuda:
        raise AlofaError("unsupported", "kernels run on CUDA tensors only", f"{name} is on {t.device}")
    if t.device.index != torch.cuda.current_device():
        raise AlofaError("invalid_argument", "kernels run on the current device only", f"{name} is on {t.device}, current is {torch.cuda.current_device()}")
    if not t.is_contiguous():
        raise AlofaError("invalid_argument", "kernel operand must be contiguous", name)
    return t


_NUMBERS, _F32, _BYTES = (torch.bfloat16, torch.float32), (torch.float32,), (torch.uint8,)


@dataclass
class MxRows:
    """Rows ``[T, width]`` in 8 bits: ``codes`` uint8 ``[T, Kp]`` (E4M3) and
    ``scales`` uint8 ``[T, Kp / 32]``, Kp being the width rounded up to 128;
    the codes behind the width are zeros."""

    codes: torch.Tensor
    scales: torch.Tensor
    width: int

    def __post_init__(self):
        t, kp = self.codes.shape[0], ops.mx_padded(self.width)
        if self.width <= 0 or tuple(self.codes.shape) != (t, kp) or tuple(self.scales.shape) != (t, kp // ops.MX_BLOCK):
            raise AlofaError("invalid_argument", "rows in 8 bits have the wrong size", f"codes={tuple(self.codes.shape)} scales={tuple(self.scales.shape)} width={self.width}")
        _check(self.codes, "codes", 2, _BYTES), _check(self.scales, "scales", 2, _BYTES)

    @classmethod
    def empty(cls, rows: int, width: int, device=None, buf=None) -> "MxRows":
        """Room for rows, from ``buf(shape, dtype)`` (a step's scratch) or new."""
        kp = ops.mx_padded(width)
        make = buf or (lambda shape, dtype: torch.empty(shape, dtype=dtype, device=device or "cuda"))
        return cls(make((rows, kp), torch.uint8), make((rows, kp // ops.MX_BLOCK), torch.uint8), width)

    @property
    def shape(self) -> tuple:
        return self.codes.shape[0], self.width

    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        """The numbers that the rows stand for (bfloat16 has them all, but for some below 2^-133)."""
        out = torch.empty(self.shape, dtype=dtype, device=self.codes.device)
        ops.mx_rows_values(_check(out, "out", 2, _NUMBERS), self.codes, self.scales)
        return out


@dataclass
class MxWeight:
    """A weight ``[n, k]`` in 4 bits, laid out in tiles of 128 rows and 128
    numbers as the product reads them.  ``gated``: the first half of the rows
    are a gate's, the second an up projection's."""

    tiles: torch.Tensor
    n: int
    k: int
    gated: bool = False

    @classmethod
    def empty(cls, n: int, k: int, gated: bool, device) -> "MxWeight":
        if n <= 0 or k <= 0 or (gated and n % 2):
            raise AlofaError("invalid_argument", "a weight has rows and a depth, a gated one an even number of rows", f"rows={n} depth={k} gated={gated}")
        shape = (-(-ops.mx_weight_rows(n, gated) // ops.MX_TILE_ROWS), ops.mx_padded(k) // ops.MX_GROUP, ops.MX_TILE_BYTES)
        return cls(torch.empty(shape, dtype=torch.uint8, device=device), n, k, gated)

    @classmethod
    def from_codes(cls, codes, scales, k: int, gated: bool = False) -> "MxWeight":
        """A weight that is in 4 bits already: ``codes`` uint8 ``[n, >= k / 2]``,
        two numbers a byte with the first in its low half, and ``scales`` uint8
        ``[n, >= k / 32]``; what they hold behind ``k`` is not read."""
        _check(codes, "codes", 2, _BYTES), _check(scales, "scales", 2, _BYTES)
        n = codes.shape[0]
        if scales.shape[0] != n or codes.shape[1] < -(-k // 2) or scales.shape[1] < -(-k // ops.MX_BLOCK):
            raise AlofaError("invalid_argument", "a weight's codes and scales disagree", f"codes={tuple(codes.shape)} scales={tuple(scales.shape)} depth={k}")
        w = cls.empty(n, k, gated, codes.device)
        tall, slices, _ = w.tiles.shape
        c = codes.new_zeros((tall * ops.MX_TILE_ROWS, slices * ops.MX_GROUP // 2))
        s = codes.new_zeros((tall * ops.MX_TILE_ROWS, slices * ops.MX_GROUP // ops.MX_BLOCK))
        half, blocks = -(-k // 2), -(-k // ops.MX_BLOCK)
        if gated:  # the gate's and the up projection's features in turns of 16
            f = torch.arange(n // 2, device=codes.device)
            at = f // ops.MX_GATE_ROWS * (2 * ops.MX_GATE_ROWS) + f % ops.MX_GATE_ROWS
            at = torch.cat([at, at + ops.MX_GATE_ROWS])
        else:
            at = torch.arange(n, device=codes.device)
        c[at, :half], s[at, :blocks] = codes[:, :half], scales[:, :blocks]
        if k % 2:
            c[:, k // 2] &= 15
        size = ops.MX_TILE_ROWS * ops.MX_GROUP // 2
        w.tiles[:, :, :size] = c.view(tall, ops.MX_TILE_ROWS, slices, ops.MX_GROUP // 2).permute(0, 2, 1, 3).reshape(tall, slices, size)
        w.tiles[:, :, size:] = s.view(tall, 4, 32, slices, 4).permute(0, 3, 2, 1, 4).reshape(tall, slices, ops.MX_TILE_BYTES - size)
        ops.mx_settle()
        return w

    @property
    def rows(self) -> int:
        """Rows of the product: a gated weight's features are padded to whole turns of 16."""
        return ops.mx_weight_rows(self.n, self.gated)

    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        """The numbers ``[n, k]`` that the weight stands for."""
        out = torch.empty((self.n, self.k), dtype=dtype, device=self.tiles.device)
        ops.mx_weight_values(_check(out, "out", 2, _NUMBERS), self.tiles, self.gated)
        return out


def pack_weight(w: torch.Tensor, gated: bool = False) -> MxWeight:
    """``w [N, K]`` (bfloat16 or float32) in 4 bits; ``gated``: a gate's N / 2
    rows above an up projection's, for :func:`gated_linear`."""
    _check(w, "w", 2, _NUMBERS)
    out = MxWeight.empty(w.shape[0], w.shape[1], gated, w.device)
    ops.mx_pack(out.tiles, w, gated)
    return out


def quantize_rows(x: torch.Tensor, buf=None) -> MxRows:
    """``x [T, K]`` (bfloat16 or float32) as rows in 8 bits."""
    _check(x, "x", 2, _NUMBERS)
    rows = MxRows.empty(x.shape[0], x.shape[1], x.device, buf)
    ops.mx_rows(rows.codes, rows.scales, x)
    return rows


def norm_rows(h: torch.Tensor, weight: torch.Tensor, eps: float, base=None, owed=None, bias=None, shift=None, buf=None) -> MxRows:
    """``h = base + sum_z owed[z] + bias`` (``base``: h itself unless given;
    all float32), in place, and the RMSNorm of its rows times ``weight`` in 8
    bits: ``h / sqrt(mean(h^2) + eps) * weight``.  With ``shift`` the layer
    norm, ``(h - mean) / sqrt(variance + eps) * weight + shift``.  ``owed
    [splits, T, K]`` are the sums that a product left (:func:`linear_parts`)."""
    _check(h, "h", 2, _F32), _check(weight, "weight", 1, _F32)
    for t, name, dims in ((base, "base", 2), (owed, "owed", 3), (bias, "bias", 1), (shift, "shift", 1)):
        if t is not None:
            _check(t, name, dims, _F32)
    rows = MxRows.empty(h.shape[0], h.shape[1], h.device, buf)
    ops.mx_norm(rows.codes, rows.scales, h, weight, eps, base, owed, bias, shift)
    return rows


def _operands(x, w, what: str, gated: bool, buf):
    if not isinstance(w, MxWeight) or w.gated != gated:
        raise AlofaError("invalid_argument", f"{what} takes a weight that was packed for it", f"gated={getattr(w, 'gated', None)} want={gated}")
    _check(w.tiles, "w", 3, _BYTES)
    if not isinstance(x, MxRows):
        x = quantize_rows(x, buf)
    if x.width != w.k:
        raise AlofaError("invalid_argument", f"{what}: rows and weight differ in depth", f"rows={x.width} weight={w.k}")
    _check(x.codes, "x", 2, _BYTES)
    return x


def plan(tokens: int, rows: int, depth: int) -> tuple:
    """(tokens a tile, parts of the depth) of a product."""
    bn = next((b for b in TOKEN_TILES if tokens <= b), TOKEN_TILES[-1])
    ctas = -(-rows // ops.MX_TILE_ROWS) * -(-tokens // bn)
    slices = ops.mx_padded(depth) // ops.MX_GROUP
    room = 148 * (1 if bn == 256 else 2)
    return bn, ops.mx_splits(depth, max(1, min(slices, room // ctas)))


def _room(shape, device, buf):
    return buf(shape, torch.float32) if buf is not None else torch.empty(shape, dtype=torch.float32, device=device)


def linear(x, w: MxWeight, bias=None, add=None, out=None, dtype=None, buf=None, status=None) -> torch.Tensor:
    """``out = x w^T (+ bias) (+ add)``.  ``x``: rows in 8 bits, or a tensor
    that is made such rows first; ``bias [N]``, ``add [T, N]`` float32
    (``add`` may be ``out``).  ``out`` (or ``dtype``): bfloat16 unless ``add``
    is given, else float32."""
    x = _operands(x, w, "linear", False, buf)
    t = x.shape[0]
    for v, name, dims in ((bias, "bias", 1), (add, "add", 2)):
        if v is not None:
            _check(v, name, dims, _F32)
    if out is None:
        out = torch.empty((t, w.n), dtype=dtype or (torch.bfloat16 if add is None else torch.float32), device=w.tiles.device)
    _check(out, "out", 2, _NUMBERS)
    bn, splits = plan(t, w.rows, w.k)
    partial = _room((splits, t, w.rows), w.tiles.device, buf) if splits > 1 else None
    ops.mx_gemm(out, x.codes, x.scales, w.tiles, w.n, w.k, bn, splits, partial, bias=bias, add=add, status=status)
    return out


def linear_parts(x, w: MxWeight, buf=None, status=None) -> torch.Tensor:
    """The sums of ``x w^T`` for each part of the depth, ``[parts, T, N]``
    float32, for a reader that adds them (:func:`norm_rows`)."""
    x = _operands(x, w, "linear_parts", False, buf)
    bn, splits = plan(x.shape[0], w.rows, w.k)
    sums = _room((splits, x.shape[0], w.rows), w.tiles.device, buf)
    ops.mx_gemm(None, x.codes, x.scales, w.tiles, w.n, w.k, bn, splits, sums, leave=True, status=status)
    return sums


def gated_linear(x, w: MxWeight, gate=ops.SILU_GATE, buf=None, status=None) -> MxRows:
    """``silu(x Wg^T) * (x Wu^T)`` as rows in 8 bits; ``gate`` = (alpha,
    limit): the clamped form ``g = min(g, limit), u = clamp(u, -limit, limit):
    g sigmoid(alpha g) (u + 1)``."""
    x = _operands(x, w, "gated_linear", True, buf)
    t = x.shape[0]
    rows = MxRows.empty(t, w.n // 2, w.tiles.device, buf)
    bn, splits = plan(t, w.rows, w.k)
    sums = _room((splits, t, w.rows), w.tiles.device, buf)
    ops.mx_gemm(None, x.codes, x.scales, w.tiles, w.n, w.k, bn, splits, sums, leave=True, gated=True, status=status)
    ops.mx_gate(rows.codes, rows.scales, sums, w.n // 2, gate)
    return rows
