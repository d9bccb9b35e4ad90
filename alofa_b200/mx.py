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
that stream.  Operands are contiguous.  The engine uses these operators where it
is given ``weight_format="mxfp4"``.

A call of the smallest sizes is a few microseconds of launching and checking
beside as much of the GPU's time: operands are checked once each, in one pass
over what a launch goes by, and rows are one allocation."""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from .csrc import ops
from .errors import AlofaError

BLOCK, GROUP, TILE_ROWS, TILE_BYTES, GATE_ROWS = 32, 128, 128, 8704, 16  # as in kernels/mx.cuh
MOST_WIDTH = 32768  # numbers of a row that the norm takes
MOST_TILES = 65535  # of tokens that the product for a few of them takes

_BF16, _F32, _U8, _I32 = torch.bfloat16, torch.float32, torch.uint8, torch.int32


def _refuse(t, name: str, want: str, here: int):
    if not isinstance(t, torch.Tensor):
        raise AlofaError("invalid_argument", f"{name} must be a tensor", f"got {type(t).__name__}")
    if not t.is_cuda:
        raise AlofaError("unsupported", "kernels run on CUDA tensors only", f"{name} is on {t.device}")
    if t.get_device() != here:
        raise AlofaError("invalid_argument", "kernels run on the current device only", f"{name} is on {t.device}, current is {here}")
    if not t.is_contiguous():
        raise AlofaError("invalid_argument", "kernel operand must be contiguous", name)
    raise AlofaError("invalid_argument", "kernel operand has the wrong type or size", f"{name} is {t.dtype} {tuple(t.shape)}, want {want}")


def _at(t, name: str, dtype, shape, here: int) -> int:
    """The address of an operand of this type and shape on the current device."""
    if not isinstance(t, torch.Tensor) or t.get_device() != here or t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        _refuse(t, name, f"{dtype} {tuple(shape)}", here)
    return t.data_ptr()


def _matrix(t, name: str, here: int) -> tuple:
    """(address, rows, columns, whether bfloat16) of a matrix in one of the compute types."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.get_device() != here or not t.is_contiguous() or (t.dtype is not _BF16 and t.dtype is not _F32):
        _refuse(t, name, "bfloat16 or float32 of two dimensions", here)
    rows, columns = t.shape
    return t.data_ptr(), rows, columns, t.dtype is _BF16


def _here() -> int:
    try:
        return torch._C._cuda_getDevice()
    except (RuntimeError, AttributeError):  # CUDA is not initialised yet, or there is none
        pass
    try:
        return torch.cuda.current_device()
    except (RuntimeError, AssertionError) as err:
        raise AlofaError("unsupported", "kernels run on CUDA tensors only", str(err)) from err


_stream = ops.current_stream_handle


class _Library:
    """The library's functions, looked up once each."""

    def __getattr__(self, name: str):
        fn = getattr(ops.mx_library(), name)
        setattr(self, name, fn)
        return fn


_lib = _Library()


def padded(k: int) -> int:
    """A depth rounded up to whole groups: the width of the codes of rows."""
    return -(-k // GROUP) * GROUP


class MxRows:
    """Rows ``[T, width]`` in 8 bits: ``codes`` uint8 ``[T, Kp]`` (E4M3) and
    ``scales`` uint8 ``[T, Kp / 32]``, Kp being the width rounded up to 128;
    the codes behind the width are zeros."""

    __slots__ = ("_data", "_codes", "_scales", "rows", "width", "device", "codes_at", "scales_at")

    def __init__(self, codes, scales, width: int):
        here = _here()
        if width <= 0 or not isinstance(codes, torch.Tensor) or codes.dim() != 2:
            raise AlofaError("invalid_argument", "rows in 8 bits are a matrix of codes", f"width={width}")
        self._data, self._codes, self._scales = None, codes, scales
        self.rows, self.width, self.device, kp = codes.shape[0], width, here, padded(width)
        self.codes_at = _at(codes, "codes", _U8, (self.rows, kp), here)
        self.scales_at = _at(scales, "scales", _U8, (self.rows, kp // BLOCK), here)
        if self.codes_at % 16 or self.scales_at % 4:
            raise AlofaError("unsupported", "codes must start on a 16-byte boundary, scales on one of 4", f"codes={self.codes_at % 16} scales={self.scales_at % 4}")

    @classmethod
    def _empty(cls, rows: int, width: int, here: int, buf) -> "MxRows":
        """Room for rows, from ``buf(shape, dtype)`` (a step's scratch) or new."""
        self = cls.__new__(cls)
        kp = -(-width // GROUP) * GROUP
        size = rows * (kp + kp // BLOCK)
        self._data = torch.empty(size, dtype=_U8, device=here) if buf is None else buf((size,), _U8)
        self._codes = self._scales = None
        self.rows, self.width, self.device = rows, width, here
        self.codes_at = self._data.data_ptr()
        self.scales_at = self.codes_at + rows * kp
        return self

    def __reduce__(self):  # a copy knows where its own memory is
        return MxRows, (self.codes, self.scales, self.width)

    @property
    def shape(self) -> tuple:
        return self.rows, self.width

    @property
    def codes(self) -> torch.Tensor:
        return self._codes if self._data is None else self._data[: self.rows * padded(self.width)].view(self.rows, -1)

    @property
    def scales(self) -> torch.Tensor:
        return self._scales if self._data is None else self._data[self.rows * padded(self.width) :].view(self.rows, -1)

    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        """The numbers that the rows stand for (bfloat16 has them all, but for some below 2^-133)."""
        here = _on(self, "rows", _here())
        if dtype is not _BF16 and dtype is not _F32:
            raise AlofaError("unsupported", "numbers come in bfloat16 or float32", f"dtype={dtype}")
        out = (self._codes if self._data is None else self._data).new_empty((self.rows, self.width), dtype=dtype)
        rc = _lib.alofa_mx_rows_values(out.data_ptr(), self.codes_at, self.scales_at, self.rows, self.width, dtype is _BF16, _stream(here))
        ops.mx_launched(rc, 1 if self.rows else 0, "mx rows' values", lambda: f"rows={self.rows} width={self.width}")
        return out


def _on(v, name: str, here: int) -> int:
    if v.device != here:
        raise AlofaError("invalid_argument", "kernels run on the current device only", f"{name} is on cuda:{v.device}, current is {here}")
    return here


class MxWeight:
    """A weight ``[n, k]`` in 4 bits, laid out in tiles of 128 rows and 128
    numbers as the product reads them.  ``gated``: the first half of the rows
    are a gate's, the second an up projection's.  Made by :func:`pack_weight`
    or :meth:`from_codes`, and constant from then on: products read it ahead of
    the kernel before them in the stream."""

    __slots__ = ("tiles", "n", "k", "gated", "rows", "device", "at", "maps", "maps_at")

    def __init__(self, n: int, k: int, gated: bool, here: int):
        if n <= 0 or k <= 0 or (gated and n % 2):
            raise AlofaError("invalid_argument", "a weight has rows and a depth, a gated one an even number of rows", f"rows={n} depth={k} gated={gated}")
        self.n, self.k, self.gated, self.device = n, k, bool(gated), here
        #: rows of the product: a gated weight's features stand in turns of 16, padded to whole turns
        self.rows = 2 * (-(-(n // 2) // GATE_ROWS) * GATE_ROWS) if gated else n
        self.tiles = torch.empty((-(-self.rows // TILE_ROWS), padded(k) // GROUP, TILE_BYTES), dtype=_U8, device=here)
        self.at = self.tiles.data_ptr()
        #: how the copies of the product see the tiles (two tensor maps)
        self.maps = ctypes.create_string_buffer(256)
        self.maps_at = ctypes.addressof(self.maps)
        ops.mx_launched(_lib.alofa_mx_weight_maps(self.maps, self.at, self.tiles.shape[0] * self.tiles.shape[1]), 0, "mx weight", lambda: f"rows={n} depth={k}")

    @classmethod
    def from_codes(cls, codes, scales, k: int, gated: bool = False) -> "MxWeight":
        """A weight that is in 4 bits already: ``codes`` uint8 ``[n, >= k / 2]``,
        two numbers a byte with the first in its low half, and ``scales`` uint8
        ``[n, >= k / 32]``; what they hold behind ``k`` is not read."""
        here = _here()
        for t, name in ((codes, "codes"), (scales, "scales")):
            if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.dtype is not _U8 or t.get_device() != here:
                _refuse(t, name, "uint8 of two dimensions", here)
        n = codes.shape[0]
        if scales.shape[0] != n or codes.shape[1] < -(-k // 2) or scales.shape[1] < -(-k // BLOCK):
            raise AlofaError("invalid_argument", "a weight's codes and scales disagree", f"codes={tuple(codes.shape)} scales={tuple(scales.shape)} depth={k}")
        w = cls(n, k, gated, here)
        tall, slices, _ = w.tiles.shape
        c = codes.new_zeros((tall * TILE_ROWS, slices * GROUP // 2))
        s = codes.new_zeros((tall * TILE_ROWS, slices * GROUP // BLOCK))
        half, blocks = -(-k // 2), -(-k // BLOCK)
        if gated:  # the gate's and the up projection's features in turns of 16
            f = torch.arange(n // 2, device=codes.device)
            at = f // GATE_ROWS * (2 * GATE_ROWS) + f % GATE_ROWS
            at = torch.cat([at, at + GATE_ROWS])
        else:
            at = torch.arange(n, device=codes.device)
        c[at, :half], s[at, :blocks] = codes[:, :half], scales[:, :blocks]
        if k % 2:
            c[:, k // 2] &= 15
        size = TILE_ROWS * GROUP // 2
        w.tiles[:, :, :size] = c.view(tall, TILE_ROWS, slices, GROUP // 2).permute(0, 2, 1, 3).reshape(tall, slices, size)
        w.tiles[:, :, size:] = s.view(tall, 4, 32, slices, 4).permute(0, 3, 2, 1, 4).reshape(tall, slices, TILE_BYTES - size)
        # the product reads tiles ahead of the kernel before it
        ops.mx_launched(_lib.alofa_mx_settle(_stream(here)), 1, "mx weight", str)
        return w

    def __copy__(self) -> "MxWeight":
        return self  # constant

    def __reduce__(self):  # a copy knows where its own memory is
        return _weight_of_tiles, (self.tiles, self.n, self.k, self.gated)

    def first_rows(self, n: int) -> "MxWeight":
        """The weight's first ``n`` rows, in the same memory."""
        if self.gated or not 0 < n <= self.n:
            raise AlofaError("invalid_argument", "the first rows of a weight that is not gated", f"rows={n} of {self.n} gated={self.gated}")
        part = MxWeight.__new__(MxWeight)
        part.n, part.rows, part.k, part.gated, part.device = n, n, self.k, False, self.device
        part.tiles, part.at, part.maps, part.maps_at = self.tiles[: -(-n // TILE_ROWS)], self.at, self.maps, self.maps_at
        return part

    def dequantize(self, dtype=torch.bfloat16) -> torch.Tensor:
        """The numbers ``[n, k]`` that the weight stands for."""
        here = _on(self, "weight", _here())
        if dtype is not _BF16 and dtype is not _F32:
            raise AlofaError("unsupported", "numbers come in bfloat16 or float32", f"dtype={dtype}")
        out = self.tiles.new_empty((self.n, self.k), dtype=dtype)
        rc = _lib.alofa_mx_weight_values(out.data_ptr(), self.at, self.n, self.k, self.gated, dtype is _BF16, _stream(here))
        ops.mx_launched(rc, 1, "mx weight's values", lambda: f"rows={self.n} depth={self.k}")
        return out


def _weight_of_tiles(tiles, n: int, k: int, gated: bool) -> MxWeight:
    here = _here()
    w = MxWeight(n, k, gated, here)
    w.tiles.copy_(tiles)
    ops.mx_launched(_lib.alofa_mx_settle(_stream(here)), 1, "mx weight", str)  # as in from_codes
    return w


def pack_weight(w: torch.Tensor, gated: bool = False) -> MxWeight:
    """``w [N, K]`` (bfloat16 or float32) in 4 bits; ``gated``: a gate's N / 2
    rows above an up projection's, for :func:`gated_linear`."""
    here = _here()
    at, n, k, bf16 = _matrix(w, "w", here)
    out = MxWeight(n, k, gated, here)
    rc = _lib.alofa_mx_pack(out.at, at, n, k, out.gated, bf16, _stream(here))
    ops.mx_launched(rc, 2, "pack_weight", lambda: f"rows={n} depth={k}")
    return out


def quantize_rows(x: torch.Tensor, buf=None) -> MxRows:
    """``x [T, K]`` (bfloat16 or float32) as rows in 8 bits."""
    here = _here()
    at, t, k, bf16 = _matrix(x, "x", here)
    if not k:
        raise AlofaError("invalid_argument", "rows have a width", "width=0")
    rows = MxRows._empty(t, k, here, buf)
    rc = _lib.alofa_mx_rows(rows.codes_at, rows.scales_at, at, t, k, bf16, _stream(here))
    ops.mx_launched(rc, 1 if t else 0, "quantize_rows", lambda: f"rows={t} width={k}")
    return rows


def norm_rows(h: torch.Tensor, weight: torch.Tensor, eps: float, base=None, owed=None, bias=None, shift=None, buf=None) -> MxRows:
    """``h = base + sum_z owed[z] + bias`` (``base``: h itself unless given;
    all float32), in place, and the RMSNorm of its rows times ``weight`` in 8
    bits: ``h / sqrt(mean(h^2) + eps) * weight``.  With ``shift`` the layer
    norm, ``(h - mean) / sqrt(variance + eps) * weight + shift``.  ``owed
    [splits, T, K]`` are sums that products left, for parts of their depth or whole."""
    here = _here()
    at, t, k, bf16 = _matrix(h, "h", here)
    if bf16 or not k:
        _refuse(h, "h", "float32 of two dimensions", here)
    splits = owed.shape[0] if isinstance(owed, torch.Tensor) and owed.dim() else 0
    rows = MxRows._empty(t, k, here, buf)
    rc = _lib.alofa_mx_norm(
        rows.codes_at, rows.scales_at, at, at if base is None else _at(base, "base", _F32, (t, k), here), None if owed is None else _at(owed, "owed", _F32, (splits, t, k), here), splits,
        None if bias is None else _at(bias, "bias", _F32, (k,), here), _at(weight, "weight", _F32, (k,), here), None if shift is None else _at(shift, "shift", _F32, (k,), here), t, k, eps, _stream(here),
    )
    ops.mx_launched(rc, 1 if t else 0, "norm_rows", lambda: f"rows={t} width={k} most={MOST_WIDTH}")
    return rows


def merge_rows(partial_o, partial_ml, positions, heads: int, window: int, split_keys: int, buf=None) -> MxRows:
    """The attention output of decode tokens whose keys were split
    (``partial_o [splits, T * heads, head_dim]``, ``partial_ml [splits, T *
    heads, 2]``: each split's maximum, in log2 units, and sum; float32), joined,
    as rows ``[T, heads * head_dim]`` in 8 bits.  ``positions [T]`` (int32): a
    token's splits of ``split_keys`` keys are those that hold keys up to its
    position, and (``window`` > 0) of its last ``window`` keys.  A head that saw
    nothing is not a number."""
    here = _here()
    if not isinstance(partial_o, torch.Tensor) or partial_o.dim() != 3 or heads <= 0 or partial_o.shape[1] % heads or not partial_o.shape[2] or partial_o.shape[2] % 8 or window < 0 or split_keys <= 0:
        raise AlofaError("invalid_argument", "splits of heads of a multiple of 8 channels", f"partial_o={tuple(getattr(partial_o, 'shape', ()))} heads={heads} window={window} split_keys={split_keys}")
    splits, n, hd = partial_o.shape
    t = n // heads
    o_at, ml_at, p_at = _at(partial_o, "partial_o", _F32, (splits, n, hd), here), _at(partial_ml, "partial_ml", _F32, (splits, n, 2), here), _at(positions, "positions", _I32, (t,), here)
    rows = MxRows._empty(t, heads * hd, here, buf)
    rc = _lib.alofa_mx_merge(rows.codes_at, rows.scales_at, o_at, ml_at, p_at, t, heads, hd, splits, window, split_keys, _stream(here))
    ops.mx_launched(rc, 1 if t else 0, "merge_rows", lambda: f"tokens={t} heads={heads} head_dim={hd} splits={splits}")
    return rows


def _operands(x, w, what: str, gated: bool, here: int, buf) -> MxRows:
    if not isinstance(w, MxWeight) or w.gated != gated:
        raise AlofaError("invalid_argument", f"{what} takes a weight that was packed for it", f"weight={type(w).__name__} gated={getattr(w, 'gated', None)}")
    if not isinstance(x, MxRows):
        x = quantize_rows(x, buf)
    if x.width != w.k:
        raise AlofaError("invalid_argument", f"{what}: rows and weight differ in depth", f"rows={x.width} weight={w.k}")
    _on(x, "x", _on(w, "w", here))
    return x


_CALL = struct.Struct("9Q4i2f4i").pack  # a product's arguments (MxCall in kernels/mx_gemm.cu)
_plans: dict = {}
_SMS: dict = {}  # of a device


def _sms(here: int) -> int:
    if here not in _SMS:
        _SMS[here] = torch.cuda.get_device_properties(here).multi_processor_count
    return _SMS[here]


# As in kernels/mx_gemm.cu: slices that one accumulator sums (for prompts, of what is stored), and accumulators of a tile by its tokens.
RUN_SLICES, RUN_SLICES_STORED, MOST_RUNS = 16, 32, {16: 13, 32: 6, 64: 3, 96: 2, 128: 1}

# What orders the ways of a product.  The numbers were searched for so that the way with the smallest sum is the one with the shortest
# measured time at the shapes of 0.5 to 7 billion parameters and 1 to 1,024 tokens: it is 1.3 % off the shortest on the average.  They are weights of that order
# and no times (a slice takes a CTA 0.21 to 0.24 us with tiles of 16 and of 32 tokens alike), and at some sizes they miss: one token,
# 896 x 9,728 gated 4.6 to 4.9 us in three parts, 4.1 in one; 768 tokens, 8,960 x 1,536 20.7 instead of 17.1.
# For a slice of 128 numbers of a CTA of the kernel for a few tokens, by its tokens: alone on its SM, and where two share one.
_FEW_SLICE = {16: (0.354, 0.400), 32: (0.225, 0.241), 64: (0.326, 0.420), 96: (0.743, 0.866), 128: (0.743, 0.866)}


def _few_us(tokens: int, rows: int, slices: int, gated: bool, bn: int, parts: int, sms: int) -> float:
    ctas = -(-rows // TILE_ROWS) * -(-tokens // bn) * parts
    alone, shared = _FEW_SLICE[bn]
    room = 2 * sms if parts == 1 else int(0.946 * 2 * sms)  # clusters do not fill every SM
    whole, rest = divmod(ctas, room)
    rounds = whole * shared + (shared if rest > sms else alone if rest else 0.0)
    last = (0.055 * (whole + (rest > 0)) if gated else 0.01) * min(tokens, bn) / parts  # a tile's last step: its tokens, over its parts
    return 4.94 + 0.226 * parts + last + rounds * -(-slices // parts) + 3.69 * (whole - (rest == 0))


def _pair_us(tokens: int, rows: int, slices: int, gated: bool, sms: int) -> float:
    tiles, runs = -(-rows // 256) * -(-tokens // 256), -(-slices // (RUN_SLICES if gated else RUN_SLICES_STORED))
    return 5.4 + -(-tiles // (sms // 2)) * (0.8 + 0.499 * slices + 1.3 * (runs - 1))


def plan(tokens: int, rows: int, depth: int, gated: bool = False, here: Optional[int] = None) -> tuple:
    """(tokens a tile, parts of the depth) of a product on device ``here`` (the
    current one); 256 tokens: pairs of CTAs.

    The kernel for a few tokens has tiles of up to 32 of them in steps of as many,
    of 32, 64 or 96 (128 beyond) in larger ones; its depth goes in as many parts as make it
    shortest (us, depth x rows): 1 token, 18,944 x 3,584 in 8 parts 10.4, in 4
    12.8; 64 tokens, 896 x 9,728 gated in tiles of 32 8.1 and of 64 8.4.  Beyond 64
    tokens it is weighed against pairs, which take long to begin and then do a
    slice of 256 x 256 in the time the others take for a quarter of it: 256
    tokens, 3,584 x 4,608 11.4 in tiles of 64 and 16.7 on pairs; 192 tokens, 3,584
    x 37,888 gated 51.8 and 33.2; 1,024 tokens, 18,944 x 3,584 91.5 and 59.3,
    8,960 x 1,536 27.0 and 30.2."""
    sms = _sms(_here() if here is None else here)
    key = (tokens, rows, depth, gated, sms)
    found = _plans.get(key)
    if found is None:
        slices = padded(depth) // GROUP
        tiles = (16,) if tokens <= 16 else (32,) if tokens <= 32 else (32, 64) if tokens <= 64 else (32, 64, 96) if tokens <= 96 else (64, 128)
        # a part's slices go in as many runs as there are accumulators for: where more parts can make them so, no longer ones than RUN_SLICES in
        # front of a rounding to 8 bits, and of four times as many else (50 leave 2.7e-7; 512 tokens, 18,944 x 3,584 49.6 us, and 61.5 with 32 at most)
        run = RUN_SLICES if gated else 4 * RUN_SLICES
        ways = [(_few_us(tokens, rows, slices, gated, bn, parts, sms), bn, parts) for bn in tiles if tokens <= MOST_TILES * bn for parts in (1, 2, 3, 4, 6, 8)
                if parts <= slices and (parts == 8 or -(-slices // parts) <= run * MOST_RUNS[bn])]
        if tokens > 64:
            ways.append((_pair_us(tokens, rows, slices, gated, sms), 256, 1))
        if len(_plans) >= 4096:
            _plans.clear()
        found = _plans[key] = min(ways)[1:]
    return found


def _product(x: MxRows, w: MxWeight, out_at, scales_at, bias_at, add_at, features: int, gate, out_bf16, status, how, here: int, what: str) -> None:
    if not x.rows:
        return
    bn, parts = how or plan(x.rows, w.rows, w.k, w.gated, here)
    status_at = 0 if status is None else _at(status, "status", _I32, getattr(status, "shape", ()), here)
    call = _CALL(out_at, scales_at, x.codes_at, x.scales_at, w.at, w.maps_at, bias_at, add_at, status_at, x.rows, w.rows, w.k, features, gate[0], gate[1], bn, parts, _sms(here), out_bf16)
    rc = _lib.alofa_mx_gemm(call, _stream(here))
    ops.mx_launched(rc, 1, what, lambda: f"tokens={x.rows} rows={w.rows} depth={w.k} how={(bn, parts)}")


def linear(x, w: MxWeight, bias=None, add=None, out=None, dtype=None, buf=None, status=None, how: Optional[tuple] = None) -> torch.Tensor:
    """``out = x w^T (+ bias) (+ add)``.  ``x``: rows in 8 bits, or a tensor
    that is made such rows first; ``bias [N]``, ``add [T, N]`` float32
    (``add`` may be ``out``).  ``out`` (or ``dtype``): bfloat16 unless ``add``
    is given, else float32.  ``status`` (int32): raised where a kernel gave up.
    ``how``: another answer than :func:`plan`'s."""
    here = _here()
    x = _operands(x, w, "linear", False, here, buf)
    t, n = x.rows, w.n
    if out is None:
        dtype = dtype or (_BF16 if add is None else _F32)
        if dtype is not _BF16 and dtype is not _F32:
            raise AlofaError("unsupported", "a product is stored in bfloat16 or float32", f"dtype={dtype}")
        out = w.tiles.new_empty((t, n), dtype=dtype) if buf is None else buf((t, n), dtype)
        out_at, out_bf16 = out.data_ptr(), dtype is _BF16
    else:
        out_at, rows, columns, out_bf16 = _matrix(out, "out", here)
        if rows != t or columns != n or (dtype is not None and out.dtype is not dtype):
            _refuse(out, "out", f"{dtype or out.dtype} ({t}, {n})", here)
    bias_at = 0 if bias is None else _at(bias, "bias", _F32, (n,), here)
    add_at = 0 if add is None else _at(add, "add", _F32, (t, n), here)
    _product(x, w, out_at, 0, bias_at, add_at, 0, ops.SILU_GATE, out_bf16, status, how, here, "linear")
    return out


def gated_linear(x, w: MxWeight, gate=ops.SILU_GATE, buf=None, status=None, how: Optional[tuple] = None) -> MxRows:
    """``silu(x Wg^T) * (x Wu^T)`` as rows in 8 bits; ``gate`` = (alpha,
    limit), both over 0: the clamped form ``g = min(g, limit), u = clamp(u, -limit, limit):
    g sigmoid(alpha g) (u + 1)``."""
    here = _here()
    if gate is not ops.SILU_GATE and gate != ops.SILU_GATE and not (gate[0] > 0 and gate[1] > 0):
        raise AlofaError("invalid_argument", "a clamped gate's alpha and limit are over 0", f"gate={gate}")
    x = _operands(x, w, "gated_linear", True, here, buf)
    features = w.n // 2
    rows = MxRows._empty(x.rows, features, here, buf)
    _product(x, w, rows.codes_at, rows.scales_at, 0, 0, features, gate, False, status, how, here, "gated_linear")
    return rows
