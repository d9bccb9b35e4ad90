"""Matrix products of the parts with weights in 4 bits and rows in 8
(``weight_format="mxfp4"``; the formats and kernels: :mod:`alofa_b200.mx`).

A :class:`MxLinear` is called as a :class:`~alofa_b200.parts.linear.Linear` is.
The weight is packed when the part loads.  Rows come in 8 bits from the norm in
front (:class:`~alofa_b200.mx.MxRows`); any other rows are made so first.  A
product into the residual stream leaves its sums to a consumer that asks
(``defer``), as the bfloat16 products do."""
from __future__ import annotations

import torch

from .. import mx
from ..errors import AlofaError
from .linear import GATED, RESIDUAL, STORE, Linear, Partial

MXFP4 = "mxfp4"
WEIGHT_FORMATS = (None, MXFP4)


class MxLinear:
    """``epi`` STORE: out = x W^T + b.  RESIDUAL: out (fp32) += x W^T + b.
    GATED: W = [gate; up]; :meth:`gated_rows` (silu) instead of a call."""

    def __init__(self, weight, bias, epi: int = STORE):
        self.weight = weight if isinstance(weight, mx.MxWeight) else mx.pack_weight(weight.contiguous(), gated=epi == GATED)
        self.bias, self.epi = bias, epi
        if bias is not None and epi == GATED:
            raise AlofaError("unsupported", "a gated product with weights in 4 bits takes no bias")

    takes_status = True  # a call may name the step's status word, which a kernel raises that gave up on a wait

    def can_accumulate(self, tokens: int) -> bool:
        return False  # its sums are added by the norm that reads the stream next

    def _rows(self, x, buf):
        if isinstance(x, mx.MxRows):
            return x
        if not isinstance(x, torch.Tensor):  # decode attention whose splits are not joined yet
            return x.mx_rows()
        return mx.quantize_rows(x, buf)

    def __call__(self, out, x, defer: bool = False, buf=None, status=None):
        x = self._rows(x, buf)
        if defer and self.epi == RESIDUAL:
            y = mx.linear(x, self.weight, dtype=torch.float32, buf=buf, status=status)
            return Partial(y.view(1, *y.shape), 1, self.bias)  # the norm that reads the stream next adds it
        mx.linear(x, self.weight, bias=self.bias, add=out if self.epi == RESIDUAL else None, out=out, buf=buf, status=status)
        return None

    def gated_rows(self, x, buf=None, status=None) -> mx.MxRows:
        return mx.gated_linear(self._rows(x, buf), self.weight, buf=buf, status=status)


def make_linear(rt, weight, bias, epi: int = STORE):
    """A product of a part's: in the model's compute dtype, or with its weight in 4 bits."""
    if rt.weight_format == MXFP4:
        return MxLinear(weight, bias, epi)
    return Linear(weight, bias, epi)
