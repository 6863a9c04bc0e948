"""8-bit products: e4m3 values with a power-of-two scale for each block of 128.

A block of values (1 x 128 along a row of activations, 128 x 128 of a weight) is held as q s: s the least
power of two, at least 2^-127, for which the block's largest finite magnitude is at most 448 s (448 is e4m3's largest
value), q = v / s rounded to e4m3; inf and NaN become NaN. Both scales of a product are applied inside the
matrix unit; sums are made in its float32 accumulators and rounded once. The unit cuts the terms of 8 neighbouring
depths off at 2^-13 of the largest of them before it adds them: about 2e-5 of a product's norm for
normally distributed operands, far below a bfloat16 output's rounding. Between an expert's two products the result is
rounded to e4m3, where this turns one activation in some thousand to its neighbour, up to 2^-3 away. Calls of up to 2^21
activations (rows times slots times expert width) add in float32 there, which larger ones would pay with up to twice
the first product's time; a larger batch called in such parts is added in float32 too.

``quantize_weight`` makes the weight that ``zmoe.functional.fp8_linear`` serves with;
``GLUMLP.quantize_fp8``, ``ExpertMLP.quantize_fp8`` and ``MoELayer.quantize_fp8`` make serving modules of
trained ones; ``fp8=True`` in ``scattermoe.parallel_experts`` trains with such products.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import library as zl
from . import ops

BLOCK = ops.FP8_BLOCK


def _values(q: torch.Tensor, scales: torch.Tensor, cols: int) -> torch.Tensor:
    """q [..., cols'] times 2^(scale - 127) of each block of columns (``scales`` [..., blocks] per row)."""
    v = q.to(torch.float32).unflatten(-1, (-1, BLOCK)) if q.numel() else q.new_zeros((*q.shape[:-1], 0, BLOCK),
                                                                                    dtype=torch.float32)
    e = scales[..., :q.shape[-1] // BLOCK].to(torch.int32)
    # 2^(e - 127) as two factors: 2^-127 is no normal float32
    half = lambda x: ((x + 127) << 23).view(torch.float32)  # noqa: E731
    e1 = (e - 127) // 2
    v = v * half(e1).unsqueeze(-1) * half(e - 127 - e1).unsqueeze(-1)
    return v.flatten(-2)[..., :cols]


def quantize_rows(x: torch.Tensor):
    """(q float8_e4m3fn [n, Kp], s uint8 [n, pitch]) of the rows of x [n, K], Kp = 128 ceil(K / 128)."""
    with torch.no_grad():
        return tuple(zl.fp8_quantize_rows(x, None, 1, None))


def dequantize_rows(q: torch.Tensor, s: torch.Tensor, K: int) -> torch.Tensor:
    """The float32 values [n, K] that quantised rows stand for."""
    return _values(q, s, K)


class Fp8Weight:
    """A weight [..., N, K] held in e4m3 with a scale for each 128 x 128 block (``quantize_weight``).

    ``q`` [..., N, Kp] and ``s`` [..., blocks of N, pitch] as the kernels read them; ``qt``, ``st``: the same
    values transposed, which gradients of a product's input need (None without). It records no gradient."""

    __slots__ = ("q", "s", "qt", "st", "K")

    def __init__(self, q: torch.Tensor, s: torch.Tensor, K: int, qt: Optional[torch.Tensor] = None,
                 st: Optional[torch.Tensor] = None):
        self.q, self.s, self.qt, self.st, self.K = q, s, qt, st, K

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.q.shape[:-1], self.K))

    @property
    def device(self) -> torch.device:
        return self.q.device

    def to(self, device) -> "Fp8Weight":
        move = lambda t: None if t is None else t.to(device)  # noqa: E731
        return Fp8Weight(move(self.q), move(self.s), self.K, move(self.qt), move(self.st))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values [..., N, K] it stands for (exact in float32 and, but for float32's denormals, bfloat16)."""
        rows = self.s.repeat_interleave(BLOCK, -2)[..., :self.q.shape[-2], :]
        return _values(self.q, rows, self.K).to(dtype)

    def __repr__(self):
        return f"Fp8Weight(shape={tuple(self.shape)}, transposed={self.qt is not None}, device={self.device})"


def quantize_weight(W: torch.Tensor, transposed: bool = False) -> Fp8Weight:
    """W [..., N, K] (bfloat16 or float32, on the device) as an ``Fp8Weight``."""
    with torch.no_grad():
        out = zl.fp8_quantize_weight(W.detach(), transposed)
    return Fp8Weight(out[0], out[1], W.shape[-1], *out[2:])
