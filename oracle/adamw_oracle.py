"""An AdamW step in float64 by its formula, and 8-bit moments by the borders between their codes, in whole numbers."""

import math
from fractions import Fraction

import torch

F64 = torch.float64
BLOCK = 256


def code(x: float, A: float, power: int, top: int) -> int:
    """The nearest code of |x| in the root's domain, half-way ones up: the number of borders ((q - 1/2) / top)^power A
    that |x| has reached, by exact fractions."""
    if A == 0.0:
        return 0
    share = Fraction(abs(x)) / Fraction(A) * (2 * top) ** power
    q = min(top, max(0, round(float(share) ** (1 / power) / 2)))
    while q < top and share >= (2 * q + 1) ** power:
        q += 1
    while q > 0 and share < (2 * q - 1) ** power:
        q -= 1
    return 1 if q == 0 and power == 4 and x > 0 else q


def through_codes(x, second: bool):
    """(codes, scales, the float32 values that they stand for) of a float32 tensor's elements in their order."""
    power, top = (4, 255) if second else (2, 127)
    flat = x.detach().float().cpu().reshape(-1)
    codes, scales, values = [], [], []
    for a in range(0, flat.numel(), BLOCK):
        block = flat[a:a + BLOCK].tolist()
        A = max((abs(v) for v in block), default=0.0)
        scales.append(A)
        for v in block:
            q = code(v, A, power, top)
            codes.append(-q if v < 0 else q)
            values.append(math.copysign(q ** power * (A / top ** power), v))
    shape = x.shape
    return (torch.tensor(codes, dtype=torch.int64).view(shape), torch.tensor(scales, dtype=torch.float32),
            torch.tensor(values, dtype=F64).float().view(shape))


def norm_and_factor(grads, max_norm):
    norm = math.sqrt(sum(float(g.detach().to(F64).square().sum()) for g in grads))
    return norm, min(1.0, max_norm / (norm + 1e-6))


def step(p, g, m, v, t, lr, betas, eps, wd, clip=1.0):
    """(p', m', v') in float64 after step number t, and the magnitude of the change that p' is made of."""
    p, g, m, v = (x.detach().to(F64) for x in (p, g, m, v))
    b1, b2 = betas
    g = g * clip
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    change = lr / (1 - b1 ** t) * m / (torch.sqrt(v) / math.sqrt(1 - b2 ** t) + eps)
    return p - lr * wd * p - change, m, v, change.abs()
