"""The block-scaled e4m3 format and the products on it, in float64 (torch, CPU or device).

A block of values is held as q s, s = 2^c with c the least whole number >= -127 for which the block's
largest finite magnitude is at most 448 s, q = e4m3(v / s), nearest even; inf and NaN become NaN.
"""

import torch

F64 = torch.float64
BLOCK = 128


def two(c: torch.Tensor) -> torch.Tensor:
    """2^c for whole c in [-1022, 1023], from the bits."""
    return ((c.to(torch.int64) + 1023) << 52).view(F64)


def log2_floor(a: torch.Tensor) -> torch.Tensor:
    """floor(log2 a) for normal float64 a > 0, from the bits."""
    return (a.view(torch.int64) >> 52) - 1023


def scale_exponent(a: torch.Tensor) -> torch.Tensor:
    """c of blocks of largest finite magnitude a >= 0."""
    c = log2_floor(a.clamp(min=2.0 ** -160)) - 8
    return torch.where(a > 448 * two(c), c + 1, c).clamp(min=-127)


def e4m3(v: torch.Tensor) -> torch.Tensor:
    """v (|v| <= 448, or not finite) rounded to e4m3."""
    ok = torch.isfinite(v)
    w = torch.where(ok, v, torch.zeros_like(v))
    step = two(log2_floor(w.abs().clamp(min=2.0 ** -60)).clamp(min=-6) - 3)
    return torch.where(ok, torch.round(w / step) * step, torch.full_like(v, float("nan")))


def _amax(v: torch.Tensor, dims) -> torch.Tensor:
    return torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(dims, keepdim=True)


def quantize_rows(x: torch.Tensor):
    """(values that x [n, K] stands for, scale exponents [n, blocks])."""
    x = x.to(F64)
    n, K = x.shape
    v = torch.nn.functional.pad(x, (0, -K % BLOCK)).view(n, -(-K // BLOCK), BLOCK)
    c = scale_exponent(_amax(v, 2))
    return (e4m3(v * two(-c)) * two(c)).view(n, v.shape[1] * BLOCK)[:, :K].contiguous(), c.squeeze(-1)


def quantize_weight(W: torch.Tensor):
    """(values that W [..., N, K] stands for, scale exponents [..., N blocks, K blocks])."""
    N, K = W.shape[-2:]
    w = torch.nn.functional.pad(W.to(F64).reshape(-1, N, K), (0, -K % BLOCK, 0, -N % BLOCK))
    v = w.view(w.shape[0], w.shape[1] // BLOCK, BLOCK, w.shape[2] // BLOCK, BLOCK)
    c = scale_exponent(_amax(v, (2, 4)))
    out = (e4m3(v * two(-c)) * two(c)).view(w.shape)[:, :N, :K]
    return out.reshape(W.shape).contiguous(), c[:, :, 0, :, 0].reshape(*W.shape[:-2], c.shape[1], c.shape[3])


def product(a, w):
    """(a w^T, the sum of |terms|, the sum over groups of 8 consecutive depths of the largest |term|)."""
    a, w = a.to(F64), w.to(F64)
    g = torch.zeros(a.shape[0], w.shape[0], dtype=F64, device=a.device)
    aa, wa = a.abs(), w.abs()
    for k in range(0, a.shape[1], 8):
        top = aa[:, None, k] * wa[None, :, k]
        for j in range(k + 1, min(k + 8, a.shape[1])):
            top = torch.maximum(top, aa[:, None, j] * wa[None, :, j])
        g += top
    return a @ w.T, aa @ wa.T, g


def grouped_product(x, W, sorted_scattered_idxs, offsets, k, x_grouped, y_grouped):
    """``product`` of sorted rows and W_e; rows of no expert are NaN."""
    R = sorted_scattered_idxs.numel()
    out = [torch.full((R, W.shape[1]), float("nan"), dtype=F64, device=x.device) for _ in range(3)]
    beg = 0
    for e, end in enumerate(offsets.tolist()):
        rows = sorted_scattered_idxs[beg:end]
        a = x[beg:end] if x_grouped else x[rows // k]
        at = torch.arange(beg, end, device=x.device) if y_grouped else rows
        if end > beg:
            for o, v in zip(out, product(a, W[e])):
                o[at] = v
        beg = end
    return out
