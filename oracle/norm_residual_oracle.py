"""norm_residual and its gradient in float64 by its formulas, with magnitudes for error bounds.

``forward`` and ``backward`` return values and, for each, the sum of the magnitudes that it is added up from (every
subtraction taken as an addition): an evaluation in float32 is off by a small multiple of 2^-24 of that."""

import torch

F64 = torch.float64


def _f(t):
    return None if t is None else t.detach().to(F64)


def forward(r, y, w_post, w_next, gate, scale, eps):
    r, y, w1, w2, g = map(_f, (r, y, w_post, w_next, gate))
    g = 1.0 if g is None else g
    rho1 = None if w1 is None else torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
    u = y if w1 is None else y * rho1 * (1 + w1)
    h, H = scale * r + g * u, (scale * r).abs() + (g * u).abs()
    val, mag = {"r": h}, {"r": H}
    rho2 = None
    if w2 is not None:
        rho2 = torch.rsqrt(h.square().mean(-1, keepdim=True) + eps)
        val["x"], mag["x"] = h * rho2 * (1 + w2), H * rho2 * (1 + w2).abs()
    return val, mag, (u, h, H, rho1, rho2)


def backward(r, y, w_post, w_next, gate, scale, eps, dr, dx):
    """Grads of (dr, dx), either None, for r, y, w_post, w_next, the gate (summed over what it broadcast over), scale."""
    _, _, (u, h, H, rho1, rho2) = forward(r, y, w_post, w_next, gate, scale, eps)
    gate_shape = None if gate is None else gate.shape
    r, y, w1, w2, g, dr, dx = map(_f, (r, y, w_post, w_next, gate, dr, dx))
    g = torch.ones((), dtype=F64, device=y.device) if g is None else g
    d = y.shape[-1]
    t = torch.zeros_like(y) if dr is None else dr
    T = t.abs()
    val, mag = {}, {}
    if w2 is not None:
        a = torch.zeros_like(y) if dx is None else dx * (1 + w2)
        t = t + rho2 * a - h * rho2 ** 3 / d * (a * h).sum(-1, keepdim=True)
        T = T + rho2 * a.abs() + H * rho2 ** 3 / d * (a.abs() * H).sum(-1, keepdim=True)
        z = torch.zeros_like(y) if dx is None else dx
        val["w_next"], mag["w_next"] = (z * h * rho2).sum(0), (z.abs() * H * rho2).sum(0)
    val["r"], mag["r"] = scale * t, abs(scale) * T
    val["scale"], mag["scale"] = (t * r).sum(), (T * r.abs()).sum()
    if gate_shape is not None:
        tu, TU = t * u, T * u.abs()
        if len(gate_shape) == 1:
            tu, TU = tu.sum(0), TU.sum(0)
        elif gate_shape[-1] == 1 and d > 1:
            tu, TU = tu.sum(-1, keepdim=True), TU.sum(-1, keepdim=True)
        val["gate"], mag["gate"] = tu, TU
    du, DU = g * t, g.abs() * T
    if w1 is None:
        val["y"], mag["y"] = du, DU
    else:
        b, B = du * (1 + w1), DU * (1 + w1).abs()
        val["y"] = rho1 * b - y * rho1 ** 3 / d * (b * y).sum(-1, keepdim=True)
        mag["y"] = rho1 * B + y.abs() * rho1 ** 3 / d * (B * y.abs()).sum(-1, keepdim=True)
        val["w_post"], mag["w_post"] = (du * y * rho1).sum(0), (DU * y.abs() * rho1).sum(0)
    return val, mag
