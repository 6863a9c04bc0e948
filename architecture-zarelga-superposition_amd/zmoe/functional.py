"""Autograd functions for the dense layers around the routed experts.

The reference computes the gate projection (modeling/moe_gate.py:26) and the shared
expert (modeling/expert_layer.py:23-24) as plain nn.Linear / F.linear under torch
autograd. Here the forward GEMMs and input grads stay library GEMMs (hipBLASLt
through torch), while the weight grads — small outputs reduced over all T tokens,
which one library launch spreads over only a few dozen tiles — run as the split-K
``zmoe_dense_wgrad`` (fp32 partials, fixed-order sum, one rounding). The shared
expert's SwiGLU is one fused HIP pass each way (``zmoe_swiglu`` /
``zmoe_swiglu_backward``) and its up and gate projections run as one GEMM.

bf16 CUDA tensors with 16-byte rows take these paths; other dtypes and widths use plain
torch ops, as the reference does.
"""

from __future__ import annotations

from typing import Optional, Union

import torch
import torch.nn.functional as F

from . import library as zl
from . import ops as _z
from .fp8 import Fp8Weight


def _fused(x, *ws) -> bool:
    """bf16 CUDA operands whose widths are whole 16-byte chunks (8 elements) take the HIP path:
    x's last dim and both dims of each [out, in] weight."""
    return (all(t.is_cuda and t.dtype == torch.bfloat16 for t in (x, *ws)) and x.shape[-1] % 8 == 0
            and all(w.shape[0] % 8 == 0 and w.shape[1] % 8 == 0 for w in ws))


class _Linear(torch.autograd.Function):
    """y = x W^T for x [M, K], W [N, K]."""

    @staticmethod
    def forward(ctx, x2, W):
        ctx.save_for_backward(x2, W)
        return F.linear(x2, W)

    @staticmethod
    def backward(ctx, dy):
        x2, W = ctx.saved_tensors
        dy = dy.contiguous()
        dx = dy @ W if ctx.needs_input_grad[0] else None
        dW = zl.dense_wgrad(dy, x2) if ctx.needs_input_grad[1] else None
        return dx, dW


def linear(x: torch.Tensor, W: torch.Tensor) -> torch.Tensor:
    """F.linear(x, W) without bias; the weight grad goes through the split-K kernel."""
    if not _fused(x, W):
        return F.linear(x, W)
    lead = x.shape[:-1]
    y = _Linear.apply(x.reshape(-1, x.shape[-1]), W)
    return y.view(*lead, W.shape[0])


class _SwiGLUMLP(torch.autograd.Function):
    """down(silu(gate(x)) * up(x)) (expert_layer.py:23-24) for x [M, d]."""

    @staticmethod
    def forward(ctx, x2, W_gate, W_up, W_down):
        f = W_up.shape[0]
        W_cat = torch.cat([W_up, W_gate], dim=0)     # [2f, d]: H = [up | gate], the GLU layout
        H = F.linear(x2, W_cat)
        A = zl.swiglu(H)                              # silu(gate) * up, one rounding
        y = F.linear(A, W_down)
        ctx.save_for_backward(x2, W_cat, W_down, H, A)
        ctx.f = f
        return y

    @staticmethod
    def backward(ctx, dy):
        x2, W_cat, W_down, H, A = ctx.saved_tensors
        f = ctx.f
        dy = dy.contiguous()
        dA = dy @ W_down                              # [M, f]
        dW_down = zl.dense_wgrad(dy, A)               # [d, f]
        dH = zl.swiglu_backward(dA, H)                # [M, 2f] = [d up | d gate]
        dx = dH @ W_cat
        dW_cat = zl.dense_wgrad(dH, x2)               # [2f, d]
        return dx, dW_cat[f:], dW_cat[:f], dW_down


def swiglu_mlp(x: torch.Tensor, W_gate: torch.Tensor, W_up: torch.Tensor, W_down: torch.Tensor) -> torch.Tensor:
    if not _fused(x, W_gate, W_up, W_down):
        return F.linear(F.silu(F.linear(x, W_gate)) * F.linear(x, W_up), W_down)
    lead = x.shape[:-1]
    y = _SwiGLUMLP.apply(x.reshape(-1, x.shape[-1]), W_gate, W_up, W_down)
    return y.view(*lead, W_down.shape[0])


class _RMSNormRows(torch.autograd.Function):
    """x = ZeroCenteredRMSNorm(hidden)[rows] (zRMSNorm.py:10-17, then moe_layer.py:39-42)."""

    @staticmethod
    def forward(ctx, hidden2, weight, eps: float, rows):
        y, rstd = zl.rmsnorm_rows(hidden2, weight, eps, rows)
        ctx.save_for_backward(hidden2, weight, rstd, rows if rows is not None else torch.empty(0))
        ctx.has_rows = rows is not None
        return y

    @staticmethod
    def backward(ctx, dy):
        hidden2, weight, rstd, rows = ctx.saved_tensors
        dx, dw = zl.rmsnorm_rows_backward(dy.contiguous(), hidden2, rows if ctx.has_rows else None, rstd, weight)
        return dx, dw, None, None


def rmsnorm_rows(hidden: torch.Tensor, weight: torch.Tensor, eps: float,
                 rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """ZeroCenteredRMSNorm of ``hidden`` [..., d], gathered at flat rows ``rows`` (None: all
    rows, keeping hidden's shape; else [len(rows), d]). One HIP pass each way."""
    d = hidden.shape[-1]
    flat = hidden.reshape(-1, d)
    y = _RMSNormRows.apply(flat, weight, float(eps), rows)
    return y.view(hidden.shape) if rows is None else y


def _compute_dtype(x: torch.Tensor) -> torch.dtype:
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else x.dtype


def _needs_graph(*ts: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def rows_on_16(t: torch.Tensor) -> torch.Tensor:
    """Rows [n, c] as the weight-grad kernels take them: unit column stride, no two rows overlapping and, where c is
    a whole number of 16-byte chunks, every row on 16 bytes (other widths go through padded copies); else a copy.
    (A tracer knows no storage offsets: there the rows are only made contiguous.)"""
    if torch.compiler.is_compiling():
        return t.contiguous()
    size = t.element_size()
    ok = t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1])
    if ok and (t.shape[1] * size) % 16 == 0:
        ok = (t.storage_offset() * size) % 16 == 0 and (t.stride(0) * size) % 16 == 0
    return t if ok else t.clone(memory_format=torch.contiguous_format)


class _Fp8Linear(torch.autograd.Function):
    """Q(x) Q(W)^T for x [M, K], W [N, K]; the quantisers pass gradients through: dx = Q(dy) Q(W) (dy's
    blocks run along N), dW = dy^T x from the unquantised operands."""

    @staticmethod
    def forward(ctx, x, W, dx: bool):
        q = zl.fp8_quantize_weight(W, dx)
        ctx.save_for_backward(x, *q[2:])
        ctx.w_dtype, ctx.N = W.dtype, W.shape[0]
        return zl.fp8_linear(x, q[0], q[1])

    @staticmethod
    def backward(ctx, dy):
        x, *qt = ctx.saved_tensors
        dx = dW = None
        if ctx.needs_input_grad[0]:
            dx = zl.fp8_linear(dy, *qt)
        if ctx.needs_input_grad[1]:
            f32 = ctx.w_dtype == torch.float32 and x.dtype != torch.float32  # fp32 master weights
            dW = zl.dense_wgrad(rows_on_16(dy), rows_on_16(x), f32).to(ctx.w_dtype)
        return dx, dW, None


class _Fp8LinearServed(torch.autograd.Function):
    """The same with a weight that was quantised before and takes no gradient."""

    @staticmethod
    def forward(ctx, x, q, s, qt, st):
        ctx.save_for_backward(qt, st)
        return zl.fp8_linear(x, q, s)

    @staticmethod
    def backward(ctx, dy):
        return zl.fp8_linear(dy, *ctx.saved_tensors), None, None, None, None


def fp8_linear(x: torch.Tensor, W: Union[torch.Tensor, Fp8Weight]) -> torch.Tensor:
    """F.linear(x, W) in e4m3 with a power-of-two scale for each block of 128 (``zmoe.fp8``), x [..., K].

    ``W``: a bfloat16 or float32 weight [N, K], quantised in the call, with gradients (of x by a product of the
    quantised output grad, of W from the unquantised operands; float32 weights get float32 grads); or an
    ``Fp8Weight``, quantised once (``fp8.quantize_weight``), which has a gradient for x only where it was made
    with ``transposed=True``. The result has x's dtype (under autocast, autocast's)."""
    x = x.to(_compute_dtype(x))
    served = isinstance(W, Fp8Weight)
    if len(W.shape) != 2 or x.dim() < 1 or x.shape[-1] != W.shape[1]:
        raise ValueError(f"fp8_linear: x [..., K] and W [N, K], got {tuple(x.shape)} and {tuple(W.shape)}")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if served:
        if not _needs_graph(x):
            with torch.no_grad():
                y = zl.fp8_linear(x2, W.q, W.s)
        elif W.qt is None:
            raise RuntimeError("fp8_linear: the gradient of x needs a weight quantised with transposed=True")
        else:
            y = _Fp8LinearServed.apply(x2, W.q, W.s, W.qt, W.st)
    else:
        y = _Fp8Linear.apply(x2, W, _needs_graph(x))
    return y if x.dim() == 2 else y.view(*x.shape[:-1], W.shape[0])


class _NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, r, y, w_post, w_next, gate, kind: int, scale, scale_value: float, eps: float):
        r_out, x, rho1, rho2 = zl.norm_residual(r, y, w_post, w_next, gate, kind, scale, scale_value, eps)
        ctx.save_for_backward(r, y, w_post, w_next, gate, scale, rho1 if w_post is not None else None,
                              rho2 if w_next is not None else None)
        ctx.kind, ctx.scale_value = kind, scale_value
        ctx.set_materialize_grads(False)
        return r_out, x if w_next is not None else None

    @staticmethod
    def backward(ctx, dr_out, dx):
        if dr_out is None and dx is None:
            return (None,) * 9
        r, y, w_post, w_next, gate, scale, rho1, rho2 = ctx.saved_tensors
        cont = lambda g: None if g is None else g.contiguous()  # noqa: E731
        dr, dy, dw1, dw2, dg, ds = zl.norm_residual_backward(cont(dr_out), cont(dx), r, y, w_post, w_next, gate,
                                                             ctx.kind, scale, ctx.scale_value, rho1, rho2)
        part = lambda t, g: None if t is None else g  # noqa: E731
        return dr, dy, part(w_post, dw1), part(w_next, dw2), part(gate, dg), None, part(scale, ds), None, None


def norm_residual(residual: torch.Tensor, y: torch.Tensor, weight: Optional[torch.Tensor] = None,
                  next_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                  residual_scale: Union[None, float, torch.Tensor] = None, eps: float = 1e-6):
    """The step from one sublayer to the next in one pass, for a residual stream and a sublayer's output y [..., d]:

      r = residual_scale * residual + gate * norm(y; weight),   x = norm(r; next_weight)

    with zero-centred RMSNorms (gain 1 + weight), either of which may be left out (not both). Returns (r, x), x
    None without ``next_weight``; r in the residual's dtype, x in y's (bfloat16 or float32 each), both rounded once from
    float32. ``gate``: [d] (a gain for each channel), [..., 1] (for each token), y's shape, or anything that
    broadcasts to it. ``residual_scale``: a number, or a tensor of one element, which gets a gradient."""
    if residual.shape != y.shape or y.dim() < 1:
        raise ValueError(f"norm_residual: residual and y must have one shape, got {tuple(residual.shape)} and "
                         f"{tuple(y.shape)}")
    if weight is None and next_weight is None:
        raise ValueError("norm_residual: neither weight nor next_weight given")
    d = y.shape[-1]
    if weight is not None and next_weight is not None and weight.dtype != next_weight.dtype:
        weight, next_weight = weight.float(), next_weight.float()
    kind = _z.GATE_NONE
    if gate is not None:
        if gate.shape == (d,):
            kind = _z.GATE_CHANNEL
        elif gate.shape == (*y.shape[:-1], 1) and d > 1:
            kind, gate = _z.GATE_ROW, gate.reshape(-1)
        else:
            if gate.shape != y.shape and _needs_graph(gate):
                gate = gate.float()  # its grad is rounded once, after the sum over what it broadcasts over
            kind, gate = _z.GATE_FULL, gate.expand(y.shape).reshape(-1, d)
    scale, value = None, 1.0
    if isinstance(residual_scale, torch.Tensor):
        if residual_scale.numel() != 1:
            raise ValueError("norm_residual: residual_scale is one number")
        scale = residual_scale.float()
    elif residual_scale is not None:
        value = float(residual_scale)
    if y.dim() == 2:
        return _NormResidual.apply(residual, y, weight, next_weight, gate, kind, scale, value, float(eps))
    r, x = _NormResidual.apply(residual.reshape(-1, d), y.reshape(-1, d), weight, next_weight, gate, kind, scale, value,
                               float(eps))
    return r.view(residual.shape), None if x is None else x.view(y.shape)
