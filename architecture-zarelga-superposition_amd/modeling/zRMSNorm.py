"""Zero-centred RMSNorm (reference modeling/zRMSNorm.py:4-20) on MI355X.

Same module name, parameter (``weight``, zeros: the gain is ``1 + weight``), ``eps``
default and arithmetic (fp32, result in the input dtype) as the reference. The
forward and backward are one HIP row pass each (``zmoe_rmsnorm_rows``). The
transformer block normalises right before the MoE layer
(modeling/transformer_block.py:41-42); passing this module to
``MoELayer.forward(..., norm=...)`` folds that normalisation and the layer's unpad
gather into the same pass.
"""

from typing import Optional

import torch
import torch.nn as nn

from zmoe import functional as _zf


class ZeroCenteredRMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.zeros(dim))

    def forward(self, x):
        return _zf.rmsnorm_rows(x, self.weight, self.eps)

    def extra_repr(self):
        return f"{tuple(self.weight.shape)}, eps={self.eps}"


class NormResidual(nn.Module):
    """The step from one sublayer of a block to the next, one HIP pass each way (``zmoe_norm_residual``):

        residual = residual_scale * residual + gate * norm(y)
        x = next_norm(residual)            # next_norm: the ZeroCenteredRMSNorm in front of the next sublayer

    ``forward(residual, y, next_norm=None)`` returns (residual, x), x None without ``next_norm``, whose weight stays its
    own (as the norm passed to ``MoELayer.forward``). ``post_norm`` False leaves the norm of y out (then next_norm
    is required), ``gate`` True adds a learned gain for each channel (ones at first), ``residual_scale`` a learned scalar
    starting there. A gate that is computed from the tokens is passed to ``forward``."""

    def __init__(self, dim: int, eps: float = 1e-6, post_norm: bool = True, gate: bool = False,
                 residual_scale: Optional[float] = None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.zeros(dim)) if post_norm else None
        self.gate = nn.Parameter(torch.ones(dim)) if gate else None
        self.residual_scale = None if residual_scale is None else nn.Parameter(torch.tensor([float(residual_scale)]))

    def forward(self, residual, y, next_norm=None, gate=None):
        if gate is not None and self.gate is not None:
            raise ValueError("NormResidual: a gate was passed to a module with one of its own")
        if next_norm is not None and next_norm.eps != self.eps:
            raise ValueError("NormResidual: the two norms' eps differ")
        return _zf.norm_residual(residual, y, self.weight, None if next_norm is None else next_norm.weight,
                                 self.gate if gate is None else gate, self.residual_scale, self.eps)

    def extra_repr(self):
        return (f"eps={self.eps}, post_norm={self.weight is not None}, gate={self.gate is not None}, "
                f"residual_scale={self.residual_scale is not None}")
