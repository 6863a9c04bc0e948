"""Shared expert (reference modeling/expert_layer.py:5-24): dense SwiGLU.

Its three bias-free projections are dense GEMMs (hipBLASLt through torch; the up
and gate projections as one GEMM), the SwiGLU is a fused HIP pass and the weight
grads are split-K HIP GEMMs (zmoe.functional.swiglu_mlp). State-dict keys
gate_proj / up_proj / down_proj are unchanged.
"""

import torch
import torch.nn as nn

from scattermoe.mlp import Fp8Module, glu_weights_fp8
from zmoe import functional as _zf
from zmoe import library as _zl


class ExpertMLP(nn.Module):
    def __init__(self, config, intermediate_size=None):
        super().__init__()
        self.config = config
        self.hidden_size = config.hidden_size
        self.intermediate_size = intermediate_size or config.intermediate_size
        self.initializer_range = config.initializer_range
        self.gate_proj = nn.Linear(self.hidden_size, self.intermediate_size, bias=False)
        self.up_proj = nn.Linear(self.hidden_size, self.intermediate_size, bias=False)
        self.down_proj = nn.Linear(self.intermediate_size, self.hidden_size, bias=False)
        self.act_fn = nn.SiLU()
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.normal_(self.gate_proj.weight, mean=0.0, std=self.initializer_range)
        nn.init.normal_(self.up_proj.weight, mean=0.0, std=self.initializer_range)
        nn.init.normal_(self.down_proj.weight, mean=0.0, std=self.initializer_range)

    def forward(self, x):
        # down_proj(act_fn(gate_proj(x)) * up_proj(x)), expert_layer.py:23-24
        return _zf.swiglu_mlp(x, self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight)

    def quantize_fp8(self) -> "Fp8ExpertMLP":
        """A serving module with the present weights in e4m3."""
        return Fp8ExpertMLP(self.gate_proj.weight, self.up_proj.weight, self.down_proj.weight)


class Fp8ExpertMLP(Fp8Module):
    """``ExpertMLP`` for serving, its weights in e4m3 with a power-of-two scale for each 128 x 128 block; the SwiGLU and
    its quantisation are the first product's epilogue. No gradients."""

    def __init__(self, W_gate: torch.Tensor, W_up: torch.Tensor, W_down: torch.Tensor):
        super().__init__()
        self.intermediate_size, self.hidden_size = W_up.shape
        W1 = torch.cat([W_up.detach(), W_gate.detach()]).unsqueeze(0)
        w1q, w1s, w2q, w2s = glu_weights_fp8(W1, W_down.unsqueeze(0))
        self._hold(w1_values=w1q, w1_scales=w1s, w2_values=w2q[0], w2_scales=w2s[0])

    def forward(self, x):
        x = self._serve(x)
        if x.shape[-1] != self.hidden_size:
            raise ValueError(f"Fp8ExpertMLP: rows of {self.hidden_size}, got {x.shape[-1]}")
        with torch.no_grad():
            y = _zl.fp8_glu_mlp(x.reshape(-1, self.hidden_size), *self._weights("w1", "w2"))
        return y.view(x.shape)
