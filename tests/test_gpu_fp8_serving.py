"""What the e4m3 serving modules refuse and promise beyond test_gpu_fp8_layers."""

import pytest
import torch

from helpers import gen, random_topk
from test_gpu_fp8_layers import activations

BF = torch.bfloat16


def test_base_module_refuses_any_gradient():
    from scattermoe.mlp import Fp8Module

    m, x, p = Fp8Module(), torch.zeros(2, 4), torch.zeros(2, 4, requires_grad=True)
    assert m._serve(x, None, x) is x
    for args in ((p,), (x, p), (x, None, p)):
        with pytest.raises(RuntimeError):
            m._serve(*args)
        with torch.no_grad():
            m._serve(*args)


@pytest.mark.gpu
def test_experts_refuse_lost_gradients(hip_device):
    """Routing weights or a residual that would lose their gradients silently."""
    from scattermoe.mlp import GLUMLP

    T, d, f, E, k = 6, 64, 32, 4, 2
    s = GLUMLP(d, f, E, k).to(hip_device).to(BF).quantize_fp8()
    x, idx = activations(T, d, BF, 1, hip_device), random_topk(T, E, k, 1).to(hip_device)
    p, res = torch.rand(T, k, generator=gen(2)).to(hip_device), activations(T, d, BF, 3, hip_device)
    out = s(x, p, idx, residual=res)
    pg, rg = p.clone().requires_grad_(True), res.clone().requires_grad_(True)
    for args, kw in (((x, pg, idx), {}), ((x, p, idx), dict(residual=rg)), ((x, pg, idx), dict(residual=rg))):
        with pytest.raises(RuntimeError):
            s(*args, **kw)
    with torch.no_grad():
        assert torch.equal(s(x, pg, idx, residual=rg), out)


@pytest.mark.gpu
def test_layer_refuses_lost_gradients(hip_device):
    """A trainable norm in front of the layer, or a gate made trainable again."""
    from modeling.model_config import ModelConfig
    from modeling.moe_layer import MoELayer
    from modeling.zRMSNorm import ZeroCenteredRMSNorm

    d = 128
    layer = MoELayer(ModelConfig(hidden_size=d, intermediate_size=64, n_experts=9, n_shared_experts=1, n_experts_per_token=2))
    served = layer.to(hip_device).bfloat16().quantize_fp8()
    served.gate.expert_biases = served.gate.expert_biases.float()
    pre = ZeroCenteredRMSNorm(d).to(hip_device)
    h = torch.randn(2, 5, d, generator=gen(1)).to(BF).to(hip_device)
    with torch.no_grad():
        ref = served(h, norm=pre)
    with pytest.raises(RuntimeError):
        served(h, norm=pre)
    pre.requires_grad_(False)
    assert torch.equal(served(h, norm=pre)[0], ref[0])
    served.gate.requires_grad_(True)
    with pytest.raises(RuntimeError):
        served(h)
