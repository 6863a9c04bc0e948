"""Grads through sigmoids near 1, whose slope p (1 - p) is far below a rounding of p: routing's and the losses' backwards against
float64 (oracle.router_oracle), with the bounds of tests/test_gpu_route.py and tests/test_gpu_router_losses.py, relative to
the slope itself."""

import math

import pytest
import torch

from helpers import gen
from oracle import router_oracle as O
from test_gpu_route import check as check_route
from test_gpu_router_losses import check as check_losses

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def saturated(T, E, dt, dev, seed=0):
    """Logits from -40 to 40, with rows of 10 to 40 alone, at the borders of the kernels' forms and past every f32 exponent."""
    g = gen(seed + 11 * T + E)
    z = torch.rand(T, E, generator=g) * 80 - 40
    z[::3] = torch.rand(z[::3].shape, generator=g) * 30 + 10
    edge = [0.0, -0.0, 17.4, 87.0, 89.0, 104.0, 1e30, -87.0, -89.0, -1e30, 1e-30, -1e-30]
    z[1 % T] = torch.tensor(edge).repeat(-(-E // len(edge)))[:E]
    return z.to(DT[dt]).to(dev)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("T,E,k", [(1, 2, 2), (7, 8, 3), (33, 64, 8), (20, 72, 5), (130, 128, 8), (40, 160, 6), (65, 256, 8),
                                   (9, 300, 7), (12, 512, 33), (11, 1024, 64)])
def test_route(T, E, k, dt, hip_device):
    z = saturated(T, E, dt, hip_device)
    bias = (torch.randn(E, generator=gen(E)) * 0.05).to(hip_device)
    for kw in (dict(bias=bias), dict(renormalize=False, scale=2.5)):
        idx, _, grad = check_route(z, k, score="sigmoid", **kw)
        if not kw.get("renormalize", True):  # logits of 20 to 40 that are taken have a grad
            taken = z.float().gather(1, idx)
            some = (taken > 20) & (taken < 40)
            assert (grad.float().gather(1, idx)[some] != 0).all() and (T < 20 or some.any())


def test_route_in_fewer_tokens_than_lanes(hip_device):
    """One expert in a renormalised row: the weight does not move, whatever its slope."""
    check_route(saturated(50, 40, "f32", hip_device), 1, score="sigmoid", scale=3.0)


def test_probabilities_alone(hip_device):
    """zmoe_route_backward without logits takes the slope of the probabilities as they are given (a gate that rounds them)."""
    from zmoe import ops

    z = saturated(30, 64, "f32", hip_device).clamp(-10, 10)
    idx, _, p = ops.route(z, None, 4, 0, 1, 1, 1, False, 1.0)
    p = p.bfloat16().float()
    dw = torch.randn(30, 4, generator=gen(3)).to(hip_device)
    got = ops.route_backward(dw, p, idx, 64, None, 0, False, 1.0, torch.float32)
    want = torch.zeros(30, 64, device=hip_device).scatter(1, idx, dw * p * (1 - p))
    assert torch.equal(got, want)


def test_strided_out_and_add(hip_device):
    """The losses' grad added and rows written into a wider buffer, as the whole layer's backward does."""
    from zmoe import ops

    z = saturated(50, 64, "bf16", hip_device)
    idx, _, p = ops.route(z, None, 6, 0, 1, 1, 1, True, 1.0)
    dw = torch.randn(50, 6, generator=gen(5)).to(hip_device)
    add = (torch.randn(50, 64, generator=gen(6)) * 1e-9).bfloat16().to(hip_device)
    wide = torch.zeros(50, 200, dtype=torch.bfloat16, device=hip_device)
    out = ops.route_backward(dw, p, idx, 64, z, 0, True, 1.0, torch.bfloat16, add, out=wide[:, 96:160])
    val, mag = O.weights_backward(z, idx, dw, "sigmoid", True, 1.0)
    val, mag = val + add.double(), mag + add.double().abs()
    bound = 2.0 ** -8 * val.abs() + (2 * 6 + 14) * 2.0 ** -24 * mag + 1e-38
    assert ((out.double() - val).abs() <= bound).all()
    assert not wide[:, :96].any() and not wide[:, 160:].any()


def test_layer_of_saturated_experts(hip_device):
    """A layer with a sigmoid form whose router saturates: the gate's grad is the composition's, and is not lost."""
    from test_gpu_router_training import D, grads_of, layer_of, tokens

    layer = layer_of(dict(router_renormalize=False, router_bias=False), hip_device)
    x = tokens(hip_device).abs()
    with torch.no_grad():
        layer.gate.weight.copy_(torch.full_like(layer.gate.weight, 24.0 / (D * 0.8)))  # logits of some 24 everywhere
    fused = grads_of(layer, x, tokens(hip_device, seed=9), False)[3]["gate.weight"].double()
    layer.fused_layer = False
    plain = grads_of(layer, x, tokens(hip_device, seed=9), False)[3]["gate.weight"].double()
    assert float((fused - plain).norm()) <= 2.0 ** -6 * float(plain.norm()) and float(plain.norm()) > 0


def test_default_form_keeps_its_probabilities(hip_device):
    """The reference's form stores p in bf16 and takes its slope from it, with the router's losses and without."""
    from test_gpu_router_training import grads_of, layer_of, tokens

    layer = layer_of({}, hip_device)
    x, dout = tokens(hip_device), tokens(hip_device, seed=9)
    without = grads_of(layer, x, dout, False)[3]
    for p in layer.parameters():
        p.grad = None
    xg = x.clone().requires_grad_(True)
    out, idx, (balance, z) = layer(xg, router_losses=True)
    torch.autograd.backward([out, balance, z], [dout, torch.zeros_like(balance), torch.zeros_like(z)])
    assert torch.equal(layer.gate.weight.grad, without["gate.weight"]) and torch.equal(xg.grad, without["x"])


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("T,E,k", [(1, 2, 2), (7, 8, 3), (33, 64, 8), (20, 72, 5), (130, 128, 8), (40, 160, 6), (65, 256, 8),
                                   (9, 300, 7), (33, 1024, 16)])
def test_losses(T, E, k, dt, hip_device):
    """Both losses, and the balance alone: the z loss would cover what the balance loses."""
    z = saturated(T, E, dt, hip_device)
    z[1 % T] = z[1 % T].clamp(-80, 80)  # (far logits apart: a z loss of 1e60)
    idx = torch.topk(z.float(), k).indices
    cu = torch.tensor([0, T // 3, T], device=hip_device)
    for gb, gz in ((0.3, 0.05), (0.3, 0.0)):
        grad = check_losses(z, idx, "sigmoid", cu, gb, gz)[2]
    far = (z.float() > 20) & (z.float() < 40)
    if T > 20:  # (two experts and more in a row: their shares pull against each other)
        assert far.any() and (grad[far] != 0).float().mean() > 0.99
