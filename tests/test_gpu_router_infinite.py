"""The router's losses where a logit is +inf: logsumexp is inf there and a sigmoid 1, so that z is inf and a sigmoid's balance
loss and its grad stay finite; a softmax of such a row is NaN. Bounds as in tests/test_gpu_router_losses.py."""

import math

import pytest
import torch

from oracle import router_oracle as O
from test_gpu_router_losses import inputs, units

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (70, 64, 4), (130, 72, 3), (40, 160, 6), (65, 256, 8), (33, 1024, 16)])
@pytest.mark.parametrize("many", [1, 3])
def test_sigmoid(T, E, k, dt, many, hip_device):
    from zmoe.functional import router_losses

    z, idx = inputs(T, E, k, dt, hip_device)
    z[T // 2, 1:1 + many] = math.inf
    cu = torch.tensor([0, T // 3, T], device=hip_device)
    finite = z.clamp(max=1e30)  # a sigmoid of 1 as well, and lse takes no part
    leaf = z.clone().requires_grad_(True)
    balance, zl = router_losses(leaf, idx, "sigmoid", cu)
    u = units(z, "sigmoid")
    want = float(O.losses(finite, idx, "sigmoid", cu)[0])
    assert abs(float(balance) - want) <= (2 * u + 18) * 2.0 ** -24 * want and float(zl) == math.inf
    got, = torch.autograd.grad(balance, leaf, torch.tensor(0.3, device=hip_device))
    val, mag = O.losses_backward(finite, idx, "sigmoid", cu, float(torch.tensor(0.3)), 0.0)
    half = 2.0 ** -8 if dt == "bf16" else 2.0 ** -24
    assert ((got.double() - val).abs() <= half * val.abs() + (3 * u + 30) * 2.0 ** -24 * mag + 1e-38).all()
    # the z loss's grad is not a number in that row alone
    both, = torch.autograd.grad(sum(router_losses(leaf, idx, "sigmoid", cu)), leaf)
    rows = torch.isfinite(both).all(1)
    assert rows.sum() == T - 1 and not rows[T // 2]


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_softmax(dt, hip_device):
    from zmoe.functional import router_losses

    z, idx = inputs(40, 64, 4, dt, hip_device)
    z[7, 5] = math.inf
    leaf = z.clone().requires_grad_(True)
    balance, zl = router_losses(leaf, idx, "softmax")
    assert math.isnan(balance) and float(zl) == math.inf
    (balance + zl).backward()
    others = [r for r in range(40) if r != 7]
    assert torch.isnan(leaf.grad[7]).all() and torch.isfinite(leaf.grad[others]).all()


def test_a_nan_beside_it(hip_device):
    from zmoe.functional import router_losses

    for score in ("sigmoid", "softmax"):
        z, idx = inputs(40, 64, 4, "f32", hip_device)
        z[7, 5], z[7, 6] = math.inf, math.nan
        balance, zl = router_losses(z, idx, score)
        assert math.isnan(balance) and math.isnan(zl)
        z[7, 6] = -math.inf
        assert float(router_losses(z, idx, score)[1]) == math.inf
