"""zmoe.adamw.AdamW where the step's denominator is small: no eps, one that is no normal f32 number, elements without a
grad, second moments that are no normal numbers.

Tolerances: tests/test_gpu_adamw.py's after one or two steps: 12 units of 2^-24 of the change for each step, 2 of the parameter,
and half a step of its type each time it is kept."""

import math

import pytest
import torch

from helpers import gen

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def made(p, **kw):
    from zmoe.adamw import AdamW

    return AdamW([p], **{**dict(lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1), **kw})


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("eps", [0.0, 1e-50, 1e-45, 1e-40, 1e-38, 1e-30, 1e-12, 1e-8])
def test_elements_without_a_grad(eps, dt, bits, hip_device):
    """Rows that no token used: decayed, and else as they were; the others by the formula."""
    p = torch.randn(900, generator=gen(1)).to(DT[dt]).to(hip_device).requires_grad_(True)
    opt = made(p, eps=eps, state_bits=bits)
    g = torch.randn(900, generator=gen(2)).to(DT[dt]).to(hip_device)
    g[g.abs() < 0.1] = 0.1
    g[200:700] = 0.0  # a block of 256 elements, and parts of two
    none = g == 0
    half = 2.0 ** -8 if dt == "bf16" else 2.0 ** -24
    want, off = p.detach().double(), 0.0
    for t in (1, 2):
        p.grad = g
        opt.step()
        m, v = (1 - 0.9 ** t) * g.double(), (1 - 0.95 ** t) * g.double().square()
        change = torch.where(none, 0.0, 1e-2 / (1 - 0.9 ** t) * m / (v.sqrt() / math.sqrt(1 - 0.95 ** t) + eps))
        if bits == 8 and t == 2:  # the first step's moments went through codes: what has no grad, alone
            change = torch.where(none, 0.0, math.nan)
        want = want * (1 - 1e-2 * 0.1) - change
        off = off + half * (want.abs() + off) + 2.0 ** -24 * (12 * t * change.abs() + 4 * want.abs()) + 1e-38
        ok = none if bits == 8 and t == 2 else torch.ones_like(none)
        assert torch.isfinite(p.detach()).all()
        assert ((p.detach().double() - want).abs() <= off)[ok].all(), t


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-40, 3e-39, 2e-38])
def test_squares_below_every_f32(eps, bits, hip_device):
    """g^2 is 0 in f32: the denominator is eps, whatever kind of number that is."""
    p = torch.zeros(600, device=hip_device, requires_grad=True)
    opt = made(p, eps=eps, state_bits=bits)
    g = torch.randn(600, generator=gen(5)).to(hip_device) * 1e-26
    p.grad = g
    opt.step()
    m = 0.1 * g.double()
    change = 0.1 * m / float(torch.tensor(eps))  # (eps is an f32 number in the step)
    # m is off by what an f32 near 2^-90 is, the quotient by two roundings and the product's
    assert ((p.detach().double() + change).abs() <= 12 * 2.0 ** -24 * change.abs()).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("beta2", [0.95, 0.999, 1 - 1e-6])
@pytest.mark.parametrize("eps", [2.0 ** -41, 2.0 ** -39, 2.0 ** -36, 2.0 ** -33, 1e-8])
def test_second_moments_below_the_normal_numbers(eps, beta2, bits, hip_device):
    """Roots of v' below 2^-126 count where eps does not drown them."""
    p = torch.zeros(512, device=hip_device, requires_grad=True)
    opt = made(p, eps=eps, betas=(0.9, beta2), state_bits=bits)
    top = math.sqrt(2.0 ** -126 / (1 - beta2))
    g = torch.linspace(0.9, 0.99, 512).to(hip_device) * top
    p.grad = g
    opt.step()
    v = ((1 - beta2) * g.double().square())
    assert (v < 2.0 ** -126).all()
    change = 0.1 * (0.1 * g.double()) / (v.sqrt() / math.sqrt(1 - beta2) + eps)
    assert ((p.detach().double() + change).abs() <= 12 * 2.0 ** -24 * change.abs()).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_second_moment_that_is_not_a_number_stays(bits, hip_device):
    """A moment of NaN makes the parameter NaN, with or without an eps."""
    for eps in (0.0, 1e-40, 1e-8):
        p = torch.zeros(256, device=hip_device, requires_grad=True)
        opt = made(p, eps=eps, state_bits=bits)
        p.grad = torch.ones(256, device=hip_device)
        opt.step()
        if bits == 32:
            opt.state[p]["exp_avg_sq"].fill_(math.nan)
        else:
            opt.state[p]["exp_avg_sq_scale"].fill_(math.nan)
        p.grad = torch.zeros(256, device=hip_device)
        opt.step()
        assert torch.isnan(p).all()
