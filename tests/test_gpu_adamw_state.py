"""zmoe.adamw.AdamW's steps around loads that it refuses."""

import pytest
import torch

from helpers import gen

pytestmark = pytest.mark.gpu


def pair(bits, dev, shapes=((700,), (40, 30)), **kw):
    """The same parameters and grads under two optimizers."""
    from zmoe.adamw import AdamW

    out = []
    for _ in range(2):
        params = [torch.randn(*s, generator=gen(3 + i)).to(dev).requires_grad_(True) for i, s in enumerate(shapes)]
        out.append((params, AdamW(params, lr=1e-2, state_bits=bits, **kw)))
    return out


def step(params, opt, seed):
    for i, p in enumerate(params):
        p.grad = torch.randn(*p.shape, generator=gen(seed + i)).to(p.device)
    opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_after_a_refused_load(bits, hip_device):
    """The moments of the other width are refused, and the next step is the one without that load."""
    (a, opt), (b, twin) = pair(bits, hip_device)
    step(a, opt, 10)
    step(b, twin, 10)
    (c, other), _ = pair(40 - bits, hip_device)
    step(c, other, 20)
    bad = opt.state_dict()
    with pytest.raises(ValueError):
        opt.load_state_dict({**bad, "state": {0: bad["state"][0], 1: other.state_dict()["state"][1]}})
    step(a, opt, 30)
    step(b, twin, 30)
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        assert all(t.dtype == twin.state[q][n].dtype and torch.equal(t, twin.state[q][n]) for n, t in opt.state[p].items())


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_under_inference_mode(bits, hip_device):
    """The state is a state for later, also of a first step under inference mode; steps go on as without it."""
    (a, opt), (b, twin) = pair(bits, hip_device, max_grad_norm=1.0)
    for seed in (10, 20, 30):
        step(b, twin, seed)
    for p in a:
        p.grad = torch.zeros_like(p)
    for seed, mode in ((10, True), (20, False), (30, True)):
        for i, p in enumerate(a):
            p.grad.copy_(torch.randn(*p.shape, generator=gen(seed + i)))
        with torch.inference_mode(mode):
            opt.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q) and not any(t.is_inference() for t in opt.state[p].values())
        assert all(torch.equal(t, twin.state[q][n]) for n, t in opt.state[p].items())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("timed", [False, True])
def test_parameters_of_inference_mode(bits, timed, hip_device):
    """Refused outside of it before anything moves, as every change in place of them."""
    from zmoe import profiling
    from zmoe.adamw import AdamW

    with torch.inference_mode():
        p = torch.ones(300, device=hip_device)
    opt = AdamW([p], state_bits=bits)
    p.grad = torch.ones(300, device=hip_device)
    if timed:  # the general form of the step
        profiling.enable("adamw")
    try:
        with pytest.raises(RuntimeError):
            opt.step()
    finally:
        profiling.disable()
        profiling.reset()
    assert torch.equal(p, torch.ones(300, device=hip_device))
    assert all(not t.any() for t in opt.state[p].values())
    with torch.inference_mode():
        opt.step()
        assert not (p == 1).any()
