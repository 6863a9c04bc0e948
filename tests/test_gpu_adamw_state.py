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
