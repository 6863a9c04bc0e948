"""oracle.norm_residual_oracle against torch's autograd of the formula and against differences (CPU, float64)."""

import pytest
import torch

from oracle import norm_residual_oracle as O


def formula(r, y, w1, w2, gate, scale, eps):
    norm = lambda a, w: a / torch.sqrt((a * a).mean(-1, keepdim=True) + eps) * (1 + w)  # noqa: E731
    u = y if w1 is None else norm(y, w1)
    h = scale * r + (u if gate is None else gate * u)
    return h, None if w2 is None else norm(h, w2)


@pytest.mark.parametrize("gate", [None, (7,), (5, 1), (5, 7)])
@pytest.mark.parametrize("post,nxt", [(True, True), (True, False), (False, True)])
def test_gradients(gate, post, nxt):
    torch.manual_seed(3)
    n, d, eps = 5, 7, 1e-3
    rnd = lambda *s: torch.randn(*s, dtype=torch.float64, requires_grad=True)  # noqa: E731
    args = [rnd(n, d), rnd(n, d), rnd(d) if post else None, rnd(d) if nxt else None, rnd(*gate) if gate else None,
            torch.tensor(0.7, dtype=torch.float64, requires_grad=True)]
    dr, dx = torch.randn(n, d, dtype=torch.float64), torch.randn(n, d, dtype=torch.float64) if nxt else None

    def loss(*leaves):
        it = iter(leaves)
        h, x = formula(*[None if a is None else next(it) for a in args], eps)
        return (h * dr).sum() + (0 if x is None else (x * dx).sum())

    leaves = [a for a in args if a is not None]
    val, mag = O.backward(*[None if a is None else a.detach() for a in args], eps, dr, dx)
    names = [m for m, a in zip(("r", "y", "w_post", "w_next", "gate", "scale"), args) if a is not None]
    for name, g in zip(names, torch.autograd.grad(loss(*leaves), leaves)):
        torch.testing.assert_close(val[name], g, rtol=1e-10, atol=1e-10)
        assert (mag[name] >= val[name].abs() * (1 - 1e-12)).all()
    h = 1e-6
    for name, leaf in zip(names, leaves):  # central differences along one random direction each
        v = torch.randn_like(leaf)
        at = lambda s: loss(*[a + s * v if a is leaf else a for a in leaves]).item()  # noqa: E731
        got = float((val[name] * v).sum())
        assert abs((at(h) - at(-h)) / (2 * h) - got) <= 1e-6 * max(1.0, abs(got))
    f, _ = formula(*args, eps), None
    val, _, _ = O.forward(*[None if a is None else a.detach() for a in args], eps)
    torch.testing.assert_close(val["r"], f[0].detach())
    if nxt:
        torch.testing.assert_close(val["x"], f[1].detach())
