"""oracle.router_oracle and oracle.adamw_oracle against torch's autograd, differences and plain statements (CPU, float64)."""

import math

import pytest
import torch

from oracle import adamw_oracle as A
from oracle import router_oracle as R

F64 = torch.float64


def difference(f, x, v, h=1e-6):
    return (f(x + h * v) - f(x - h * v)) / (2 * h)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renormalize,scale", [(True, 1.0), (True, 2.5), (False, 1.0), (False, 16.0)])
def test_weights_gradient(score, renormalize, scale):
    torch.manual_seed(1)
    z = torch.randn(6, 10, dtype=F64, requires_grad=True)
    idx = R.select(z.float(), 3, torch.randn(10) * 0.1, score, 2, 1, 2)
    dw = torch.randn(6, 3, dtype=F64)
    p = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, -1)
    w = p.gather(1, idx)
    w = scale * (w / w.sum(1, keepdim=True) if renormalize else w)
    torch.testing.assert_close(R.weights(z, idx, score, renormalize, scale), w.detach())
    val, mag = R.weights_backward(z, idx, dw, score, renormalize, scale)
    g, = torch.autograd.grad((w * dw).sum(), z)
    torch.testing.assert_close(val, g, rtol=1e-10, atol=1e-12)
    assert (mag >= val.abs() * (1 - 1e-12)).all()
    v = torch.randn_like(z)
    f = lambda x: float((R.weights(x, idx, score, renormalize, scale) * dw).sum())  # noqa: E731
    assert abs(difference(f, z.detach(), v) - float((val * v).sum())) < 1e-7


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("cu", [None, [0, 9], [1, 4, 4, 8], [2, 2, 7]])
def test_losses_gradient(score, cu):
    torch.manual_seed(2)
    z = torch.randn(9, 7, dtype=F64, requires_grad=True)
    idx = torch.topk(z.detach(), 2).indices
    cu_t = None if cu is None else torch.tensor(cu)
    balance, zl, _, n = R.losses(z, idx, score, cu_t)
    cu = [0, 9] if cu is None else cu
    p = torch.softmax(z, -1) if score == "softmax" else torch.sigmoid(z) / torch.sigmoid(z).sum(-1, keepdim=True)
    parts = []
    for a, b in zip(cu[:-1], cu[1:]):
        if b > a:
            f = torch.bincount(idx[a:b].reshape(-1), minlength=7).to(F64) * 7 / (2 * (b - a))
            parts.append((f * p[a:b].mean(0)).sum())
    want = sum(parts) / len(parts)
    want_z = torch.logsumexp(z[cu[0]:cu[-1]], -1).square().mean()
    assert n == cu[-1] - cu[0]
    torch.testing.assert_close(balance, want.detach())
    torch.testing.assert_close(zl, want_z.detach())
    val, mag = R.losses_backward(z, idx, score, cu_t, 0.3, 0.7)
    g, = torch.autograd.grad(0.3 * want + 0.7 * want_z, z)
    torch.testing.assert_close(val, g, rtol=1e-10, atol=1e-12)
    assert (mag >= val.abs() * (1 - 1e-12)).all()
    v = torch.randn_like(z)

    def f(x):
        b, q, _, _ = R.losses(x, idx, score, cu_t)
        return float(0.3 * b + 0.7 * q)

    assert abs(difference(f, z.detach(), v) - float((val * v).sum())) < 1e-7


def test_even_routing_balances_at_one():
    T, E, k = 12, 6, 2
    idx = (torch.arange(T * k) % E).view(T, k)
    for score in ("sigmoid", "softmax"):
        balance, _, _, _ = R.losses(torch.zeros(T, E), idx, score)
        assert abs(float(balance) - 1) < 1e-12


def test_selection():
    z = torch.tensor([[0.0, 3.0, 1.0, 3.0, -1.0, 2.0], [math.nan, 1.0, 1.0, 1.0, 9.0, 1.0], [-math.inf] * 6])
    assert R.select(z, 3, None, "softmax", 1, 1, 1).tolist() == [[1, 3, 5], [0, 4, 1], [0, 1, 2]]
    # groups of two: best ones 3 (experts 0, 1), 3 (2, 3), 2 (4, 5); by the sum of two, 1 + 3 comes first
    assert R.select(z[:1], 2, None, "sigmoid", 3, 1, 1).tolist() == [[1, 0]]
    assert R.select(z[:1], 2, None, "sigmoid", 3, 1, 2).tolist() == [[3, 2]]
    assert R.select(z[:1], 2, torch.tensor([0.0, 0, 0, 0, 5, 5]), "sigmoid", 3, 1, 2).tolist() == [[5, 4]]


def test_codes():
    for x, A_, want in ((0.25, 1.0, (64, 180)), (0.0625, 1.0, (32, 128)), (1.0, 1.0, (127, 255)), (0.0, 1.0, (0, 0)),
                        (1e-30, 1.0, (0, 1)), (3e-40, 3e-40, (127, 255)), (0.0, 0.0, (0, 0))):
        assert (A.code(x, A_, 2, 127), A.code(x, A_, 4, 255)) == want
    # 1/4 lies half-way between codes 63 and 64 (of the second moment, 1/16 between 127 and 128): up; a hair below: down
    assert A.code(0.25 - 2.0 ** -26, 1.0, 2, 127) == 63 and A.code(0.0625 - 2.0 ** -28, 1.0, 4, 255) == 127
    x = torch.randn(700)
    q, s, v = A.through_codes(x, False)
    assert s.numel() == 3 and (v.sign() == q.sign()).all()
    A_ = s.repeat_interleave(256)[:700]
    step = ((q.abs() + 1).double() ** 2 - q.abs().double() ** 2) / 127 ** 2 * A_.double()
    assert ((x.double() - v.double()).abs() <= step).all()


def test_step_is_torchs():
    torch.manual_seed(3)
    p = torch.randn(50, dtype=F64).requires_grad_(True)
    opt = torch.optim.AdamW([p], lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    q, m, v = p.detach().clone(), torch.zeros(50, dtype=F64), torch.zeros(50, dtype=F64)
    for t in range(1, 5):
        g = torch.randn(50, dtype=F64)
        p.grad = g
        opt.step()
        q, m, v, _ = A.step(q, g, m, v, t, 1e-2, (0.9, 0.95), 1e-8, 0.1)
        torch.testing.assert_close(q, p.detach(), rtol=1e-12, atol=1e-14)
