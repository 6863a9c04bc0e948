"""zmoe.functional.router_losses on the GPU against float64 (oracle.router_oracle).

Tolerances. An exponential is off by 2 |z| + 2 roundings: the difference z - max and its product with log2 e, each rounded to
2^-24 of it, and the instruction itself (and one more for a reciprocal). A share ph = p / sum p has those, as many in the sum,
which adds at most 16 in a lane and 6 over lanes, and 3 in quotients: 2 (2 range + 2) + 25 =: u units of 2^-24, range the largest
|z - max| (or |z| for a sigmoid) of the inputs. The losses add up shares of up to 16 tokens in f32 and the rest in double, and
are rounded once: u + 16 + 2 (twice u for the square of the logsumexp, which is a logarithm of such a sum: off by u / |lse|
units at most, and lse^2 is its own magnitude where |lse| >= 1; below, u 2^-24 absolute). A grad has two shares, a sum over a row of
16 + 6, a sigmoid and four products: 3 u + 30. Half a step for the grad's own type."""

import math

import pytest
import torch

from helpers import gen
from oracle import router_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def inputs(T, E, k, dt, dev, seed=0):
    g = gen(seed + 7 * T + E)
    z = (torch.randn(T, E, generator=g) * 1.5 + torch.randn(E, generator=g) * 0.5).to(DT[dt]).to(dev)
    return z, torch.topk(z.float(), k).indices


def units(z, score):
    f = z.float()
    f = f[torch.isfinite(f) & (f > torch.finfo(z.dtype).min)]
    span = 0.0 if f.numel() == 0 else float(f.abs().max()) * (2 if score == "softmax" else 1)
    return 2 * (2 * span + 2) + 25


def check(z, idx, score, cu=None, gb=0.3, gz=0.05):
    from zmoe.functional import router_losses

    leaf = z.detach().clone().requires_grad_(True)
    balance, zl = router_losses(leaf, idx, score, cu)
    assert balance.shape == zl.shape == () and balance.dtype == zl.dtype == torch.float32
    vb, vz, _, _ = O.losses(z, idx, score, cu)
    u = units(z, score)
    for what, got, val in (("balance", balance, vb), ("z", zl, vz)):
        bound = (2 * u + 18) * 2.0 ** -24 * max(abs(float(val)), 1.0 if what == "z" else 0.0)
        assert abs(float(got) - float(val)) <= bound, (what, float(got), float(val), bound)
    torch.autograd.backward([balance, zl], [torch.tensor(gb, device=z.device), torch.tensor(gz, device=z.device)])
    val, mag = O.losses_backward(z, idx, score, cu, float(torch.tensor(gb)), float(torch.tensor(gz)))
    half = 2.0 ** -8 if z.dtype == torch.bfloat16 else 2.0 ** -24
    bound = half * val.abs() + (3 * u + 30) * 2.0 ** -24 * mag + 1e-38
    bad = (leaf.grad.double() - val).abs() > bound
    assert not bad.any(), (int(bad.sum()), float(((leaf.grad.double() - val).abs() / bound).max()))
    assert leaf.grad.dtype == z.dtype
    return balance.detach(), zl.detach(), leaf.grad


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (2, 64, 4), (63, 32, 2), (64, 65, 3), (65, 128, 8), (517, 60, 6),
                                   (1000, 256, 8), (130, 300, 4), (97, 512, 8), (70, 1000, 10), (33, 1024, 16)])
def test_widths(T, E, k, score, dt, hip_device):
    z, idx = inputs(T, E, k, dt, hip_device)
    check(z, idx, score)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
def test_sequences(score, wide, hip_device):
    """Ragged ones, empty ones, ones that end in and at the borders of a workgroup's tile, tokens outside."""
    T = 1000
    z, idx = inputs(T, 96, 4, "f32", hip_device)
    for cu in ([0, T], [3, 997], [0, 1, 2, 3, 64, 128, 129, 500, T], [0, 0, 0, 10, 10, 640, 640], [64, 128], [63, 65, 191, 192],
               list(range(0, T + 1, 10)), [5, 5], [0, T, T, T], list(range(100, 300))):
        cu_t = torch.tensor(cu, dtype=wide, device=hip_device)
        _, _, grad = check(z, idx, score, cu_t)
        assert not grad[:cu[0]].any() and not grad[cu[-1]:].any()


def test_one_sequence_is_all_tokens(hip_device):
    from zmoe.functional import router_losses

    z, idx = inputs(333, 64, 2, "bf16", hip_device)
    a = check(z, idx, "softmax")
    b = check(z, idx, "softmax", torch.tensor([0, 333], device=hip_device))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    c = router_losses(z.view(3, 111, 64), idx.view(3, 111, 2), "softmax")
    assert torch.equal(c[0], a[0]) and torch.equal(c[1], a[1])


def test_no_tokens(hip_device):
    from zmoe.functional import router_losses

    z = torch.zeros(0, 16, device=hip_device, requires_grad=True)
    idx = torch.zeros(0, 2, dtype=torch.int64, device=hip_device)
    for cu in (None, torch.tensor([0, 0, 0], device=hip_device)):
        b, zl = router_losses(z, idx, "softmax", cu)
        (b + zl).backward()
        assert float(b) == 0.0 and float(zl) == 0.0 and z.grad.shape == (0, 16)
    z, idx = inputs(20, 16, 2, "f32", hip_device)
    b, zl, grad = check(z, idx, "sigmoid", torch.tensor([7, 7, 7], device=hip_device))
    assert float(b) == 0.0 and float(zl) == 0.0 and not grad.any()


def test_borders_out_of_range(hip_device):
    """Borders outside the tokens are cut to them."""
    from zmoe.functional import router_losses

    z, idx = inputs(100, 32, 2, "f32", hip_device)
    a = router_losses(z, idx, "softmax", torch.tensor([-5, 40, 1 << 20], device=hip_device))
    b = router_losses(z, idx, "softmax", torch.tensor([0, 40, 100], device=hip_device))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_masked_logits(hip_device):
    """Experts of -inf, and tokens that have nothing else: no part in either loss, no grad. Ids outside are not counted."""
    for score in ("sigmoid", "softmax"):
        for dt in ("f32", "bf16"):
            z, idx = inputs(150, 48, 4, dt, hip_device)
            z[:, 40:] = -math.inf
            z[7] = -math.inf
            z[100:103] = -math.inf
            _, _, grad = check(z, idx, score, torch.tensor([0, 90, 150], device=hip_device))
            assert torch.isfinite(grad).all() and not grad[7].any() and not grad[:, 40:].any()
    from zmoe.functional import router_losses

    z, idx = inputs(50, 16, 2, "f32", hip_device)
    a, _ = router_losses(z, idx, "softmax")
    more = torch.cat([idx, torch.full((50, 2), 16, device=hip_device), torch.full((50, 2), -1, device=hip_device)], 1)
    b, _ = router_losses(z, more, "softmax")
    torch.testing.assert_close(a, b * 3)  # the mean is over k = 6 now


def test_nan_and_inf(hip_device):
    """A NaN reaches the losses and its own token's grad, and no other row's own terms."""
    from zmoe.functional import router_losses

    z, idx = inputs(40, 16, 2, "f32", hip_device)
    _, _, clean = check(z, idx, "softmax")
    z[9, 3] = math.nan
    leaf = z.requires_grad_(True)
    b, zl = router_losses(leaf, idx, "softmax")
    torch.autograd.backward([b, zl], [torch.tensor(0.3, device=hip_device), torch.tensor(0.05, device=hip_device)])
    assert torch.isnan(b) and torch.isnan(zl) and torch.isnan(leaf.grad[9]).all()
    ok = torch.arange(40) != 9
    assert torch.equal(leaf.grad[ok.to(hip_device)], clean[ok.to(hip_device)])


def test_one_loss_unused(hip_device):
    from zmoe.functional import router_losses

    z, idx = inputs(90, 64, 4, "f32", hip_device)
    for which in (0, 1):
        leaf = z.clone().requires_grad_(True)
        router_losses(leaf, idx, "sigmoid")[which].backward()
        val, mag = O.losses_backward(z, idx, "sigmoid", None, 1.0 - which, float(which))
        assert ((leaf.grad.double() - val).abs() <= (3 * units(z, "sigmoid") + 30) * 2.0 ** -24 * mag + 1e-38).all()


def test_runs_alike(hip_device):
    """Sums in a fixed order: the same bits every time."""
    z, idx = inputs(20000, 128, 8, "bf16", hip_device)
    cu = torch.tensor([0, 3000, 3001, 15000, 20000], device=hip_device)
    a = check(z, idx, "softmax", cu)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(a, check(z, idx, "softmax", cu)))


def test_strides(hip_device):
    from zmoe.functional import router_losses

    z, idx = inputs(64, 200, 4, "f32", hip_device)
    a = router_losses(z[:, 20:148].contiguous(), idx.clamp(max=127), "softmax")
    b = router_losses(z[:, 20:148], idx.clamp(max=127).t().contiguous().t().to(torch.int32), "softmax")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals(hip_device):
    from zmoe.functional import router_losses

    z, idx = inputs(10, 16, 2, "f32", hip_device)
    cu = torch.tensor([0, 10], device=hip_device)
    for args in ((z, idx[:5], "softmax"), (z, idx, "tanh"), (z.half(), idx, "softmax"), (z.cpu(), idx.cpu(), "softmax"),
                 (z, idx.cpu(), "softmax"), (z, idx, "softmax", cu.float()), (z, idx, "softmax", cu[:1]),
                 (z, idx, "softmax", cu.cpu()), (z, idx, "softmax", cu.view(1, 2)),
                 (torch.zeros(2, 1025, device=hip_device), idx[:2], "softmax"),
                 (z[:, :1], idx, "softmax")):
        with pytest.raises(ValueError):
            router_losses(*args)


def test_graph(hip_device):
    """A captured training step on sequences that change between replays; two graphs in turn."""
    from zmoe.functional import router_losses

    def step(leaf, idx, cu):
        b, zl = router_losses(leaf, idx, "sigmoid", cu)
        grad, = torch.autograd.grad(0.02 * b + 0.001 * zl, leaf)
        return b.detach(), zl.detach(), grad

    def make(seed):
        z, idx = inputs(600, 64, 4, "bf16", hip_device, seed)
        g = gen(seed)
        return z.requires_grad_(True), idx, torch.randint(0, 601, (8,), generator=g).sort().values.int().to(hip_device)

    sets = [make(1), make(2)]
    side = torch.cuda.Stream(hip_device)
    side.wait_stream(torch.cuda.current_stream(hip_device))
    with torch.cuda.stream(side):
        for s in sets:
            step(*s)
    torch.cuda.current_stream(hip_device).wait_stream(side)
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*s)
        graphs.append((g, out))
    for seed in (3, 4, 5):
        for i, ((g, out), s) in enumerate(zip(graphs, sets)):
            with torch.no_grad():
                for t, n in zip(s, make(seed + 20 * i)):
                    t.copy_(n)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, out), s in zip(graphs, sets):
            for a, b in zip(out, step(*s)):
                assert torch.equal(a, b)


def test_compiled(hip_device):
    from zmoe.functional import router_losses

    z, idx = inputs(50, 64, 4, "bf16", hip_device)
    cu = torch.tensor([0, 20, 50], device=hip_device)

    def f(z):
        b, zl = router_losses(z, idx, "softmax", cu)
        return 0.5 * b + 0.25 * zl

    a, b = z.clone().requires_grad_(True), z.clone().requires_grad_(True)
    f(a).backward()
    torch.compile(f, fullgraph=True)(b).backward()
    assert torch.equal(a.grad, b.grad)
