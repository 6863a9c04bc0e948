"""zmoe.functional.route on the GPU against float64 (oracle.router_oracle): the experts exactly, weights and grads within
bounds counted from the roundings.

Tolerances. A probability is rounded once, a weight is a sum of k of them, a quotient and a product: (k + 4) 2^-24 of the
value. The grad of a sigmoid's or a renormalised softmax's logit goes through two such sums, a quotient and some six
products of f32 numbers: (2 k + 12) 2^-24 of the magnitudes that it is added up from. Where a softmax is formed again in f32
(not renormalised) its p is off by 2 |z - max| + 2 roundings (the difference, its product with log2 e, the instruction), and as
much again in their sum, which adds at most 16 in a lane and 6 over lanes: 2 (2 range + 2) + 22 more. Rounding to the grad's type adds
half a step.
"""

import math

import pytest
import torch

from helpers import gen
from oracle import router_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def logits_of(T, E, dt, dev, seed=0, std=1.5):
    g = gen(seed + 31 * T + E)
    return (torch.randn(T, E, generator=g) * std + torch.randn(E, generator=g) * 0.5).to(DT[dt]).to(dev)


def close(what, got, val, mag, units):
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    assert got.shape == val.shape, (what, got.shape, val.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(val)), what
    bound = half * val.abs() + units * 2.0 ** -24 * mag + 1e-38
    bad = (got.double() - val).abs() > bound
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - val).abs() / bound).nan_to_num().max()))


def check(z, k, bias=None, score="sigmoid", groups=1, top_groups=1, group_scores=2, renormalize=True, scale=1.0, seed=5):
    from zmoe.functional import route

    gs = group_scores if groups > 1 else 1
    leaf = z.detach().clone().requires_grad_(True)
    idx, w = route(leaf, k, bias, score, groups, top_groups, group_scores, renormalize, scale)
    want = O.select(z, k, bias, score, groups, top_groups, gs)
    assert idx.dtype == torch.int64 and torch.equal(idx, want), (idx[(idx != want).any(1)][:3], want[(idx != want).any(1)][:3])
    val = O.weights(z, idx, score, renormalize, scale)
    assert w.dtype == torch.float32
    close("w", w.detach(), val, val.abs(), k + 4)
    dw = torch.randn(w.shape, generator=gen(seed)).to(z.device)
    w.backward(dw)
    val, mag = O.weights_backward(z, idx, dw, score, renormalize, scale)
    zf = z.float()
    span = (zf.amax(-1) - zf.masked_fill(zf == -math.inf, math.inf).amin(-1)).nan_to_num(0, 0, 0).clamp(0, 200).max() if z.numel() else 0
    again = 0 if score == "sigmoid" or renormalize else 2 * (2 * float(span) + 2) + 22
    assert leaf.grad.dtype == z.dtype
    close("d logits", leaf.grad, val, mag, 2 * k + 12 + again)
    with torch.no_grad():
        idx2, w2 = route(z, k, bias, score, groups, top_groups, group_scores, renormalize, scale)
    assert torch.equal(idx, idx2) and torch.equal(w.detach(), w2)
    return idx, w.detach(), leaf.grad


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (3, 2, 2), (5, 5, 3), (17, 8, 8), (1, 64, 8), (33, 60, 6), (70, 65, 1),
                                   (257, 72, 4), (300, 128, 8), (64, 130, 9), (31, 200, 16), (130, 256, 8), (9, 256, 64),
                                   (20, 300, 7), (12, 512, 33), (7, 1000, 10), (11, 1024, 64)])
def test_widths(T, E, k, score, dt, hip_device):
    z = logits_of(T, E, dt, hip_device)
    bias = (torch.randn(E, generator=gen(E)) * 0.05).to(hip_device)
    check(z, k, bias, score)
    check(z, k, None, score, renormalize=False, scale=2.5)


@pytest.mark.parametrize("E,G,g,k", [(8, 2, 1, 4), (12, 3, 2, 5), (32, 8, 4, 4), (64, 64, 7, 7), (160, 8, 3, 6), (256, 8, 4, 8),
                                     (96, 6, 6, 8), (250, 5, 2, 8), (384, 16, 3, 8), (1024, 32, 5, 12), (74, 2, 1, 3)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("group_scores", [1, 2])
def test_groups(E, G, g, k, score, with_bias, group_scores, hip_device):
    if group_scores > E // G:
        group_scores = 1
    bias = (torch.randn(E, generator=gen(E)) * 0.05).to(hip_device) if with_bias else None
    for T, dt, renormalize in ((37, "bf16", True), (21, "f32", False)):
        check(logits_of(T, E, dt, hip_device, seed=3), k, bias, score, G, g, group_scores, renormalize, 1.5)


def test_many_tokens(hip_device):
    """More tokens than the grid holds at once."""
    for E, score in ((64, "softmax"), (256, "sigmoid"), (520, "softmax")):
        check(logits_of(70001 if E < 512 else 9001, E, "bf16", hip_device), 4, None, score, renormalize=E != 64)


def test_equal_scores(hip_device):
    """Equal scores go to the lowest numbers, with and without a bias and over groups."""
    z = torch.zeros(5, 48, device=hip_device)
    z[1, 40], z[2, 7], z[2, 9] = 1.0, -1.0, 2.0
    z[3], z[4] = -0.0, torch.arange(48, device=hip_device) % 3
    for bias in (None, torch.zeros(48, device=hip_device), torch.full((48,), 0.5, device=hip_device)):
        for score in ("sigmoid", "softmax"):
            check(z, 6, bias, score)
            check(z, 6, bias, score, groups=4, top_groups=2, group_scores=2)
    few = logits_of(2000, 256, "bf16", hip_device).mul(4).round().div(4)  # many equal logits
    check(few, 8, torch.zeros(256, device=hip_device), "sigmoid", 8, 4)
    check(few, 8, None, "softmax")


def test_masked_experts_and_rows(hip_device):
    """Experts of -inf, of the type's lowest value, rows of them alone; the bias decides among what has no probability."""
    from zmoe.functional import route

    for dt in ("f32", "bf16"):
        z = logits_of(9, 64, dt, hip_device)
        z[0, 5:] = -math.inf
        z[1, ::2] = torch.finfo(z.dtype).min
        z[2] = -math.inf
        z[3] = torch.finfo(z.dtype).min
        z[4, :60] = -math.inf
        bias = (torch.randn(64, generator=gen(2)) * 0.1).to(hip_device)
        for score in ("sigmoid", "softmax"):
            for renormalize in (True, False):
                idx, w, grad = check(z, 8, None, score, renormalize=renormalize)
                assert not w[2].any() and not grad[2].any() and torch.isfinite(w).all() and torch.isfinite(grad).all()
                check(z, 8, bias, score, 4, 2, renormalize=renormalize)
    idx, w = route(torch.full((1, 4), -math.inf, device=hip_device), 2, torch.tensor([0.0, 0, 1, 2], device=hip_device), "softmax")
    assert idx.tolist() == [[3, 2]] and not w.any()


def test_values_that_are_not_finite(hip_device):
    """NaN ranks first and stays in its own row; +inf is a sigmoid of 1, and a softmax row of NaN."""
    from zmoe.functional import route

    z = logits_of(6, 32, "f32", hip_device)
    clean = route(z, 4, None, "softmax")
    z[1, 9], z[4, 3] = math.nan, math.inf
    for score in ("sigmoid", "softmax"):
        for bias in (None, torch.zeros(32, device=hip_device)):
            leaf = z.clone().requires_grad_(True)
            idx, w = route(leaf, 4, bias, score)
            w.sum().backward()
            assert idx[1, 0] == 9 if score == "sigmoid" or bias is None else True
            assert torch.isnan(w[1]).all() and torch.isnan(leaf.grad[1, idx[1]]).all()
            if score == "sigmoid":
                assert idx[4, 0] == 3 and torch.isfinite(w[4]).all() and torch.isfinite(leaf.grad[4]).all()
            else:
                assert torch.isnan(w[4]).all()
            for r in (0, 2, 3, 5):
                assert torch.isfinite(w[r]).all() and torch.isfinite(leaf.grad[r]).all()
    got = route(z, 4, None, "softmax")
    ok = [0, 2, 3, 5]
    assert torch.equal(got[0][ok], clean[0][ok]) and torch.equal(got[1][ok], clean[1][ok])


def test_one_expert_of_one(hip_device):
    """k = 1, renormalised: the weight is the scale whatever the logits are, the grad rounding errors of it at most."""
    z = logits_of(50, 40, "f32", hip_device)
    for score in ("sigmoid", "softmax"):
        check(z, 1, None, score, scale=3.0)


def test_strides_shapes_and_types(hip_device):
    from zmoe.functional import route

    big = logits_of(40, 300, "f32", hip_device)
    ref = route(big[:, 8:136].contiguous(), 5, None, "softmax")
    for view in (big[:, 8:136], big[:, 8:136].t().contiguous().t()):
        got = route(view, 5, None, "softmax")
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    off = torch.empty(40 * 128 + 3, device=hip_device)[3:].view(40, 128).copy_(big[:, 8:136])  # off 16 bytes
    assert torch.equal(route(off, 5, None, "softmax")[0], ref[0])
    shaped = big[:, 8:136].reshape(2, 4, 5, 128).requires_grad_(True)
    idx, w = route(shaped, 5, torch.zeros(128, device=hip_device, dtype=torch.bfloat16), "softmax")
    assert idx.shape == w.shape == (2, 4, 5, 5)
    # an output grad that is expanded
    w.sum().backward()
    assert shaped.grad.shape == shaped.shape
    none = torch.zeros(0, 128, device=hip_device, requires_grad=True)
    idx, w = route(none, 5)
    w.sum().backward()
    assert idx.shape == (0, 5) and none.grad.shape == (0, 128)


def test_refusals(hip_device):
    from zmoe.functional import route

    z = torch.zeros(3, 32, device=hip_device)
    b = torch.zeros(32, device=hip_device)
    for args, kw in (((z, 0), {}), ((z, 33), {}), ((z, 65), {}), ((z, 4, b[:5]), {}), ((z, 4), dict(score="tanh")),
                     ((z, 4), dict(groups=5)), ((z, 4), dict(groups=0)), ((z, 4), dict(groups=4, top_groups=5)),
                     ((z, 4), dict(groups=4, top_groups=0)), ((z, 9), dict(groups=4, top_groups=1)),
                     ((z, 4), dict(groups=32, top_groups=8)), ((z, 4), dict(groups=4, group_scores=3)),
                     ((z.half(), 4), {}), ((z.cpu(), 4), {}), ((z, 4, b.cpu()), {}), ((z.double(), 4), {}),
                     ((torch.zeros(2, 1025, device=hip_device), 4), {})):
        with pytest.raises(ValueError):
            route(*args, **kw)
    with pytest.raises(RuntimeError):
        route(z, 4, b.requires_grad_(True))


def test_other_stream_and_graphs(hip_device):
    """Two graphs of training steps with tensors of their own, replayed in turn, also on another stream."""
    from zmoe.functional import route

    def step(leaf, dw, bias):
        idx, w = route(leaf, 6, bias, "softmax", 8, 3, 1, False, 4.0)
        grad, = torch.autograd.grad(w, leaf, dw)
        return idx, w.detach(), grad

    def make(seed):
        z = logits_of(700, 160, "f32", hip_device, seed=seed).requires_grad_(True)
        return z, torch.randn(700, 6, generator=gen(seed)).to(hip_device), (torch.randn(160, generator=gen(seed + 1)) * 0.1).to(hip_device)

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
    for seed in (5, 6, 7):
        for (g, out), s in zip(graphs, sets):
            with torch.no_grad():
                for t, n in zip(s, make(seed)):
                    t.copy_(n)
            side.wait_stream(torch.cuda.current_stream(hip_device))
            with torch.cuda.stream(side):
                g.replay()
            torch.cuda.current_stream(hip_device).wait_stream(side)
            torch.cuda.synchronize()
            for a, b in zip(out, step(*s)):
                assert torch.equal(a, b)
            seed += 10


def test_compiled(hip_device):
    from zmoe.functional import route

    def f(z, dw):
        idx, w = route(z, 4, None, "softmax", 4, 2, 1, False, 2.0)
        return idx, (w * dw).sum()

    z, dw = logits_of(50, 64, "bf16", hip_device), torch.randn(50, 4, device=hip_device)
    a, b = z.clone().requires_grad_(True), z.clone().requires_grad_(True)
    ia, la = f(a, dw)
    ib, lb = torch.compile(f, fullgraph=True)(b, dw)
    la.backward()
    lb.backward()
    assert torch.equal(ia, ib) and torch.equal(a.grad, b.grad)
    torch.testing.assert_close(la, lb)


@pytest.mark.parametrize("E,G,g,k", [(130, 10, 3, 8), (160, 8, 3, 6), (200, 4, 2, 9), (250, 5, 2, 8), (256, 8, 4, 8), (256, 64, 9, 17),
                                     (192, 64, 64, 12), (300, 6, 2, 8), (384, 16, 3, 8), (512, 8, 4, 8), (510, 2, 1, 5)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T", [600, 4097])
def test_groups_of_many_tokens(E, G, g, k, score, T, hip_device):
    """A token's experts over fewer or more lanes, by the number of tokens: groups and biases in each of them, experts
    that a bias rules out among those that have to be taken, rows without any."""
    bias = (torch.randn(E, generator=gen(E)) * 0.05).to(hip_device)
    out = bias.clone()
    out[torch.randperm(E, generator=gen(E + 1))[: E - 3].to(hip_device)] = -math.inf  # three are left, fewer than k
    for dt, with_bias, two in (("bf16", bias, 2), ("f32", None, 1), ("f32", out, 2), ("bf16", out, 1)):
        z = logits_of(T, E, dt, hip_device, seed=7)
        z[T // 2], z[-1, 3:] = -math.inf, -math.inf
        two = min(two, E // G)
        check(z, k, with_bias, score, G, g, two, dt == "bf16", 1.5)
        if G < 64:
            check(z, min(k, E // G), with_bias, score, renormalize=False)


def test_no_tokens(hip_device):
    from zmoe.functional import route

    for shape in ((0, 16), (3, 0, 200)):
        z = torch.zeros(*shape, device=hip_device, dtype=torch.bfloat16, requires_grad=True)
        idx, w = route(z, 4, torch.zeros(shape[-1], device=hip_device), "softmax")
        assert idx.shape == w.shape == (*shape[:-1], 4) and idx.dtype == torch.int64
        w.sum().backward()
        assert z.grad.shape == z.shape and z.grad.dtype == z.dtype
        with torch.no_grad():
            assert route(z, 4)[1].shape == (*shape[:-1], 4)
