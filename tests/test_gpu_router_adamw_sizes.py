"""Calls of the router's forms, its losses and the AdamW step at the far ends: offsets past 2^31 elements, one token, the most
experts, slots, groups, sequences and tensors; and what autograd does around them."""

import math

import pytest
import torch

from helpers import gen

pytestmark = pytest.mark.gpu


def test_logits_past_2_31_elements(hip_device):
    """The last tokens of 4.4 GB of logits, as a call on them alone gives them."""
    from zmoe.functional import route, router_losses

    T, E, k, tail = (1 << 21) + 4099, 1024, 8, 500
    z = torch.empty(T, E, dtype=torch.bfloat16, device=hip_device)
    g = torch.Generator(device=hip_device).manual_seed(1)
    for a in range(0, T, 1 << 18):
        z[a:a + (1 << 18)].normal_(generator=g)
    z.requires_grad_(True)
    end = z.detach()[-tail:].clone().requires_grad_(True)
    dw = torch.randn(T, k, device=hip_device, generator=g)
    for score, renormalize in (("softmax", False), ("sigmoid", True)):
        idx, w = route(z, k, None, score, 8, 3, 2, renormalize)
        idx2, w2 = route(end, k, None, score, 8, 3, 2, renormalize)
        assert torch.equal(idx[-tail:], idx2) and torch.equal(w[-tail:], w2)
        grad, = torch.autograd.grad(w, z, dw)
        grad2, = torch.autograd.grad(w2, end, dw[-tail:])
        assert torch.equal(grad[-tail:], grad2)
        del grad
    # the last sequence alone has tokens: the losses are those of its tokens
    cu = torch.tensor([T - tail, T], dtype=torch.int64, device=hip_device)
    a = router_losses(z, idx, "softmax", cu)
    b = router_losses(end, idx2, "softmax")
    for x, y in zip(a, b):
        assert abs(float(x) - float(y)) <= 2e-6 * abs(float(y))
    ga, = torch.autograd.grad(a[0] + a[1], z)
    gb, = torch.autograd.grad(b[0] + b[1], end)
    assert not ga[:T - tail].any()
    assert float((ga[-tail:].double() - gb.double()).norm()) <= 2.0 ** -8 * float(gb.double().norm())


@pytest.mark.parametrize("bits", [32, 8])
def test_tensor_past_2_31_elements(bits, hip_device):
    """One bf16 parameter of 2^31 + 5003 elements: its first and last blocks as small tensors have them."""
    from zmoe.adamw import AdamW

    n, part = (1 << 31) + 5003, 4096
    start = (n - part) // 256 * 256  # a whole number of blocks in
    p = torch.zeros(n, dtype=torch.bfloat16, device=hip_device)
    g = torch.zeros(n, dtype=torch.bfloat16, device=hip_device)
    for a in (0, start):
        p[a:a + part].normal_()
        g[a:a + part].normal_()
    g[start:].normal_()
    parts = [p[:part].clone(), p[start:].clone()]
    big = p.requires_grad_(True)
    big.grad = g
    opt = AdamW([big], lr=1e-2, state_bits=bits, max_grad_norm=1.0)
    small = [t.requires_grad_(True) for t in parts]
    two = AdamW(small, lr=1e-2, state_bits=bits, max_grad_norm=1.0)
    small[0].grad, small[1].grad = g[:part].clone(), g[start:].clone()
    for _ in range(2):
        opt.step()
        two.step()
    assert abs(float(opt.grad_norm) - float(two.grad_norm)) <= 2.0 ** -23 * float(two.grad_norm)
    for a, q in zip((slice(0, part), slice(start, n)), small):
        assert torch.equal(big[a], q)
        for name in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(opt.state[big][name][a], two.state[q][name])
    if bits == 8:
        assert torch.equal(opt.state[big]["exp_avg_scale"][start // 256:], two.state[small[1]]["exp_avg_scale"])


def test_many_sequences(hip_device):
    """More sequences than are counted at once, most of one token or none (1e-5: some 170 roundings of 2^-24, where the losses'
    own tests count 3 (2 (2 range + 2) + 25) + 30 for a grad of logits in a range of 8)."""
    from oracle import router_oracle as O
    from zmoe.functional import router_losses

    T, S = 6000, 5000
    z = torch.randn(T, 16, generator=gen(1)).to(hip_device)
    idx = torch.topk(z, 2).indices
    cu = torch.randint(0, T + 1, (S + 1,), generator=gen(2)).sort().values.to(hip_device)
    leaf = z.clone().requires_grad_(True)
    b, q = router_losses(leaf, idx, "softmax", cu)
    vb, vz, _, _ = O.losses(z, idx, "softmax", cu)
    assert abs(float(b) - float(vb)) <= 1e-5 * float(vb) and abs(float(q) - float(vz)) <= 1e-5 * float(vz)
    (0.5 * b + 0.1 * q).backward()
    val, mag = O.losses_backward(z, idx, "softmax", cu, 0.5, float(torch.tensor(0.1)))
    assert ((leaf.grad.double() - val).abs() <= 1e-5 * mag + 1e-38).all()


def test_most_sequences(hip_device):
    """As many sequences as a call takes, of one token each and a few of none: a's formula is then a token's own counts
    (tolerances as above)."""
    from zmoe.functional import router_losses

    S, E, k = 1 << 20, 40, 2
    T = S - 3
    z = torch.randn(T, E, generator=gen(3)).to(hip_device)
    idx = torch.topk(z, k).indices
    cu = torch.arange(S + 1, device=hip_device).clamp(max=T)
    leaf = z.clone().requires_grad_(True)
    b, q = router_losses(leaf, idx, "softmax", cu)
    (0.5 * b + 0.25 * q).backward()
    z = z.double()
    ph, lse = torch.softmax(z, -1), torch.logsumexp(z, -1)
    a = torch.zeros_like(z).scatter_(1, idx, E / (k * T))
    vb, vz = float((a * ph).sum()), float(lse.square().mean())
    assert abs(float(b) - vb) <= 1e-5 * vb and abs(float(q) - vz) <= 1e-5 * vz
    dot = (a * ph).sum(-1, keepdim=True)
    zpart = 0.5 * lse[:, None] / T * ph
    val, mag = 0.5 * ph * (a - dot) + zpart, 0.5 * ph * (a + dot) + zpart.abs()
    assert ((leaf.grad.double() - val).abs() <= 1e-5 * mag + 1e-38).all()
    with pytest.raises(ValueError):
        router_losses(leaf, idx, "softmax", torch.arange(S + 2, device=hip_device).clamp(max=T))


def test_most_tensors(hip_device):
    """Some thousand tensors: many launches, each with its own table."""
    from zmoe.adamw import AdamW

    ps = [torch.zeros(1 + i % 300, device=hip_device, requires_grad=True) for i in range(2000)]
    for i, p in enumerate(ps):
        p.grad = torch.full_like(p, (-1.0) ** i)
    opt = AdamW(ps, lr=0.5, weight_decay=0.0, eps=0.0, max_grad_norm=1e9)
    opt.step()
    n = sum(p.numel() for p in ps)
    assert abs(float(opt.grad_norm) - math.sqrt(n)) <= 2.0 ** -22 * math.sqrt(n)
    for i, p in enumerate(ps):
        assert float((p.detach() + 0.5 * (-1.0) ** i).abs().max()) <= 1e-6, i


def test_eps_of_zero_and_subnormal_second_moments(hip_device):
    """Without eps an element with grads of 1e-21 (a subnormal second moment) still steps by about lr."""
    from zmoe.adamw import AdamW

    for bits in (32, 8):
        p = torch.zeros(512, device=hip_device, requires_grad=True)
        p.grad = torch.full_like(p, 1e-21)
        opt = AdamW([p], lr=1e-3, betas=(0.9, 0.9), weight_decay=0.0, eps=0.0, state_bits=bits)
        opt.step()
        # v = 1e-43 is 71 units of 2^-149: its root is off by 1 / 142 at most
        assert float((p.detach() / -1e-3 - 1).abs().max()) <= 0.01


def test_second_derivatives_are_refused(hip_device):
    """create_graph gives the same first derivative; one through it raises, as for the framework's other functions."""
    from zmoe.functional import route, router_losses

    z = torch.randn(6, 16, generator=gen(3)).to(hip_device).requires_grad_(True)
    idx, w = route(z, 3, None, "softmax", renormalize=False)
    balance, _ = router_losses(z, idx, "softmax")
    for out in ((w * w.detach()).sum(), balance):
        a, = torch.autograd.grad(out, z, retain_graph=True)
        b, = torch.autograd.grad(out, z, create_graph=True)
        assert torch.equal(a, b)
        with pytest.raises(RuntimeError):
            b.sum().backward()


def test_under_checkpointing_and_hooks(hip_device):
    from torch.utils.checkpoint import checkpoint

    from zmoe.functional import route, router_losses

    def f(z):
        idx, w = route(z, 3, None, "softmax", renormalize=False)
        b, q = router_losses(z, idx, "softmax")
        return (w * w).sum() + b + 0.1 * q

    z = torch.randn(40, 16, generator=gen(4)).to(hip_device)
    a, b, c = (z.clone().requires_grad_(True) for _ in range(3))
    f(a).backward()
    checkpoint(f, b, use_reentrant=False).backward()
    with torch.autograd.graph.save_on_cpu():
        out = f(c)
    out.backward()
    assert torch.equal(a.grad, b.grad) and torch.equal(a.grad, c.grad)


def test_changed_inputs_are_noticed(hip_device):
    from zmoe.functional import route, router_losses

    z = torch.randn(6, 16, generator=gen(5)).to(hip_device).requires_grad_(True)
    y = z * 1.0
    idx, w = route(y, 2, None, "softmax")
    b, _ = router_losses(y, idx, "softmax")
    with torch.no_grad():
        y.add_(1.0)
    for out in (w.sum(), b):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()


def test_two_calls_at_once(hip_device):
    """Calls on two streams side by side: each has scratch of its own."""
    from zmoe.adamw import AdamW
    from zmoe.functional import router_losses

    zs = [torch.randn(3000, 64, generator=gen(i)).to(hip_device) for i in range(2)]
    idxs = [torch.topk(z, 4).indices for z in zs]
    want = [router_losses(z, i, "softmax") for z, i in zip(zs, idxs)]
    ps = [[torch.randn(50000, generator=gen(10 + i)).to(hip_device).requires_grad_(True)] for i in range(2)]
    twins = [[p[0].detach().clone().requires_grad_(True)] for p in ps]
    opts, ones = ([AdamW(p, state_bits=8, max_grad_norm=1.0) for p in group] for group in (ps, twins))
    for p, q in zip(ps, twins):
        p[0].grad = q[0].grad = torch.ones_like(p[0])
    for o in ones:
        for _ in range(5):
            o.step()
    streams = [torch.cuda.Stream(hip_device) for _ in range(2)]
    got = [None, None]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream(hip_device))
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = router_losses(zs[i], idxs[i], "softmax")
                opts[i].step()
    for s in streams:
        torch.cuda.current_stream(hip_device).wait_stream(s)
    for i in range(2):
        assert torch.equal(got[i][0], want[i][0]) and torch.equal(got[i][1], want[i][1])
        assert torch.equal(ps[i][0], twins[i][0])


def test_grads_of_other_layouts_and_types(hip_device):
    """A list that the native form does not take: both types in a group, a grad that is a view of another order."""
    from zmoe.adamw import AdamW

    a = torch.randn(30, 20, generator=gen(6)).to(hip_device)
    mixed = [a.clone().requires_grad_(True), a.bfloat16().requires_grad_(True)]
    alone = [a.clone().requires_grad_(True), a.bfloat16().requires_grad_(True)]
    g = torch.randn(20, 30, generator=gen(7)).to(hip_device).t()
    for group in (mixed, alone):
        group[0].grad, group[1].grad = g, g.bfloat16().contiguous()
    one = AdamW(mixed)
    two = [AdamW([alone[0]]), AdamW([alone[1]])]
    one.step()
    for o in two:
        o.step()
    assert all(torch.equal(p, q) for p, q in zip(mixed, alone))
