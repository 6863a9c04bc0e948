"""zmoe.adamw.AdamW on the GPU: against float64 (oracle.adamw_oracle), 8-bit codes exactly.

Tolerances. A moment in f32 has a product, a product and a fused sum: 4 roundings of its magnitude M = b1 M + (1 - b1) |g| (the
coefficients' own roundings among them; the clipped grad one or two more), and carries those of the steps before: 6 t units of
2^-24 M after t steps, for v, all of whose terms are positive, 8 t of itself. The change of a parameter is a quotient of m
and a root of v: m's units of M, half of v's, and some eight of its own; the decayed parameter has 2 units of its own, and
half a step of its type each time it is kept."""

import copy
import math

import pytest
import torch

from helpers import gen
from oracle import adamw_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
LR, BETAS, EPS, WD = 1e-2, (0.9, 0.95), 1e-8, 0.1


def tensors(shapes, dt, dev, seed=0, std=1.0):
    return [(torch.randn(*s, generator=gen(seed + 13 * i)) * std).to(DT[dt]).to(dev) for i, s in enumerate(shapes)]


def optimizer(params, **kw):
    from zmoe.adamw import AdamW

    return AdamW(params, **{**dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=WD), **kw})


SHAPES = [(1,), (3,), (5, 7), (256,), (255,), (257,), (4, 4, 33), (4096,), (4097,), (8191,), (64, 512), (100003,), (1, 1)]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("clip", [None, 0.5, 1e6])
def test_32_bits(dt, clip, hip_device):
    params = [p.requires_grad_(True) for p in tensors(SHAPES, dt, hip_device)]
    opt = optimizer(params, max_grad_norm=clip)
    half = 2.0 ** -8 if dt == "bf16" else 2.0 ** -24
    p64 = [p.detach().double() for p in params]
    m64 = [torch.zeros_like(p) for p in p64]
    v64 = [torch.zeros_like(p) for p in p64]
    mags = [torch.zeros_like(p) for p in p64]
    drift = [torch.zeros_like(p) for p in p64]  # how far a parameter may be off
    for t in range(1, 4):
        grads = tensors(SHAPES, dt, hip_device, seed=100 * t, std=0.1)
        for p, g in zip(params, grads):
            g[0] = 0
            p.grad = g
        opt.step()
        factor = 1.0
        if clip is not None:
            norm, factor = O.norm_and_factor(grads, clip)
            assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm
        for i, (p, g, (m, v)) in enumerate(zip(params, grads, opt.moments())):
            p64[i], m64[i], v64[i], change = O.step(p64[i], g, m64[i], v64[i], t, LR, BETAS, EPS, WD, factor)
            mags[i] = BETAS[0] * mags[i] + (1 - BETAS[0]) * g.double().abs() * factor
            assert ((m.double() - m64[i]).abs() <= 6 * t * 2.0 ** -24 * mags[i] + 1e-38).all(), (i, t)
            assert ((v.double() - v64[i]).abs() <= 8 * t * 2.0 ** -24 * v64[i] + 1e-38).all(), (i, t)
            size = torch.where(m64[i] != 0, change * mags[i] / m64[i].abs(), change)  # as m was added up from
            unit = 2.0 ** -24 * (6 * t * size + (4 * t + 8) * change)
            drift[i] = drift[i] + unit + 2 * 2.0 ** -24 * p64[i].abs() + half * (p64[i].abs() + drift[i])
            assert ((p.detach().double() - p64[i]).abs() <= drift[i] + 1e-38).all(), (i, t)
            assert p.dtype == DT[dt]


def _reference_8(p, g, m, v, t, factor):
    """As defined: moments formed in double from f32 values, rounded to f32, then the codes."""
    b1, b2 = BETAS
    gd = g.double().cpu() * factor
    m1 = (b1 * m.double() + (1 - b1) * gd).float()
    v1 = (b2 * v.double() + (1 - b2) * (gd * gd)).float()
    return m1, v1


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_8_bits(dt, clip, hip_device):
    """Codes and scales exactly, step after step; the parameters against the step from those moments."""
    shapes = [(1,), (5, 7), (256,), (255,), (257,), (4097,), (30, 41)]
    params = [p.requires_grad_(True) for p in tensors(shapes, dt, hip_device)]
    opt = optimizer(params, state_bits=8, max_grad_norm=clip)
    half = 2.0 ** -8 if dt == "bf16" else 2.0 ** -24
    m = [torch.zeros(s) for s in shapes]
    v = [torch.zeros(s) for s in shapes]
    for t in range(1, 5):
        grads = tensors(shapes, dt, hip_device, seed=100 * t, std=0.1)
        for p, g in zip(params, grads):
            g.view(-1)[::5] = 0
            p.grad = g
        before = [p.detach().double().cpu() for p in params]
        opt.step()
        factor = 1.0
        if clip is not None:
            norm = torch.tensor(O.norm_and_factor(grads, clip)[0]).float()
            factor = float((clip / (norm + torch.tensor(1e-6))).clamp(max=1.0))
        for i, (p, g) in enumerate(zip(params, grads)):
            m1, v1 = _reference_8(p, g, m[i], v[i], t, factor)
            st = opt.state[p]
            for name, x, second in (("exp_avg", m1, False), ("exp_avg_sq", v1, True)):
                codes, scales, values = O.through_codes(x, second)
                assert torch.equal(st[name].cpu().long(), codes), (i, t, name)
                assert torch.equal(st[name + "_scale"].cpu(), scales), (i, t, name)
                got = opt.moments()[i][int(second)]
                assert got.dtype == torch.float32 and torch.equal(got.cpu(), values), (i, t, name)
                if second:
                    v[i] = values
                else:
                    m[i] = values
            change = LR / (1 - BETAS[0] ** t) * m1.double() / (v1.double().sqrt() / math.sqrt(1 - BETAS[1] ** t) + EPS)
            want = before[i] * (1 - LR * WD) - change
            bound = half * want.abs() + 2.0 ** -24 * (12 * change.abs() + 2 * before[i].abs()) + 1e-38
            assert ((p.detach().double().cpu() - want).abs() <= bound).all(), (i, t)


def test_8_bits_of_every_size_of_moment(hip_device):
    """Blocks of subnormal, huge, equal and zero moments, of one element far above the others, and of half-way values."""
    rows = [torch.full((256,), 1e-3), torch.zeros(256), torch.randn(256, generator=gen(1)) * 1e-22,
            torch.randn(256, generator=gen(2)) * 1e18, torch.cat([torch.ones(1), torch.full((255,), 1e-12)]),
            2.0 ** -torch.arange(256.0).clamp(max=60), -torch.rand(256, generator=gen(3)), torch.cat([torch.ones(1), torch.full((255,), 0.25)]),
            torch.randn(256, generator=gen(4)) * 3e-39]
    g = torch.stack(rows).to(hip_device)
    p = torch.zeros_like(g).requires_grad_(True)
    opt = optimizer([p], state_bits=8)
    p.grad = g
    opt.step()
    m1, v1 = _reference_8(p, g, torch.zeros(g.shape), torch.zeros(g.shape), 1, 1.0)
    for name, x, second in (("exp_avg", m1, False), ("exp_avg_sq", v1, True)):
        codes, scales, values = O.through_codes(x, second)
        got = opt.state[p][name].cpu().long()
        assert torch.equal(got, codes), (name, (got != codes).any(1).nonzero())
        assert torch.equal(opt.state[p][name + "_scale"].cpu(), scales)
        assert torch.equal(opt.moments()[0][int(second)].cpu(), values)
    assert torch.isfinite(p).all() and (opt.state[p]["exp_avg_sq"][4] >= 1).all()


def test_8_bits_follow_32(hip_device):
    """Over many steps of a noisy quadratic the 8-bit moments stay near the 32-bit ones, and the grads that stop let them
    decay (a scale that could not shrink by 5% would hold them)."""
    target = torch.randn(3000, generator=gen(7)).to(hip_device)
    ps = [torch.zeros(3000, device=hip_device, requires_grad=True) for _ in range(2)]
    opts = [optimizer([p], state_bits=b, weight_decay=0.0) for p, b in zip(ps, (32, 8))]
    for t in range(60):
        noise = torch.randn(3000, generator=gen(t)).to(hip_device) * 0.1
        for p, o in zip(ps, opts):
            p.grad = (p.detach() - target) + noise
            o.step()
    (m32, v32), (m8, v8) = opts[0].moments()[0], opts[1].moments()[0]
    assert float((m8 - m32).norm() / m32.norm()) < 0.1 and float((v8 - v32).norm() / v32.norm()) < 0.1
    top = float(v8.max())
    for p in ps:
        p.grad = torch.zeros_like(p)
    for _ in range(40):
        opts[1].step()
    assert float(opts[1].moments()[0][1].max()) < top * 0.95 ** 40 * 1.01


def test_grads_that_are_not_finite(hip_device):
    """inf and NaN: 32 bits keep them in their element, 8 bits in their block of 256; the norm says so."""
    for bits in (32, 8):
        p = torch.zeros(1000, device=hip_device, requires_grad=True)
        opt = optimizer([p], state_bits=bits)
        g = torch.ones(1000, device=hip_device)
        g[300], g[900] = math.nan, math.inf
        p.grad = g
        opt.step()
        m, v = opt.moments()[0]
        bad = torch.zeros(1000, dtype=torch.bool, device=hip_device)
        if bits == 32:
            bad[300] = True
            assert torch.equal(torch.isnan(m), bad) and m[900] == math.inf and torch.isnan(p[300])
            bad[900] = True
        else:
            bad[256:512] = True
            bad[768:] = True
            assert torch.equal(torch.isnan(m), bad) and torch.equal(torch.isnan(v), bad)
        assert torch.isfinite(p.detach()[~bad]).all()
    p = torch.zeros(10, device=hip_device, requires_grad=True)
    opt = optimizer([p], max_grad_norm=1.0)
    p.grad = torch.full((10,), math.nan, device=hip_device)
    opt.step()
    assert torch.isnan(opt.grad_norm) and torch.isnan(p).all()


def test_many_tensors(hip_device):
    """More tensors than a launch's arguments hold, empty ones among them, and both types in one group."""
    shapes = [(i % 7 * 100,) for i in range(150)]
    params = [p.requires_grad_(True) for p in tensors(shapes, "f32", hip_device) + tensors(shapes, "bf16", hip_device)]
    alone = [p.detach().clone().requires_grad_(True) for p in params]
    opt, ones = optimizer(params, max_grad_norm=2.0), [optimizer([p]) for p in alone]
    for t in range(2):
        grads = tensors(shapes, "f32", hip_device, seed=t) + tensors(shapes, "bf16", hip_device, seed=t + 50)
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        for p, q, g in zip(params, alone, grads):
            p.grad = g
            # (a factor applied by hand: in f32, as the kernel multiplies)
            q.grad = g if g.dtype == torch.bfloat16 else g * torch.tensor(min(1.0, 2.0 / (norm + 1e-6)), device=hip_device)
        opt.step()
        for o in ones:
            o.step()
    assert abs(float(opt.grad_norm) - norm) <= 2.0 ** -23 * norm
    for p, q in zip(params[:150], alone[:150]):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-7)
    assert all(float(opt.state[p]["step"]) == 2.0 for p in params)


def test_a_tensor_alone_or_among_others(hip_device):
    """The same bits either way, whatever the tensor starts on."""
    for bits in (32, 8):
        for dt in ("f32", "bf16"):
            flat = tensors([(5000,)], dt, hip_device)[0]
            grads = tensors([(5000,)], dt, hip_device, seed=3)[0]
            params = [flat[a:b].detach().clone().requires_grad_(True) for a, b in ((0, 700), (701, 2000), (2003, 5000))]
            views = [flat[a:b].detach() for a, b in ((0, 700), (701, 2000), (2003, 5000))]
            for v in views:
                v.requires_grad_(True)
            one = optimizer(params, state_bits=bits)
            many = optimizer(views, state_bits=bits)
            for p, v, (a, b) in zip(params, views, ((0, 700), (701, 2000), (2003, 5000))):
                p.grad, v.grad = grads[a:b].clone(), grads[a:b]
            one.step()
            many.step()
            for p, v in zip(params, views):
                assert torch.equal(p, v)
            gaps = flat.detach()[[700, 2000, 2001, 2002]]
            assert torch.equal(gaps, tensors([(5000,)], dt, hip_device)[0][[700, 2000, 2001, 2002]])


def test_orders_in_memory(hip_device):
    """A transposed parameter, a grad of other strides than its parameter's, an expanded grad."""
    base = tensors([(40, 30)], "f32", hip_device)[0]
    p, q = base.t().detach().requires_grad_(True), base.t().contiguous().detach().requires_grad_(True)
    g = tensors([(30, 40)], "f32", hip_device, seed=9)[0]
    for bits in (32, 8):
        a, b = optimizer([p], state_bits=bits), optimizer([q], state_bits=bits)
        for grad in (g, g[:1].expand(30, 40)):
            p.grad, q.grad = grad, grad.contiguous()
            a.step()
            b.step()
        if bits == 32:
            assert torch.equal(p, q) and torch.equal(a.moments()[0][0], b.moments()[0][0])
    assert p.stride() == (1, 30) and a.state[p]["exp_avg"].stride() == (1, 30)


def test_groups_learning_rates_and_missing_grads(hip_device):
    a, b, c = (t.requires_grad_(True) for t in tensors([(50,), (60,), (70,)], "f32", hip_device))
    lr = torch.tensor(0.5, device=hip_device)
    opt = optimizer([{"params": [a], "lr": lr, "weight_decay": 0.0}, {"params": [b, c], "lr": torch.tensor(0.25), "state_bits": 8}])
    ref = [t.detach().clone() for t in (a, b, c)]
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.step()
    torch.testing.assert_close(a.detach(), ref[0] - 0.5)
    torch.testing.assert_close(b.detach(), ref[1] * (1 - 0.25 * WD) - 0.25)
    assert torch.equal(c, ref[2]) and not opt.state[c] and len(opt.moments()) == 3
    lr.fill_(0.0)
    before = a.detach().clone()
    opt.step()
    assert torch.equal(a, before)

    def closure():
        opt.zero_grad()
        loss = (a * a).sum()
        loss.backward()
        return loss

    assert float(opt.step(closure)) == float((before * before).sum())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_state_dict(bits, dt, hip_device, tmp_path):
    shapes = [(300,), (20, 30)]
    def run(opt, params, steps, start):
        for t in range(start, start + steps):
            for p, g in zip(params, tensors(shapes, dt, hip_device, seed=t)):
                p.grad = g
            opt.step()

    params = [p.requires_grad_(True) for p in tensors(shapes, dt, hip_device)]
    opt = optimizer(params, state_bits=bits)
    run(opt, params, 2, 0)
    torch.save({"o": opt.state_dict(), "p": [p.detach() for p in params]}, tmp_path / "s.pt")
    saved = torch.load(tmp_path / "s.pt", weights_only=True)
    others = [p.requires_grad_(True) for p in saved["p"]]
    two = optimizer(others, state_bits=bits)
    two.load_state_dict(saved["o"])
    run(opt, params, 2, 2)
    kept = copy.deepcopy(saved["o"]["state"])
    run(two, others, 2, 2)
    for p, q in zip(params, others):
        assert torch.equal(p, q)
        for name, t in opt.state[p].items():
            assert t.dtype == two.state[q][name].dtype and torch.equal(t, two.state[q][name])
    for i, st in kept.items():  # loading copied it
        assert all(torch.equal(t, saved["o"]["state"][i][n]) for n, t in st.items())


def test_torchs_state_loads(hip_device):
    p = tensors([(300,)], "f32", hip_device)[0].requires_grad_(True)
    q = p.detach().clone().requires_grad_(True)
    theirs = torch.optim.AdamW([p], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD)
    ours = optimizer([q])
    for t in range(2):
        p.grad = tensors([(300,)], "f32", hip_device, seed=t)[0]
        theirs.step()
    with torch.no_grad():
        q.copy_(p)
    ours.load_state_dict(theirs.state_dict())
    p.grad = q.grad = tensors([(300,)], "f32", hip_device, seed=8)[0]
    theirs.step()
    ours.step()
    torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-6)
    eight = optimizer([q.detach().clone().requires_grad_(True)], state_bits=8)
    q8 = eight.param_groups[0]["params"][0]
    q8.grad = torch.ones_like(q8)
    eight.step()
    with pytest.raises(ValueError):
        ours.load_state_dict({**ours.state_dict(), "state": eight.state_dict()["state"]})


def test_captured(hip_device):
    """Steps captured into two graphs and replayed in turn with new grads and rates count on like eager ones."""
    for bits in (32, 8):
        sets = []
        for s in range(2):
            params = [p.requires_grad_(True) for p in tensors([(700,), (40, 50)], "f32", hip_device, seed=s)]
            lr = torch.tensor(LR, device=hip_device)
            opt = optimizer(params, state_bits=bits, lr=lr, max_grad_norm=1.0)
            twin = [p.detach().clone().requires_grad_(True) for p in params]
            lr2 = torch.tensor(LR, device=hip_device)
            eager = optimizer(twin, state_bits=bits, lr=lr2, max_grad_norm=1.0)
            for p, q in zip(params, twin):
                p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
            with pytest.raises(RuntimeError):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    opt.step()
            side = torch.cuda.Stream(hip_device)
            side.wait_stream(torch.cuda.current_stream(hip_device))
            with torch.cuda.stream(side):
                opt.step()
                eager.step()
            torch.cuda.current_stream(hip_device).wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                opt.step()
                norm = opt.grad_norm
            sets.append((g, params, opt, lr, twin, eager, lr2, norm))
        for t in range(3):
            for s, (g, params, opt, lr, twin, eager, lr2, norm) in enumerate(sets):
                for p, q, new in zip(params, twin, tensors([(700,), (40, 50)], "f32", hip_device, seed=10 * t + s)):
                    p.grad.copy_(new)
                    q.grad.copy_(new)
                lr.fill_(LR / (t + 1))
                lr2.fill_(LR / (t + 1))
            for s in sets:
                s[0].replay()
            torch.cuda.synchronize()
            for g, params, opt, lr, twin, eager, lr2, norm in sets:
                eager.step()
                assert torch.equal(norm, eager.grad_norm)
                for p, q in zip(params, twin):
                    assert torch.equal(p, q)
                    assert all(torch.equal(a, eager.state[q][n]) for n, a in opt.state[p].items())


def test_autograd_sees_the_change(hip_device):
    p = torch.ones(5, device=hip_device, requires_grad=True)
    opt = optimizer([p])
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(hip_device):
    from zmoe.adamw import AdamW

    p = torch.zeros(4, 6, device=hip_device, requires_grad=True)
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-1.0),
               dict(state_bits=16), dict(max_grad_norm=0.0), dict(max_grad_norm=-1.0),
               dict(lr=torch.zeros(2)), dict(lr=torch.zeros((), device=hip_device, dtype=torch.float64))):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    for bad in (torch.zeros(3, device=hip_device, dtype=torch.float16), torch.zeros(4, 6, device=hip_device)[:, :3],
                torch.zeros(1, 6, device=hip_device).expand(4, 6)):
        with pytest.raises(ValueError):
            AdamW([bad.requires_grad_(True)])
    opt = AdamW([p])
    p.grad = torch.zeros(4, 6, device=hip_device).to_sparse()
    with pytest.raises(RuntimeError):
        opt.step()
    cpu = torch.zeros(3, requires_grad=True)
    cpu.grad = torch.zeros(3)
    with pytest.raises(ValueError):
        AdamW([cpu]).step()


def test_parameters_and_groups_that_changed(hip_device):
    """What no longer fits the state is refused; a copy goes on as its original."""
    import copy

    from zmoe.adamw import AdamW

    def made(bits):
        p = torch.randn(40, 30, generator=gen(11)).to(hip_device).requires_grad_(True)
        opt = AdamW([p], state_bits=bits, max_grad_norm=0.5)
        p.grad = torch.randn(40, 30, generator=gen(12)).to(hip_device)
        opt.step()
        return p, opt

    p, opt = made(8)
    q, twin = made(8)
    other = copy.deepcopy(twin)
    opt.step()
    other.param_groups[0]["params"][0].grad = p.grad
    other.step()
    assert torch.equal(p, other.param_groups[0]["params"][0])
    p.data = p.data.t().contiguous().t()
    with pytest.raises(RuntimeError, match="order in memory"):
        opt.step()
    for bits in (8, 32):
        p, opt = made(bits)
        before = p.detach().clone()
        opt.param_groups[0]["state_bits"] = 40 - bits
        with pytest.raises(ValueError):
            opt.step()
        assert torch.equal(p, before)


@pytest.mark.parametrize("bits", [32, 8])
def test_called_from_a_compiled_function(bits, hip_device):
    from zmoe.adamw import AdamW

    x = torch.randn(8, 32, generator=gen(21)).to(hip_device)
    grads = [torch.randn(16, 32, generator=gen(22 + i)).to(hip_device) for i in range(3)]
    ps = [torch.randn(16, 32, generator=gen(20)).to(hip_device).requires_grad_(True) for _ in range(2)]
    opts = [AdamW([p], state_bits=bits, max_grad_norm=1.0) for p in ps]

    def step(p, opt, g):
        y = (x @ g.t()).relu()  # something to compile around it
        p.grad = g * 2.0
        opt.step()
        return y.sum()

    compiled = torch.compile(step)
    for g in grads:
        step(ps[0], opts[0], g)
        compiled(ps[1], opts[1], g)
        assert torch.equal(ps[0], ps[1])
    torch.compile(opts[1].step)()
    opts[0].step()
    assert torch.equal(ps[0], ps[1])
