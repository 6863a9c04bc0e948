"""norm_residual on the GPU against float64 (oracle.norm_residual_oracle).

Tolerance: the kernel works in float32. A row sum is at most 32 additions in a thread, 6 in a wave and 16 over waves, so
it and what is formed from it (a few products, one rsqrt) is off by less than 128 * 2^-24 of the magnitudes it is added
up from; a gradient goes through two of them and twice the sums: 512 * 2^-24. Sums over n rows add n more.
Rounding to the output's type adds half a step, 2^-8 (bf16) or 2^-24 (f32) of the value.
"""

import pytest
import torch

from helpers import gen
from oracle import norm_residual_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def make(n, d, rt, yt, gate, post, nxt, scale, dev, seed=1, wt="bf16"):
    g = gen(seed + 7 * n + d)
    rnd = lambda *s, std=1.0, t="f32": (torch.randn(*s, generator=g) * std).to(DT[t]).to(dev)  # noqa: E731
    shape = {"none": None, "channel": (d,), "row": (n, 1), "full": (n, d)}[gate]
    return {"r": rnd(n, d, std=2.0, t=rt), "y": rnd(n, d, t=yt), "w_post": rnd(d, std=0.2, t=wt) if post else None,
            "w_next": rnd(d, std=0.2, t=wt) if nxt else None, "gate": None if shape is None else rnd(*shape, t=wt),
            "scale": rnd(1, std=0.1) + 0.9 if scale else None, "dr": rnd(n, d, t=rt),
            "dx": rnd(n, d, t=yt) if nxt else None}


def close(name, got, val, mag, units):
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    assert got.shape == val.shape, (name, got.shape, val.shape)
    bound = half * val.abs() + units * 2.0 ** -24 * mag
    bad = ~((got.double() - val).abs() <= bound)
    assert not bad.any(), (name, int(bad.sum()), float(((got.double() - val).abs() / bound.clamp(min=1e-300)).max()))


def run(t, use_dr=True, use_dx=True):
    from zmoe.functional import norm_residual

    leaves = {n: v.detach().clone().requires_grad_(True) for n, v in t.items() if v is not None and n not in ("dr", "dx")}
    r, x = norm_residual(leaves["r"], leaves["y"], leaves.get("w_post"), leaves.get("w_next"), leaves.get("gate"),
                         leaves.get("scale"), EPS)
    outs, grads = [], []
    if use_dr:
        outs, grads = [r], [t["dr"]]
    if x is not None and use_dx:
        outs.append(x)
        grads.append(t["dx"])
    torch.autograd.backward(outs, grads)
    return r.detach(), None if x is None else x.detach(), {n: v.grad for n, v in leaves.items()}


def check(t, use_dr=True, use_dx=True):
    n = t["y"].shape[0]
    scale = 1.0 if t["scale"] is None else float(t["scale"])
    args = (t["r"], t["y"], t["w_post"], t["w_next"], t["gate"], scale, EPS)
    r, x, grads = run(t, use_dr, use_dx)
    val, mag, _ = O.forward(*args)
    close("r out", r, val["r"], mag["r"], 128)
    assert r.dtype == t["r"].dtype
    if x is not None:
        close("x", x, val["x"], mag["x"], 256)
        assert x.dtype == t["y"].dtype
    val, mag = O.backward(*args, t["dr"] if use_dr else None, t["dx"] if use_dx else None)
    for name, g in grads.items():
        rows = name in ("w_post", "w_next", "scale") or (name == "gate" and t["gate"].dim() == 1)
        close("d " + name, g, val[name].reshape(g.shape), mag[name].reshape(g.shape), 512 + (n if rows else 0))
        assert g.dtype == t[name].dtype


@pytest.mark.parametrize("rt,yt", [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("n,d", [(1, 8), (3, 1), (5, 510), (9, 512), (130, 1024), (33, 2048), (7, 4096), (5, 7168),
                                 (3, 8190), (2, 16384), (2, 30000)])
def test_types_and_widths(n, d, rt, yt, hip_device):
    check(make(n, d, rt, yt, "channel", True, True, True, hip_device))


@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("post,nxt", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("d", [96, 2048])
def test_forms(gate, post, nxt, scale, d, hip_device):
    check(make(37, d, "f32", "bf16", gate, post, nxt, scale, hip_device, wt="f32" if scale else "bf16"))


def test_many_rows(hip_device):
    """More rows than the backward's grid has blocks, at every number of rows per block."""
    for n, d in ((2600, 512), (1200, 1000), (1030, 2048), (1025, 4096), (520, 8192)):
        check(make(n, d, "bf16", "bf16", "channel", True, True, True, hip_device))


def test_one_output_unused(hip_device):
    for use_dr, use_dx in ((True, False), (False, True)):
        for gate in ("row", "full", "none"):
            check(make(12, 2048, "f32", "bf16", gate, True, True, True, hip_device), use_dr, use_dx)
            check(make(12, 300, "bf16", "bf16", gate, gate != "row", True, True, hip_device), use_dr, use_dx)


def test_no_rows(hip_device):
    t = make(0, 64, "bf16", "bf16", "channel", True, True, True, hip_device)
    r, x, g = run(t)
    assert r.shape == x.shape == (0, 64) and not g["w_post"].any() and not g["scale"].any() and not g["gate"].any()


def test_strides_and_broadcasts(hip_device):
    """Row strides, starts off 16 bytes, expanded rows, leading dims, a gate that broadcasts, mixed weight types."""
    from zmoe.functional import norm_residual

    d = 200
    big = torch.randn(30, 500, generator=gen(1)).to(torch.bfloat16).to(hip_device)
    w1, w2 = (torch.randn(d, generator=gen(s)).mul_(0.2).to(hip_device) for s in (2, 3))
    for r, y in ((big[:, 3:3 + d], big[:, 256:256 + d]), (big[::2, :d], big[1::2, 300:]), (big[:1, :d].expand(30, d), big[:, :d])):
        got = norm_residual(r, y, w1, w2.bfloat16(), None, 0.5, EPS)
        ref = norm_residual(r.contiguous(), y.contiguous(), w1, w2.bfloat16().float(), None, 0.5, EPS)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    r, y = big[:24, :d].reshape(2, 3, 4, d), big[:24, 200:400].reshape(2, 3, 4, d)
    per_seq = torch.randn(2, 1, 1, d, generator=gen(5)).to(hip_device).requires_grad_(True)
    got, _ = norm_residual(r, y, w1, None, per_seq, None, EPS)
    full = per_seq.detach().expand(2, 3, 4, d).contiguous().requires_grad_(True)
    ref, _ = norm_residual(r, y, w1, None, full, None, EPS)
    assert got.shape == r.shape and torch.equal(got, ref)
    go = torch.randn(2, 3, 4, d, generator=gen(6)).to(torch.bfloat16).to(hip_device)
    got.backward(go)
    ref.backward(go)
    torch.testing.assert_close(per_seq.grad, full.grad.sum((1, 2), keepdim=True))


def test_expanded_output_grad(hip_device):
    t = make(6, 96, "bf16", "bf16", "none", True, True, False, hip_device)
    leaves = [t[k].requires_grad_(True) for k in ("r", "y")]
    from zmoe.functional import norm_residual

    r, x = norm_residual(*leaves, t["w_post"], t["w_next"], None, None, EPS)
    got = torch.autograd.grad([r, x], leaves, [torch.ones_like(r), torch.ones((), device=hip_device, dtype=x.dtype).expand(x.shape)])
    r, x = norm_residual(*leaves, t["w_post"], t["w_next"], None, None, EPS)
    ref = torch.autograd.grad((r.float() + x.float()).sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_masked_rows(hip_device):
    """Rows of zeros give zeros and finite grads; a row with inf or NaN stays in its own row."""
    t = make(9, 512, "bf16", "bf16", "none", True, True, False, hip_device)
    t["y"][2] = 0
    t["r"][2] = 0
    r, x, g = run(t)
    assert not r[2].any() and not x[2].any()
    for v in g.values():
        assert torch.isfinite(v).all()
    clean = run(t)
    t["y"][5, 3], t["y"][6, 4] = float("inf"), float("nan")
    r, x, g = run(t)
    ok = [i for i in range(9) if i not in (5, 6)]
    assert torch.equal(r[ok], clean[0][ok]) and torch.equal(x[ok], clean[1][ok])
    assert torch.equal(g["r"][ok], clean[2]["r"][ok]) and torch.isnan(x[6]).all()


def test_module_and_layer(hip_device):
    """Between two sublayers, as a block uses it: MoELayer's output, the residual and the next norm."""
    from modeling.model_config import ModelConfig
    from modeling.moe_layer import MoELayer
    from modeling.zRMSNorm import NormResidual, ZeroCenteredRMSNorm

    torch.manual_seed(0)
    d = 64
    layer = MoELayer(ModelConfig(hidden_size=d, intermediate_size=32, n_experts=9, n_shared_experts=1,
                                 n_experts_per_token=2)).to(hip_device).bfloat16()
    layer.gate.expert_biases.data = layer.gate.expert_biases.data.float()
    step, pre, nxt = NormResidual(d, gate=True, residual_scale=0.8), ZeroCenteredRMSNorm(d), ZeroCenteredRMSNorm(d)
    for m in (step, pre, nxt):
        m.to(hip_device)
        m.weight.data.normal_(0, 0.2)
    h = torch.randn(2, 12, d, device=hip_device, dtype=torch.bfloat16, requires_grad=True)
    y, _ = layer(h, norm=pre)
    r, x = step(h, y, nxt)
    val, mag, _ = O.forward(h.view(-1, d), y.view(-1, d), step.weight, nxt.weight, step.gate, 0.8, 1e-6)
    close("r", r.view(-1, d), val["r"], mag["r"], 128)
    close("x", x.view(-1, d), val["x"], mag["x"], 256)
    (r.float().sum() + x.float().square().sum()).backward()
    for p in (*step.parameters(), nxt.weight, pre.weight, *layer.parameters()):
        assert p.grad is not None and torch.isfinite(p.grad).all()


def test_captured(hip_device):
    """A training step captured into a graph, replayed with new inputs, against the eager step."""
    t = make(70, 1024, "bf16", "bf16", "channel", True, True, True, hip_device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(t)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(t)
    for seed in (5, 6, 7):
        new = make(70, 1024, "bf16", "bf16", "channel", True, True, True, hip_device, seed=seed)
        for k, v in new.items():
            t[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        ref = run(new)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        for k, v in ref[2].items():
            assert torch.equal(got[2][k], v), k


def test_refusals(hip_device):
    from zmoe.functional import norm_residual

    r = torch.zeros(4, 32, device=hip_device, dtype=torch.bfloat16)
    w = torch.zeros(32, device=hip_device)
    for args, kw in (((r, r[:2]), dict(weight=w)), ((r, r), {}), ((r, r), dict(weight=w[:16])),
                     ((r.half(), r.half()), dict(weight=w)), ((r, r), dict(weight=w, residual_scale=torch.zeros(2, device=hip_device))),
                     ((r.cpu(), r.cpu()), dict(weight=w))):
        with pytest.raises(ValueError):
            norm_residual(*args, **kw)
    with pytest.raises(RuntimeError):
        norm_residual(r, r, w, gate=torch.zeros(3, 32, device=hip_device))
