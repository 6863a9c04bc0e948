"""The router's forms, its losses and AdamW as a training loop uses them together: MoELayer with a softmax or grouped router,
the losses of its router, a backward pass, a step; eager, unpadded, under autocast, captured and compiled. What has no other
reference is compared between the layer's one-function path and its composition of modules, whose ops are tested alone."""

import math

import pytest
import torch

from helpers import gen
from oracle import router_oracle as O

pytestmark = pytest.mark.gpu

FORMS = [dict(), dict(router_score="softmax", router_bias=False), dict(router_groups=4, router_top_groups=2, router_scale=2.5),
         dict(router_score="softmax", router_renormalize=False, router_scale=4.0, router_groups=4, router_top_groups=3,
              router_group_scores=1)]
D, F, E, K = 128, 64, 16, 4


def layer_of(form, dev, dtype=torch.bfloat16, seed=0):
    from modeling.model_config import ModelConfig
    from modeling.moe_layer import MoELayer

    torch.manual_seed(seed)
    layer = MoELayer(ModelConfig(hidden_size=D, intermediate_size=F, n_experts=E + 1, n_shared_experts=1,
                                 n_experts_per_token=K, **form)).to(dev).to(dtype)
    layer.gate.expert_biases.data = (torch.randn(E, generator=gen(seed)) * 0.05).to(dev)
    return layer


def tokens(dev, b=2, s=90, seed=0, dtype=torch.bfloat16):
    return torch.randn(b, s, D, generator=gen(seed)).to(dtype).to(dev)


@pytest.mark.parametrize("form", FORMS)
def test_gate_routes_by_its_form(form, hip_device):
    layer = layer_of(form, hip_device)
    x = tokens(hip_device)
    idx, w, logits = layer.gate(x, return_logits=True)
    if not form:  # the reference's form stores p in bf16
        assert layer.gate.form is None
        return
    f = layer.gate.form
    want = O.select(logits, K, layer.gate.expert_biases if f.bias else None, layer.gate.score, f.groups, f.top_groups,
                    f.group_scores)
    assert torch.equal(idx.view(-1, K), want)
    val = O.weights(logits, want, layer.gate.score, f.renormalize, f.scale)
    assert ((w.view(-1, K).double() - val).abs() <= (K + 4) * 2.0 ** -24 * val + 1e-38).all()


def grads_of(layer, x, dout, losses, **kw):
    for p in layer.parameters():
        p.grad = None
    x = x.clone().requires_grad_(True)
    out, idx, *more = layer(x, router_losses=losses, **kw)
    total = [out]
    seeds = [dout]
    if losses:
        total += list(more[0])
        seeds += [torch.tensor(0.5, device=x.device), torch.tensor(0.05, device=x.device)]
    torch.autograd.backward(total, seeds)
    return out.detach(), idx, more, {"x": x.grad, **{n: p.grad for n, p in layer.named_parameters()}}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("losses", [False, True])
def test_one_function_is_the_composition(form, losses, hip_device):
    """Outputs alike, choices and losses equal; grads within bf16's roundings of their sums (2^-7 of the tensor's norm: the
    two differ in where products are rounded to bf16, half a step 2^-9 each, of which a handful follow each other)."""
    layer = layer_of(form, hip_device)
    x = tokens(hip_device)
    dout = tokens(hip_device, seed=9)
    fused = grads_of(layer, x, dout, losses)
    layer.fused_layer = False
    plain = grads_of(layer, x, dout, losses)
    assert torch.equal(fused[1], plain[1])
    if losses:
        assert all(torch.equal(a, b) for a, b in zip(fused[2][0], plain[2][0]))
    for name in fused[3]:
        a, b = fused[3][name].double(), plain[3][name].double()
        assert float((a - b).norm()) <= 2.0 ** -6 * float(b.norm()), name
    # the losses reach the router, and without them its grad is another
    if losses:
        layer.fused_layer = True
        without = grads_of(layer, x, dout, False)
        d = fused[3]["gate.weight"].double() - without[3]["gate.weight"].double()
        assert float(d.norm()) > 0 and torch.equal(fused[3]["routed_experts.experts.weight"],
                                                   without[3]["routed_experts.experts.weight"])


@pytest.mark.parametrize("form", FORMS)
def test_losses_alone(form, hip_device):
    """A backward pass from the losses alone: the gate's weight grad is d_logits^T x, the experts' zero."""
    layer = layer_of(form, hip_device)
    x = tokens(hip_device)
    out, idx, (balance, z) = layer(x, router_losses=True)
    (0.5 * balance + 0.05 * z).backward()
    _, _, logits = layer.gate(x, return_logits=True)
    cu = torch.tensor([0, 90, 180])
    vb, vz, _, _ = O.losses(logits, idx.view(-1, K), layer.gate.score, cu)
    assert abs(float(balance) - float(vb)) <= 2e-5 * float(vb) and abs(float(z) - float(vz)) <= 2e-5 * float(vz)
    val, _ = O.losses_backward(logits, idx.view(-1, K), layer.gate.score, cu, 0.5, 0.05)
    want = val.T @ x.view(-1, D).double()
    got = layer.gate.weight.grad.double()
    # d_logits is rounded to bf16 once (2^-9 of each), the grad once more
    assert float((got - want).norm()) <= 2.0 ** -7 * float(want.norm())
    assert not layer.routed_experts.experts.weight.grad.any()


def test_sequences_of_unpadded_tokens(hip_device):
    layer = layer_of(FORMS[1], hip_device)
    x = tokens(hip_device, 3, 50)
    keep = torch.cat([torch.arange(0, 20), torch.arange(50, 100), torch.arange(100, 111)]).to(hip_device)
    cu = torch.tensor([0, 20, 70, 81], dtype=torch.int32, device=hip_device)
    out, idx, (balance, z) = layer(x, unpad_indices=keep, router_losses=True, cu_seqlens=cu)
    assert out.shape == x.shape and idx.shape == (3, 50, K)
    flat = x.view(-1, D)[keep]
    _, _, logits = layer.gate(flat.unsqueeze(0), return_logits=True)
    vb, vz, _, _ = O.losses(logits, idx.view(-1, K)[keep], "softmax", cu)
    assert abs(float(balance) - float(vb)) <= 2e-5 * float(vb) and abs(float(z) - float(vz)) <= 2e-5 * float(vz)
    layer.fused_layer = False
    _, _, again = layer(x, unpad_indices=keep, router_losses=True, cu_seqlens=cu)
    assert torch.equal(again[0], balance) and torch.equal(again[1], z)
    one = layer(x, unpad_indices=keep, router_losses=True)[2]  # all tokens one sequence
    vb, _, _, _ = O.losses(logits, idx.view(-1, K)[keep], "softmax")
    assert abs(float(one[0]) - float(vb)) <= 2e-5 * float(vb)


def test_served_in_e4m3(hip_device):
    layer = layer_of(FORMS[3], hip_device)
    served = layer.quantize_fp8()
    x = tokens(hip_device)
    with torch.no_grad():
        a, ia = layer(x)
        b, ib = served(x)
    assert torch.equal(ia, ib) and float((a.double() - b.double()).norm()) <= 0.1 * float(a.double().norm())


def loop(layer, opt, xs, step):
    x = xs[step % len(xs)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out, idx, (balance, z) = layer(x, router_losses=True)
    loss = (out.float() - x).square().mean() + 0.01 * balance + 0.001 * z
    opt.zero_grad(set_to_none=False)
    loss.backward()
    opt.step()
    return loss.detach(), idx


@pytest.mark.parametrize("bits", [32, 8])
def test_training_step_under_autocast(bits, hip_device):
    """fp32 master weights under bf16 autocast: the loop runs, every parameter moves and stays finite, and a captured step
    replayed on new tokens is the eager one, bit for bit."""
    from zmoe.adamw import AdamW

    xs = [tokens(hip_device, seed=i, dtype=torch.float32) for i in range(3)]
    runs = []
    for captured in (False, True):
        layer = layer_of(FORMS[3], hip_device, torch.float32)
        opt = AdamW(layer.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=1.0)
        before = [p.detach().clone() for p in layer.parameters()]
        static = xs[0].clone()
        side = torch.cuda.Stream(hip_device)
        side.wait_stream(torch.cuda.current_stream(hip_device))
        with torch.cuda.stream(side):
            for _ in range(2):
                loop(layer, opt, [static], 0)
        torch.cuda.current_stream(hip_device).wait_stream(side)
        seen = []
        if captured:
            for p in layer.parameters():
                assert p.grad is not None
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                loss, idx = loop(layer, opt, [static], 0)
        for t in range(1, 4):
            static.copy_(xs[t % 3])
            if captured:
                graph.replay()
            else:
                loss, idx = loop(layer, opt, [static], 0)
            torch.cuda.synchronize()
            seen.append((loss.clone(), idx.clone(), opt.grad_norm.clone()))
        after = [p.detach().clone() for p in layer.parameters()]
        assert all(torch.isfinite(p).all() and not torch.equal(p, q) for p, q in zip(after, before))
        runs.append((seen, after, [m for pair in opt.moments() for m in pair]))
    (sa, pa, ma), (sb, pb, mb) = runs
    for a, b in zip(sa, sb):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(x, y) for x, y in zip(pa + ma, pb + mb))


@pytest.mark.parametrize("form", [FORMS[1], FORMS[3]])
def test_compiled(form, hip_device):
    layer = layer_of(form, hip_device)
    x = tokens(hip_device)

    def f(x):
        out, idx, (balance, z) = layer(x, router_losses=True)
        return out, idx, 0.5 * balance + 0.05 * z

    a, ia, la = f(x)
    b, ib, lb = torch.compile(f, dynamic=True, fullgraph=True)(x)
    assert torch.equal(ia, ib) and torch.equal(a, b)
    torch.testing.assert_close(la, lb)


def test_config_refusals():
    from modeling.model_config import ModelConfig

    base = dict(hidden_size=D, intermediate_size=F, n_experts=E + 1, n_shared_experts=1, n_experts_per_token=K)
    for bad in (dict(router_score="relu"), dict(router_groups=3), dict(router_groups=0), dict(router_groups=4, router_top_groups=5),
                dict(router_groups=8, router_top_groups=1), dict(router_group_scores=3),
                dict(router_groups=16, router_top_groups=8)):
        with pytest.raises(ValueError):
            ModelConfig(**{**base, **bad})
