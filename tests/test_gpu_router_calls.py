"""MoELayer with its router's losses in the calls between the usual ones: compiled and timed passes, no tokens, the losses
alone, a frozen router, other streams; AdamW's states loaded under inference mode."""

import pytest
import torch

from helpers import gen
from test_gpu_router_training import FORMS, K, grads_of, layer_of, tokens

pytestmark = pytest.mark.gpu


def passed(layer, x, dout, f=None):
    for p in layer.parameters():
        p.grad = None
    x = x.clone().requires_grad_(True)
    out, idx, (balance, z) = (layer if f is None else f)(x, router_losses=True)
    torch.autograd.backward([out, 0.5 * balance + 0.05 * z], [dout, torch.ones((), device=x.device)])
    return [out.detach(), idx, balance.detach(), z.detach(), x.grad] + [p.grad for p in layer.parameters()]


@pytest.mark.parametrize("form", FORMS)
def test_watched_passes(form, hip_device):
    """A pass that zmoe.profiling times (the ops' general forms) is the usual one, bit for bit."""
    from zmoe import profiling

    layer, x, dout = layer_of(form, hip_device), tokens(hip_device), tokens(hip_device, seed=9)
    want = passed(layer, x, dout)
    profiling.enable("route_backward", "router_losses")
    try:
        got = passed(layer, x, dout)
        assert len(profiling.durations_ms("route_backward")) == 1 and len(profiling.durations_ms("router_losses")) == 1
    finally:
        profiling.disable()
        profiling.reset()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("form", FORMS)
def test_compiled_training(form, hip_device):
    """The compiled pass' grads: the layer is one node, the losses' sum compiled around it may round once more (d_logits in
    bf16, 2^-9 of a part of the grads)."""
    layer, x, dout = layer_of(form, hip_device), tokens(hip_device), tokens(hip_device, seed=9)
    want = passed(layer, x, dout)
    got = passed(layer, x, dout, torch.compile(layer, dynamic=False))
    assert all(torch.equal(a, b) for a, b in zip(want[:2], got[:2]))
    for a, b in zip(want[2:], got[2:]):
        assert float((a.double() - b.double()).norm()) <= 2.0 ** -8 * float(a.double().norm())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("shape", [(0, 5), (2, 0), (1, 1), (1, 3)])
def test_few_tokens_and_none(shape, fused, form, hip_device):
    layer = layer_of(form, hip_device)
    layer.fused_layer = fused
    x = tokens(hip_device, *shape)
    out, idx, balance, z, gx, *grads = passed(layer, x, torch.ones_like(x))
    assert out.shape == gx.shape == x.shape and idx.shape == (*shape, K)
    assert all(g is not None and torch.isfinite(g).all() for g in grads)
    if x.numel() == 0:
        assert float(balance) == float(z) == 0.0 and not any(g.any() for g in grads)


@pytest.mark.parametrize("form", FORMS)
def test_frozen_parts(form, hip_device):
    """Without grads of the router's weight, or of the input: the others' are the usual ones."""
    layer, x, dout = layer_of(form, hip_device), tokens(hip_device), tokens(hip_device, seed=9)
    want = grads_of(layer, x, dout, True)[3]
    layer.gate.weight.requires_grad_(False)
    got = grads_of(layer, x, dout, True)[3]
    assert got["gate.weight"] is None
    assert all(torch.equal(g, want[n]) for n, g in got.items() if g is not None) and len(got) == len(want)
    layer.gate.weight.requires_grad_(True)
    for p in layer.parameters():
        p.grad = None
    out, _, (balance, z) = layer(x, router_losses=True)
    torch.autograd.backward([out, balance, z], [dout, torch.tensor(0.5, device=x.device), torch.tensor(0.05, device=x.device)])
    assert all(torch.equal(p.grad, want[n]) for n, p in layer.named_parameters())


@pytest.mark.parametrize("form", FORMS)
def test_without_a_graph(form, hip_device):
    layer, x = layer_of(form, hip_device), tokens(hip_device)
    out, idx, (balance, z) = layer(x, router_losses=True)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            o, i, (b, zz) = layer(x, router_losses=True)
        assert torch.equal(o, out) and torch.equal(i, idx) and torch.equal(b, balance) and torch.equal(zz, z)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_two_threads_at_once(score, hip_device):
    """Calls of two threads on streams of their own, each with scratch of its own."""
    import threading

    from zmoe.functional import route, router_losses

    zs = [(torch.randn(3000, 160, generator=gen(40 + i))).to(hip_device) for i in range(2)]
    cu = torch.tensor([0, 700, 701, 2999], device=hip_device)

    def once(z):
        leaf = z.clone().requires_grad_(True)
        idx, w = route(leaf, 6, None, score, 8, 3, 1, False, 2.0)
        balance, zl = router_losses(leaf, idx, score, cu)
        (w.square().sum() + balance + zl).backward()
        return idx, w.detach(), balance.detach(), zl.detach(), leaf.grad

    want = [once(z) for z in zs]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        stream = torch.cuda.Stream(hip_device)
        with torch.cuda.stream(stream):
            for _ in range(10):
                got[i].append(once(zs[i]))
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for w, runs in zip(want, got):
        assert len(runs) == 10 and all(torch.equal(a, b) for run in runs for a, b in zip(w, run))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_loaded_under_inference_mode(bits, hip_device):
    from zmoe.adamw import AdamW

    ps = [torch.ones(600, device=hip_device, requires_grad=True) for _ in range(2)]
    a, b = (AdamW([p], state_bits=bits) for p in ps)
    for p in ps:
        p.grad = torch.randn(600, generator=gen(1)).to(hip_device)
    a.step()
    with torch.no_grad():
        ps[1].copy_(ps[0])
    with torch.inference_mode():
        b.load_state_dict(a.state_dict())
    a.step()
    b.step()
    assert torch.equal(ps[0], ps[1])
    assert all(torch.equal(t, b.state[ps[1]][n]) and not b.state[ps[1]][n].is_inference() for n, t in a.state[ps[0]].items())
