"""Calls of the e4m3 entry points that their documentation allows beyond the shapes of test_gpu_fp8_layers: float32 rows,
no rows, any number of slots, routing in views, copies of modules, a backward twice, recomputation."""

import copy
import io

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from helpers import gen, random_topk
from oracle import fp8_oracle as O
from test_gpu_fp8 import activations, check
from test_gpu_fp8_layers import wgrad_close, weight

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("wt", [BF, F32])
@pytest.mark.parametrize("T,K,N,E,k", [(30, 130, 200, 5, 1), (90, 256, 130, 4, 3)])
def test_parallel_linear_float32_rows(T, K, N, E, k, wt, hip_device):
    from scattermoe.parallel_experts import flatten_sort_count, parallel_linear

    idx = random_topk(T, E, k, T).to(hip_device)
    se, ss, off = flatten_sort_count(idx, E)
    x = activations(T, K, F32, 1, hip_device).requires_grad_(True)
    W = weight((E, N, K), 2, wt, hip_device).requires_grad_(True)
    dy = activations(T * k, N, F32, 3, hip_device)
    y = parallel_linear(x, W.permute(0, 2, 1), k, se, ss, off, grouped_out=True, fp8=True)
    y.backward(dy)
    assert y.dtype == x.grad.dtype == F32 and W.grad.dtype == wt
    wr = O.quantize_weight(W.detach())[0]
    check(y.detach(), *O.grouped_product(O.quantize_rows(x.detach())[0], wr, ss, off, k, False, True), K)
    v, S, G = O.grouped_product(O.quantize_rows(dy)[0], wr.transpose(1, 2), ss, off, 1, True, False)
    fold = lambda t: t.view(T, k, K).sum(1)  # noqa: E731
    # each slot's sum and its rounding to f32, then k additions
    b = fold(7 * 2.0 ** -13 * G + (17 * -(-N // 128) * 2.0 ** -23 + (k + 2) * 2.0 ** -24) * S)
    assert ((x.grad.double() - fold(v)).abs() <= 1.01 * b).all()
    beg = 0
    for e, end in enumerate(off.tolist()):
        wgrad_close(W.grad[e], dy[beg:end], x.detach()[ss[beg:end] // k])
        beg = end


def test_no_rows(hip_device):
    from modeling.model_config import ModelConfig
    from modeling.moe_layer import MoELayer
    from scattermoe.mlp import GLUMLP
    from scattermoe.parallel_experts import flatten_sort_count, parallel_linear

    d, f, E, k = 64, 32, 4, 2
    none = dict(device=hip_device, dtype=BF)
    idx, p = torch.zeros(0, k, dtype=torch.int64, device=hip_device), torch.zeros(0, k, device=hip_device)
    se, ss, off = flatten_sort_count(idx, E)
    x, W = torch.zeros(0, d, **none).requires_grad_(True), weight((E, f, d), 1, BF, hip_device).requires_grad_(True)
    y = parallel_linear(x, W.permute(0, 2, 1), k, se, ss, off, grouped_out=True, fp8=True)
    assert y.shape == (0, f)
    y.sum().backward()
    assert x.grad.shape == (0, d) and not W.grad.any()
    m = GLUMLP(d, f, E, k, fp8=True).to(hip_device)
    with torch.autocast("cuda", dtype=BF):
        out = m(torch.zeros(0, d, device=hip_device, requires_grad=True), p.clone().requires_grad_(True), idx)
    assert out.shape == (0, d)
    out.sum().backward()
    assert all(not w.grad.any() for w in m.parameters())
    layer = MoELayer(ModelConfig(hidden_size=d, intermediate_size=f, n_experts=5, n_shared_experts=1, n_experts_per_token=k))
    served = layer.to(hip_device).bfloat16().quantize_fp8()
    served.gate.expert_biases = served.gate.expert_biases.float()
    h = torch.randn(2, 3, d, generator=gen(1)).to(BF).to(hip_device)
    rows = torch.zeros(0, dtype=torch.int64, device=hip_device)
    with torch.no_grad():
        out, ids = served(h, unpad_indices=rows)
        assert out.shape == h.shape and not out.any() and ids.shape == (2, 3, k) and not ids.any()
        out, ids = served(h[:0])
        assert out.shape == (0, 3, d) and ids.shape == (0, 3, k)
        assert served.shared_experts(h[:0]).shape == (0, 3, d)


@pytest.mark.parametrize("k", [1, 3, 7, 16])
def test_slots_and_views(k, hip_device):
    """Any number of slots; routing, rows and residual as views, against the same in rows of their own."""
    from scattermoe.mlp import GLUMLP

    T, d, f, E = 21, 128, 96, 20
    s = GLUMLP(d, f, E, k).to(hip_device).to(BF).quantize_fp8()
    idx, p = random_topk(T, E, k, 1).to(hip_device), torch.rand(T, k, generator=gen(2)).to(hip_device)
    x, res = activations(T, d, BF, 3, hip_device), activations(T, d, BF, 4, hip_device)
    out = s(x, p, idx, residual=res)
    wide = torch.cat([x, res], 1)
    got = s(wide[:, :d], p.t().contiguous().t(), idx.t().contiguous().t().to(torch.int32), residual=wide[:, d:])
    assert torch.equal(got, out)
    assert torch.equal(s(x.view(3, 7, d), p, idx, residual=res.view(3, 7, d)).view(T, d), out)
    one = s(x, p, idx, residual=res[:1].expand(T, d))
    assert torch.equal(one, s(x, p, idx, residual=res[:1].repeat(T, 1)))


def test_copies_of_modules(hip_device):
    from scattermoe.mlp import GLUMLP
    from zmoe import fp8
    from zmoe.functional import fp8_linear

    T, d, f, E, k = 9, 128, 96, 4, 2
    s = GLUMLP(d, f, E, k).to(hip_device).to(BF).quantize_fp8()
    idx, p = random_topk(T, E, k, 1).to(hip_device), torch.rand(T, k, generator=gen(2)).to(hip_device)
    x = activations(T, d, BF, 3, hip_device)
    out = s(x, p, idx)
    other = GLUMLP(d, f, E, k).to(hip_device).to(BF).quantize_fp8()
    file = io.BytesIO()
    torch.save(s.state_dict(), file)
    file.seek(0)
    other.load_state_dict(torch.load(file, weights_only=True))
    for m in (copy.deepcopy(s), other, s.cpu().to(hip_device)):
        assert torch.equal(m(x, p, idx), out)
    q = fp8.quantize_weight(weight((72, d), 5, BF, hip_device), True)
    for c in (copy.deepcopy(q), q.to("cpu").to(hip_device)):
        assert torch.equal(fp8_linear(x, c), fp8_linear(x, q)) and torch.equal(c.qt.view(torch.uint8), q.qt.view(torch.uint8))


def test_backward_twice_and_recomputed(hip_device):
    """A graph gone through twice gives the same gradients; checkpointed calls those of plain ones."""
    from scattermoe.mlp import GLUMLP
    from zmoe.functional import fp8_linear, norm_residual

    T, d, f, E, k = 40, 128, 96, 4, 2
    m = GLUMLP(d, f, E, k, fp8=True).to(hip_device).to(BF)
    W, w1, w2 = (weight(s, i, BF, hip_device).requires_grad_(True) for i, s in enumerate(((d, d), (d,), (d,))))
    idx = random_topk(T, E, k, 1).to(hip_device)
    x, p = activations(T, d, BF, 3, hip_device).requires_grad_(True), torch.rand(T, k, generator=gen(2)).to(hip_device).requires_grad_(True)
    dout = activations(T, d, BF, 6, hip_device)

    def block(x, p):
        y = fp8_linear(m(x, p, idx), W)
        r, n = norm_residual(x, y, w1, w2)
        return r + n

    leaves = [x, p, W, w1, w2, *m.parameters()]
    out = block(x, p)
    first = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    second = torch.autograd.grad(out, leaves, dout)
    for reentrant in (False, True):
        again = checkpoint(block, x, p, use_reentrant=reentrant)
        assert torch.equal(again, out)
        for v in leaves:
            v.grad = None
        again.backward(dout)
        for a, b, v in zip(first, second, leaves):
            assert torch.equal(a, b) and torch.equal(a, v.grad)


def test_training_step_captured(hip_device):
    """SwiGLU experts trained in e4m3, forward and backward in a graph: replays on new inputs and routing, with eager steps
    between, bit for bit."""
    from scattermoe.mlp import GLUMLP

    T, d, f, E, k = 50, 136, 100, 6, 2
    m = GLUMLP(d, f, E, k, fp8=True).to(hip_device).to(BF)
    names = [n for n, _ in m.named_parameters()]
    weights = {n: p.detach().clone() for n, p in m.named_parameters()}

    def inputs(seed):
        return [activations(T, d, BF, seed, hip_device), torch.rand(T, k, generator=gen(seed)).to(hip_device),
                random_topk(T, E, k, seed).to(hip_device), activations(T, d, BF, seed + 1, hip_device)]

    def step(x, p, idx, dout):
        leaves = [x.detach().requires_grad_(True), p.detach().requires_grad_(True)]
        own = {n: w.detach().requires_grad_(True) for n, w in weights.items()}
        out = torch.func.functional_call(m, own, (leaves[0], leaves[1], idx))
        return [out.detach(), *torch.autograd.grad(out, leaves + [own[n] for n in names], dout)]

    held = inputs(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for seed in (3, 5, 7):
        new = inputs(seed)
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step(*new)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("what", ["norm", "experts", "served", "layer"])
def test_compiled_as_eager(what, hip_device):
    """Training of norm_residual and of SwiGLU experts in e4m3, and the served modules, compiled in one graph."""
    from modeling.model_config import ModelConfig
    from modeling.moe_layer import MoELayer
    from scattermoe.mlp import GLUMLP
    from zmoe.functional import norm_residual

    T, d, f, E, k = 24, 128, 64, 8, 2
    idx, p = random_topk(T, E, k, 1).to(hip_device), torch.rand(T, k, generator=gen(2)).to(hip_device)
    x = activations(T, d, BF, 3, hip_device)
    torch._dynamo.reset()
    if what in ("norm", "experts"):
        m = GLUMLP(d, f, E, k, fp8=True).to(hip_device).to(BF)
        w1, w2, g = (weight((d,), i, BF, hip_device).requires_grad_(True) for i in (5, 6, 7))
        scale = torch.full((1,), 0.9, device=hip_device, requires_grad=True)

        def fn(x, p):
            if what == "experts":
                return m(x, p, idx)
            r, n = norm_residual(x, x * 0.5, w1, w2, g, scale)
            return r + n

        dout, outs = activations(T, d, BF, 4, hip_device), []
        for call in (fn, torch.compile(fn, fullgraph=True, backend="aot_eager")):
            xi, pi = x.clone().requires_grad_(True), p.clone().requires_grad_(True)
            leaves = [xi, pi, *m.parameters()] if what == "experts" else [xi, w1, w2, g, scale]
            out = call(xi, pi)
            outs.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
        assert all(torch.equal(a, b) for a, b in zip(*outs))
        return
    if what == "served":
        s = GLUMLP(d, f, E, k).to(hip_device).to(BF).quantize_fp8()
        call = lambda x: s(x, p, idx, residual=x)  # noqa: E731
    else:
        layer = MoELayer(ModelConfig(hidden_size=d, intermediate_size=f, n_experts=9, n_shared_experts=1, n_experts_per_token=k))
        s = layer.to(hip_device).bfloat16().quantize_fp8()
        s.gate.expert_biases = s.gate.expert_biases.float()
        call = lambda x: s(x.view(2, T // 2, d))[0]  # noqa: E731
    with torch.no_grad():
        assert torch.equal(torch.compile(call, fullgraph=True, backend="aot_eager")(x), call(x))
