"""The public entry points over the e4m3 products: fp8_linear, parallel_linear(fp8=True), the serving modules.

Their products are held to float64 by the same bound as the kernels' own (test_gpu_fp8), their compositions to the
ops they are made of, bit for bit."""

import pytest
import torch
import torch.nn as nn

from helpers import gen, random_topk
from oracle import fp8_oracle as O
from test_gpu_fp8 import activations, check, some

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def zl():
    from zmoe import library

    return library


def rows_values(q, s, K):
    from zmoe import fp8

    return fp8.dequantize_rows(q, s, K).double()


def weight(shape, seed, dtype, dev, std=0.05):
    return (torch.randn(*shape, generator=gen(seed)) * std).to(dtype).to(dev)


# ------------------------------------------------------------------ the SwiGLU product
def swiglu_check(aq, as_, f, xr, up_w, gate_w, d):
    """Quantised silu(gate) up of rows xr (values) against float64. With eu, eg the products' bounds,
    |delta a| <= |silu(g)| eu + 1.1 (|u| + eu) eg + 2^-18 |a| =: D (|silu'| <= 1.1, the sigmoid is good to 2^-19);
    the scale has to be one that an amax within D of the exact one gives, the values within half a step of
    e4m3, 2^-4 (|a| + D), or of its denormals, 2^-10 of the scale, on top of D."""
    u, Su, Gu = O.product(xr, up_w)
    g, Sg, Gg = O.product(xr, gate_w)
    n = -(-d // 128)
    eu, eg = (7 * 2.0 ** -13 * G + 17 * n * 2.0 ** -23 * S for G, S in ((Gu, Su), (Gg, Sg)))
    silu = g * torch.sigmoid(g)
    a = silu * u
    D = silu.abs() * eu + 1.1 * (u.abs() + eu) * eg + 2.0 ** -18 * a.abs()
    got = rows_values(aq, as_, f)
    assert not rows_values(aq, as_, aq.shape[1])[:, f:].any()
    for b in range(-(-f // 128)):
        sl = slice(128 * b, min(f, 128 * b + 128))
        c = as_[:, b].to(torch.int64) - 127
        lo = (a[:, sl].abs() - D[:, sl]).clamp(min=0).amax(1)
        hi = (a[:, sl].abs() + D[:, sl]).amax(1)
        assert (c >= O.scale_exponent(lo)).all() and (c <= O.scale_exponent(hi)).all()
        bound = D[:, sl] + 2.0 ** -4 * (a[:, sl].abs() + D[:, sl]) + 2.0 ** -10 * O.two(c).unsqueeze(1)
        assert ((got[:, sl] - a[:, sl]).abs() <= bound).all()


@pytest.mark.parametrize("T,d,f", [(1, 256, 128), (5, 100, 30), (40, 512, 160), (130, 384, 200), (300, 256, 768)])
def test_swiglu_dense(T, d, f, hip_device):
    x, W1 = activations(T, d, BF, T, hip_device), weight((2, f, d), f, BF, hip_device)
    xq, xs = zl().fp8_quantize_rows(x, None, 1, None)
    w1q, w1s = zl().fp8_quantize_weight(W1, False)
    from zmoe import ops

    aq, as_ = ops.fp8_glu_w1_forward(xq, xs, w1q, w1s, d)
    wr = O.quantize_weight(W1)[0]
    swiglu_check(aq, as_, f, O.quantize_rows(x)[0], wr[0], wr[1], d)


@pytest.mark.parametrize("T,d,f,E,k,skew", [(1, 256, 128, 8, 2, 0.0), (40, 200, 160, 8, 2, 0.5), (300, 256, 130, 4, 2, 1.0),
                                            (900, 128, 256, 3, 2, 0.0), (64, 256, 100, 130, 4, 1.0)])
def test_swiglu_grouped(T, d, f, E, k, skew, hip_device):
    from zmoe import ops

    idx = random_topk(T, E, k, T, skew).to(hip_device)
    _, ss, off, _ = ops.flatten_sort_count(idx, E)
    x, W1 = activations(T, d, BF, T, hip_device), weight((E, 2 * f, d), f, BF, hip_device)
    w1q, w1s = zl().fp8_quantize_weight(W1.view(2 * E, f, d), False)
    aq, as_ = ops.fp8_glu_w1_forward(*ops.fp8_quantize_rows(x), w1q, w1s, d, ss, off, k)
    wr, xr = O.quantize_weight(W1.view(2 * E, f, d))[0], O.quantize_rows(x)[0]
    beg = 0
    for e, end in enumerate(off.tolist()):
        if end > beg:
            swiglu_check(aq[beg:end], as_[beg:end], f, xr[ss[beg:end] // k], wr[2 * e], wr[2 * e + 1], d)
        beg = end


@pytest.mark.parametrize("T,d,f,E,k", [(600, 300, 1700, 1, 1), (1100, 256, 2000, 1, 1), (1500, 200, 3000, 1, 1),
                                       (1500, 4100, 3000, 1, 1), (1000, 8300, 4300, 1, 1), (1500, 200, 4300, 1, 1),
                                       (700, 8300, 1700, 1, 1), (500, 260, 1300, 16, 4),
                                       (1500, 8300, 4300, 1, 1), (2000, 300, 520, 16, 2), (6000, 260, 520, 16, 2),
                                       (5000, 4100, 1200, 3, 1)])
def test_swiglu_tiles(T, d, f, E, k, hip_device):
    """Sizes for every tile, sampled rows."""
    from zmoe import ops

    x, W1 = activations(T, d, BF, T, hip_device), weight((2 * E, f, d), f, BF, hip_device)
    idx = random_topk(T, E, k, T, 0.0).to(hip_device) if E > 1 else torch.zeros(T, 1, dtype=torch.int64, device=hip_device)
    w1q, w1s = zl().fp8_quantize_weight(W1, False)
    _, ss, off, _ = ops.flatten_sort_count(idx, E)
    route = (ss, off, k) if E > 1 else ()
    aq, as_ = ops.fp8_glu_w1_forward(*ops.fp8_quantize_rows(x), w1q, w1s, d, *route)
    wr, xr = O.quantize_weight(W1)[0], O.quantize_rows(x)[0]
    ri = some(T * k, 24, 3).to(hip_device)
    slots = ss[ri] if E > 1 else ri
    experts = idx.flatten()[slots]
    for e in experts.unique().tolist():
        at = ri[experts == e]
        swiglu_check(aq[at], as_[at], f, xr[slots[experts == e] // k], wr[2 * e], wr[2 * e + 1], d)


# ------------------------------------------------------------------ fp8_linear
def wgrad_close(got, dy, x):
    """dy^T x of 16- or 32-bit operands, summed in f32: half a step of the result, and one rounding of the
    partial sum, at most S = sum |terms|, for each of M terms."""
    ref, S = dy.double().T @ x.double(), dy.double().abs().T @ x.double().abs()
    half = 2.0 ** -8 if got.dtype == BF else 2.0 ** -24
    assert ((got.double() - ref).abs() <= half * ref.abs() + (dy.shape[0] + 2) * 2.0 ** -24 * S).all()


@pytest.mark.parametrize("xt,wt", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("lead,K,N", [((1,), 256, 128), ((3, 5), 100, 260), ((150,), 501, 333), ((0,), 64, 64)])
def test_linear(lead, K, N, xt, wt, hip_device):
    from zmoe.functional import fp8_linear

    x = activations(max(1, torch.Size(lead).numel()), K, DT[xt], K, hip_device)[:torch.Size(lead).numel()].view(*lead, K)
    W = weight((N, K), N, DT[wt], hip_device)
    dy = activations(x.numel() // K, N, DT[xt], 7, hip_device).view(*lead, N) if x.numel() else x.new_zeros(*lead, N)
    x.requires_grad_(True)
    W.requires_grad_(True)
    y = fp8_linear(x, W)
    assert y.shape == (*lead, N) and y.dtype == x.dtype
    y.backward(dy)
    assert x.grad.dtype == x.dtype and W.grad.dtype == W.dtype
    x2, dy2 = x.detach().reshape(-1, K), dy.reshape(-1, N)
    wr = O.quantize_weight(W.detach())[0]
    check(y.detach().reshape(-1, N), *O.product(O.quantize_rows(x2)[0], wr), K)
    check(x.grad.reshape(-1, K), *O.product(O.quantize_rows(dy2)[0], wr.T), N)
    wgrad_close(W.grad, dy2, x2)


def test_linear_gradient_against_differences(hip_device):
    """With the quantisers passing gradients through, <dy, x Q(W)^T> changes along v as <dx, v>: dx holds
    dy rounded to e4m3, off by at most 2^-4 of each term (block scales: no denormals at these values)."""
    from zmoe.functional import fp8_linear

    x, W = activations(20, 256, BF, 1, hip_device), weight((384, 256), 2, BF, hip_device)
    dy = (torch.randn(20, 384, generator=gen(3)).clamp(-2, 2) + 3).to(BF).to(hip_device)
    x.requires_grad_(True)
    fp8_linear(x, W).backward(dy)
    wr = O.quantize_weight(W)[0]
    v = torch.randn(20, 256, generator=gen(4)).to(hip_device).double()
    f = lambda s: float((dy.double() * ((x.detach().double() + s * v) @ wr.T)).sum())  # noqa: E731
    slope = (f(1e-3) - f(-1e-3)) / 2e-3
    terms = float((dy.double().abs() * (v @ wr.T).abs()).sum())
    assert abs(float((x.grad.double() * v).sum()) - slope) <= (2.0 ** -4 + 2.0 ** -8) * terms


@pytest.mark.parametrize("transposed", [False, True])
def test_linear_served(transposed, hip_device):
    from zmoe import fp8
    from zmoe.functional import fp8_linear

    x, W = activations(33, 300, BF, 1, hip_device), weight((200, 300), 2, torch.float32, hip_device)
    q = fp8.quantize_weight(W, transposed)
    assert q.shape == W.shape and torch.equal(q.dequantize().double(), O.quantize_weight(W)[0])
    assert torch.equal(fp8_linear(x, q), fp8_linear(x, W))
    x.requires_grad_(True)
    if not transposed:
        with pytest.raises(RuntimeError):
            fp8_linear(x, q)
        return
    dy = activations(33, 200, BF, 3, hip_device)
    ga, gb = (torch.autograd.grad(fp8_linear(x, w), x, dy)[0] for w in (q, W))
    assert torch.equal(ga, gb)


def test_linear_operand_views(hip_device):
    """Strided, expanded and off-16-byte inputs and output grads; autocast; a frozen weight or input."""
    from zmoe.functional import fp8_linear

    big = activations(64, 700, BF, 1, hip_device)
    W = weight((96, 256), 2, BF, hip_device)
    for x in (big[:, 3:259], big[::2, :256], big[:1, :256].expand(40, 256), big.t()[:256].t(), big.view(-1)[1:1 + 16 * 256].view(16, 256)):
        xr = x.detach().requires_grad_(True)
        xc = x.contiguous().clone().requires_grad_(True)
        Wa, Wb = W.clone().requires_grad_(True), W.clone().requires_grad_(True)
        a, b = fp8_linear(xr, Wa), fp8_linear(xc, Wb)
        assert torch.equal(a, b)
        a.backward(torch.ones((), device=hip_device, dtype=BF).expand(a.shape))
        b.backward(torch.ones_like(b))
        assert torch.equal(xr.grad, xc.grad) and torch.equal(Wa.grad, Wb.grad)
    x32 = big[:, :256].float()
    with torch.autocast("cuda", dtype=BF):
        assert torch.equal(fp8_linear(x32, W), fp8_linear(big[:, :256], W))
    x, Wf = big[:, :256].clone().requires_grad_(True), W.clone().requires_grad_(True)
    fp8_linear(x, W).sum().backward()
    fp8_linear(big[:, :256], Wf).sum().backward()
    assert x.grad is not None and Wf.grad is not None


# ------------------------------------------------------------------ parallel_linear(fp8=True)
@pytest.mark.parametrize("wt", ["bf16", "f32"])
@pytest.mark.parametrize("T,K,N,E,k,skew", [(1, 128, 256, 8, 2, 0.0), (90, 130, 200, 6, 3, 0.7), (400, 256, 264, 4, 2, 1.0)])
def test_parallel_linear_gathered(T, K, N, E, k, skew, wt, hip_device):
    """An expert MLP's first product: rows gathered, sorted output rows."""
    from scattermoe.parallel_experts import flatten_sort_count, parallel_linear

    idx = random_topk(T, E, k, T, skew).to(hip_device)
    se, ss, off = flatten_sort_count(idx, E)
    x = activations(T, K, BF, T, hip_device).requires_grad_(True)
    W = weight((E, N, K), N, DT[wt], hip_device).requires_grad_(True)
    dy = activations(T * k, N, BF, 5, hip_device)
    y = parallel_linear(x, W.permute(0, 2, 1), k, se, ss, off, grouped_out=True, fp8=True)
    y.backward(dy)
    wr = O.quantize_weight(W.detach())[0]
    check(y.detach(), *O.grouped_product(O.quantize_rows(x.detach())[0], wr, ss, off, k, False, True), K)
    v, S, G = O.grouped_product(O.quantize_rows(dy)[0], wr.transpose(1, 2), ss, off, 1, True, False)
    # a slot's row is held to 2^-12 of each value (2^-11 half steps of f16, or 2^-25 beside one of 2^14) and the k of a
    # token are added before the one rounding to bf16
    fold = lambda t: t.view(T, k, K).sum(1)  # noqa: E731
    top = torch.nn.functional.pad(v.abs(), (0, -K % 64)).view(T * k, -1, 64).amax(-1, keepdim=True).expand(-1, -1, 64)
    top = top.reshape(T * k, -1)[:, :K]
    b = 2.0 ** -8 * fold(v).abs() + 1.01 * fold(2.0 ** -11 * v.abs() + 2.0 ** -38 * top + 7 * 2.0 ** -13 * G
                                               + 17 * -(-N // 128) * 2.0 ** -23 * S)
    assert ((x.grad.double() - fold(v)).abs() <= b).all()
    assert W.grad.dtype == W.dtype and W.grad.shape == W.shape
    beg = 0
    for e, end in enumerate(off.tolist()):
        wgrad_close(W.grad[e], dy[beg:end], x.detach()[ss[beg:end] // k])
        beg = end


def test_parallel_linear_gates(hip_device):
    """An expert MLP's second product: sorted rows in, gate-weighted sums out. The pieces, from the ops."""
    from scattermoe.kernels import ops as ko
    from scattermoe.parallel_experts import flatten_sort_count, parallel_linear

    T, K, N, E, k = 60, 200, 130, 5, 2
    idx = random_topk(T, E, k, 3).to(hip_device)
    se, ss, off = flatten_sort_count(idx, E)
    x = activations(T * k, K, BF, 1, hip_device).requires_grad_(True)
    W = weight((E, N, K), 2, BF, hip_device).requires_grad_(True)
    p = torch.rand(T, k, generator=gen(4)).to(hip_device).requires_grad_(True)
    dy = activations(T, N, BF, 5, hip_device)
    out = parallel_linear(x, W.permute(0, 2, 1), 1, se, ss, off, gates=p, grouped_in=True, fp8=True)
    out.backward(dy)
    with torch.no_grad():
        q = zl().fp8_quantize_weight(W, True)
        Y = zl().fp8_mm(*zl().fp8_quantize_rows(x, None, 1, None), *q[:2], K, ss, off, 1, True, False, False)
        assert torch.equal(out, zl().combine(Y, p, k, None, None, 0))
        G = dy.float()[ss // k] * p.reshape(-1)[ss].unsqueeze(1)
        gr, cr = O.quantize_rows(G)
        v, S, Gm = O.grouped_product(gr, O.quantize_weight(W)[0].transpose(1, 2), ss, off, 1, True, True)
        check(x.grad, v, S, Gm, N)
        ref = ko.rowwise_sum_product(Y.view(T, k, N), dy, dtype=torch.float32)
        assert torch.equal(p.grad, ref)
        grouped = ko.group(dy, ss, coeff=p.reshape(-1), fan_out=k)
        assert torch.equal(W.grad, zl().group_bwd_w(grouped, x, off, E, None, 1))


def test_expert_mlps_train(hip_device):
    """MLP and GLUMLP with fp8 products: every grad, and grads near those of the 16-bit module (e4m3 operands
    are within 2^-4 each: a product of two chained ones within a quarter of the norm)."""
    from scattermoe.mlp import GLUMLP, MLP

    T, d, f, E, k = 64, 128, 96, 4, 2
    idx = random_topk(T, E, k, 1).to(hip_device)
    for make in (lambda fp8: GLUMLP(d, f, E, k, fp8=fp8), lambda fp8: MLP(d, f, E, k, activation=nn.GELU(), fp8=fp8)):
        torch.manual_seed(0)
        a = make(True).to(hip_device)
        b = make(False).to(hip_device)
        b.load_state_dict(a.state_dict())
        p = torch.rand(T, k, generator=gen(2)).to(hip_device)
        x = torch.randn(T, d, generator=gen(3)).to(hip_device)
        dout = torch.randn(T, d, generator=gen(4)).to(hip_device)
        got = []
        for m in (a, b):
            xi, pi = x.clone().requires_grad_(True), p.clone().requires_grad_(True)
            with torch.autocast("cuda", dtype=BF):
                out = m(xi, pi, idx)
            out.backward(dout.to(out.dtype))
            got.append([out.detach(), xi.grad, pi.grad, *(w.grad for w in m.parameters())])
        for u, v in zip(*got):
            assert u.dtype == v.dtype and float((u.double() - v.double()).norm() / v.double().norm()) < 0.25


# ------------------------------------------------------------------ f16 rows and their sums
def row_top(v):
    """The largest magnitude of each 64 columns, in each of them."""
    K = v.shape[1]
    t = torch.nn.functional.pad(v.abs(), (0, -K % 64)).view(v.shape[0], -1, 64).amax(-1, keepdim=True).expand(-1, -1, 64)
    return t.reshape(v.shape[0], -1)[:, :K]


def half_check(Y, Ys, val, S, G, K):
    """f16 rows over their scales: 2^-11 of a value (half a step, and the product's own error), or half a
    step of f16's denormals, 2^-25 where the largest of the 64 is 2^14: 2^-39 of it."""
    N = val.shape[1]
    got = (Y.double() * O.two(Ys.to(torch.int64) - 127).repeat_interleave(64, 1))[:, :N]
    bound = 2.0 ** -11 * val.abs() + 2.0 ** -38 * row_top(val) + 1.01 * (7 * 2.0 ** -13 * G + 17 * -(-K // 128) * 2.0 ** -23 * S)
    assert ((got - val).abs() <= bound).all()
    assert not Y[:, N:].any()


@pytest.mark.parametrize("T,k,N,K", [(1, 1, 1, 64), (5, 2, 130, 200), (33, 3, 64, 256), (300, 8, 264, 128), (70, 4, 511, 130)])
def test_half_rows_and_their_sums(T, k, N, K, hip_device):
    from zmoe import ops

    E = 9
    idx = random_topk(T, E, k, T).to(hip_device)
    _, ss, off, _ = ops.flatten_sort_count(idx, E)
    x = activations(T * k, K, BF, 1, hip_device) * torch.exp2(torch.arange(T * k) % 40 - 20.).to(hip_device).unsqueeze(1).to(BF)
    W = weight((E, N, K), 2, BF, hip_device)
    Y, Ys = ops.fp8_scatter2scatter_half(*ops.fp8_quantize_rows(x), *ops.fp8_quantize_weight(W), K, ss, off, 1, True, False)
    half_check(Y, Ys, *O.grouped_product(O.quantize_rows(x)[0], O.quantize_weight(W)[0], ss, off, 1, True, False), K)
    rows = (Y.double() * O.two(Ys.to(torch.int64) - 127).repeat_interleave(64, 1))[:, :N].view(T, k, N)
    g = torch.randn(T, k, generator=gen(3)).to(hip_device)
    for dt in (BF, torch.float32):
        add = torch.randn(T, N, generator=gen(4)).to(dt).to(hip_device)
        at = torch.randperm(T + 3, generator=gen(5))[:T].to(hip_device)
        for gates, addend, out_rows in ((None, None, None), (g, None, None), (g, add, None), (g, add, at)):
            out = ops.combine_half(Y, Ys, gates, k, N, addend, out_rows, T + 3, out_dtype=dt)
            w = torch.ones_like(g) if gates is None else gates
            a = torch.zeros_like(add) if addend is None else addend
            ref = (w.double().unsqueeze(-1) * rows).sum(1) + a.double()
            mag = (w.double().abs().unsqueeze(-1) * rows.abs()).sum(1) + a.double().abs()
            got = out if out_rows is None else out[at]
            half = 2.0 ** -8 if dt == BF else 2.0 ** -24
            assert ((got.double() - ref).abs() <= half * ref.abs() + (k + 2) * 2.0 ** -24 * mag).all()
            if out_rows is not None:
                assert not out[[i for i in range(T + 3) if i not in at.tolist()]].any()


@pytest.mark.parametrize("T", [1, 2, 5])
def test_few_rows_of_narrow_experts_are_exact_before_the_rounding(T, hip_device):
    """The activations of a small launch are rounded to e4m3 from f32 sums, so that none lands on a neighbour (2^-3 away,
    0.018 of the result in single rows) and the result's error is its own rounding to bf16: at most 2^-8 of each value,
    uniform below half a step, so of a norm hardly over 2^-8 / sqrt(3 * 1.5 / ln 2) = 0.0015; the bound is half of 2^-8."""
    d, f, E, k = 512, 160, 32, 2
    for seed in range(20):
        x, W1 = activations(T, d, BF, seed, hip_device), weight((2 * E, f, d), seed + 1, BF, hip_device, d ** -0.5)
        W2 = weight((E, d, f), seed + 2, BF, hip_device, f ** -0.5)
        idx = random_topk(T, E, k, seed).to(hip_device)
        p = torch.softmax(torch.randn(T, k, generator=gen(seed)), -1).to(hip_device)
        out, _ = zl().fp8_glu_experts(x, p, idx, *zl().fp8_quantize_weight(W1, False), *zl().fp8_quantize_weight(W2, False),
                                      None, None, 0)
        xr, w1, w2 = O.quantize_rows(x)[0], O.quantize_weight(W1)[0], O.quantize_weight(W2)[0]
        ref = torch.zeros(T, d, dtype=torch.float64, device=hip_device)
        for t in range(T):
            for j in range(k):
                e = int(idx[t, j])
                u, g = xr[t] @ w1[2 * e].T, xr[t] @ w1[2 * e + 1].T
                a = O.quantize_rows((g * torch.sigmoid(g) * u).unsqueeze(0))[0]
                ref[t] += p[t, j].double() * (a @ w2[e].T)[0]
        assert float((out.double() - ref).norm() / ref.norm()) <= 2.0 ** -9


@pytest.mark.parametrize("T,d,f,E,k", [(1500, 512, 160, 32, 2), (300, 1000, 512, 16, 4), (1300, 512, 1500, 1, 1)])
def test_exact_sums_do_not_depend_on_the_tile(T, d, f, E, k, hip_device):
    """Rows of a launch on 64-row tiles are those of launches of their own on 32-row ones, bit for bit."""
    from zmoe import ops

    x, W1 = activations(T, d, BF, T, hip_device), weight((2 * E, f, d), 1, BF, hip_device)
    idx = random_topk(T, E, k, 1).to(hip_device) if E > 1 else torch.zeros(T, 1, dtype=torch.int64, device=hip_device)
    w = ops.fp8_quantize_weight(W1)

    def run(rows):
        _, ss, off, _ = ops.flatten_sort_count(idx[rows], E)
        aq, as_ = ops.fp8_glu_w1_forward(*ops.fp8_quantize_rows(x[rows]), *w, d, ss, off, k)
        out = torch.empty_like(aq.view(torch.uint8)), torch.empty_like(as_[:, :-(-f // 128)])
        out[0][ss], out[1][ss] = aq.view(torch.uint8), as_[:, :-(-f // 128)]
        return out

    q, s = run(torch.arange(T, device=hip_device))
    for rows in (some(T, 7, 1), some(T, 30, 2)):
        rows = rows.to(hip_device)
        slots = (rows.unsqueeze(1) * k + torch.arange(k, device=hip_device)).flatten()
        a, b = run(rows)
        assert torch.equal(a, q[slots]) and torch.equal(b, s[slots])


def test_experts_not_finite_and_twice_the_same(hip_device):
    """A row with a NaN and one with an inf spoil themselves alone; a token may name one expert twice."""
    from zmoe import ops

    T, d, f, E, k = 9, 256, 130, 4, 2
    x, idx = activations(T, d, BF, 1, hip_device), random_topk(T, E, k, 3).to(hip_device)
    idx[4, 1] = idx[4, 0]
    p = torch.rand(T, k, generator=gen(2)).to(hip_device)
    w = [*ops.fp8_quantize_weight(weight((2 * E, f, d), 3, BF, hip_device)), *ops.fp8_quantize_weight(weight((E, d, f), 4, BF, hip_device))]
    out, off = ops.fp8_glu_experts(x, p, idx, *w)
    bad = x.clone()
    bad[2, 7], bad[6, 200] = float("nan"), float("inf")
    got, _ = ops.fp8_glu_experts(bad, p, idx, *w)
    spoilt = torch.tensor([t in (2, 6) for t in range(T)], device=hip_device)
    assert torch.isnan(got[spoilt]).all() and torch.equal(got[~spoilt], out[~spoilt])
    one = torch.stack([p[4].sum(), torch.zeros((), device=hip_device)]).view(1, 2)
    alone, _ = ops.fp8_glu_experts(x[4:5], one, idx[4:5], *w)
    assert float((alone - out[4:5]).float().norm()) <= 2.0 ** -7 * float(alone.float().norm())


def test_on_another_stream(hip_device):
    """Work queued on a side stream, while the default one is busy with other calls of the same ops."""
    from zmoe import ops

    T, d, f, E, k = 300, 512, 160, 8, 2
    x, idx = activations(T, d, BF, 1, hip_device), random_topk(T, E, k, 3).to(hip_device)
    p = torch.rand(T, k, generator=gen(2)).to(hip_device)
    w = [*ops.fp8_quantize_weight(weight((2 * E, f, d), 3, BF, hip_device)), *ops.fp8_quantize_weight(weight((E, d, f), 4, BF, hip_device))]
    run = lambda: (ops.fp8_glu_experts(x, p, idx, *w)[0], ops.fp8_linear(x, w[0][0], w[1][0]))  # noqa: E731
    ref = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        theirs = [run() for _ in range(5)]
    ours = [run() for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for pair in theirs + ours:
        for a, b in zip(pair, ref):
            assert torch.equal(a, b)


def test_half_rows_not_finite(hip_device):
    """inf and NaN reach their own rows only, and the largest finite sums do not overflow."""
    from zmoe import ops

    x = torch.ones(6, 128, dtype=torch.float32, device=hip_device)
    x[1, 5], x[2, 7], x[3] = float("inf"), float("nan"), 3e37
    W = torch.ones(70, 128, device=hip_device)
    Y, Ys = ops.fp8_scatter2scatter_half(*ops.fp8_quantize_rows(x), *ops.fp8_quantize_weight(W), 128)
    out = ops.combine_half(Y, Ys, None, 1, 70, out_dtype=torch.float32)
    assert torch.isnan(out[1]).all() and torch.isnan(out[2]).all()
    assert (out[0] == 128).all() and (out[5] == 128).all()
    ref = O.quantize_rows(x[3:4])[0].sum()  # beyond f32: infinite; below: itself
    big = float(ref) if float(ref) < 3.4e38 else float("inf")
    assert (out[3] == big).all() or abs(float(out[3, 0]) / big - 1) < 1e-3


# ------------------------------------------------------------------ serving modules
@pytest.mark.parametrize("T,d,f,E,k", [(1, 128, 64, 8, 2), (37, 200, 100, 8, 3), (600, 256, 160, 4, 2), (0, 64, 64, 4, 2)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_served_experts(T, d, f, E, k, dtype, hip_device):
    from scattermoe.mlp import GLUMLP
    from zmoe import ops

    torch.manual_seed(1)
    m = GLUMLP(d, f, E, k).to(hip_device).to(DT[dtype])
    s = m.quantize_fp8()
    idx = random_topk(T, E, k, T + 1).to(hip_device)
    p = torch.rand(T, k, generator=gen(2)).to(hip_device)
    x = activations(T, d, DT[dtype], 3, hip_device) if T else torch.zeros(0, d, device=hip_device, dtype=DT[dtype])
    res = torch.randn(T, d, generator=gen(4)).to(DT[dtype]).to(hip_device)
    with torch.no_grad():
        out = s(x, p, idx)
        assert out.shape == x.shape and out.dtype == x.dtype
        if T == 0:
            return
        W1, W2 = m.experts.weight, m.output_experts.weight
        _, ss, off, _ = ops.flatten_sort_count(idx, E)
        aq, as_ = ops.fp8_glu_w1_forward(*ops.fp8_quantize_rows(x), *ops.fp8_quantize_weight(W1.view(2 * E, f, d)), d, ss, off, k)
        w2 = ops.fp8_quantize_weight(W2)
        val, S, G = O.grouped_product(rows_values(aq, as_, f), O.quantize_weight(W2)[0], ss, off, 1, True, False)
        if dtype == "f32":
            Y = ops.fp8_scatter2scatter(aq, as_, *w2, f, ss, off, 1, True, False, DT[dtype])
            check(Y, val, S, G, f)
            total = lambda *a, **kw: ops.combine(Y, p, k, *a, **kw)  # noqa: E731
        else:
            Y, Ys = ops.fp8_scatter2scatter_half(aq, as_, *w2, f, ss, off, 1, True, False)
            total = lambda *a, **kw: ops.combine_half(Y, Ys, p, k, d, *a, **kw)  # noqa: E731
            half_check(Y, Ys, val, S, G, f)
        assert torch.equal(out, total()) and torch.equal(s.last_expert_offsets, off)
        pe = p.double().unsqueeze(-1)
        ref, err = ((pe * v.view(T, k, d)).sum(1) for v in (val, 2.0 ** -11 * val.abs() + 7 * 2.0 ** -13 * G
                                                            + (17 * -(-f // 128) * 2.0 ** -23 + 2.0 ** -22) * S + 2.0 ** -38 * row_top(val)))
        half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
        assert ((out.double() - ref).abs() <= half * ref.abs() + 1.01 * err).all()
        assert torch.equal(s(x, p, idx, residual=res), total(res))
        rows = torch.randperm(T + 5, generator=gen(5))[:T].to(hip_device)
        assert torch.equal(s(x, p, idx, pad=(rows, T + 5)), total(out_rows=rows, out_total=T + 5))
        # near the 16-bit experts: two quantised products, 2^-4 of each operand at most
        assert float((out.float() - m(x, p, idx).float()).norm()) < 0.25 * float(out.float().norm())
        again = s.to(torch.float16)  # a module-wide cast leaves the weights alone
        assert torch.equal(again(x, p, idx), out)
    with pytest.raises(RuntimeError):
        s(x.requires_grad_(True), p, idx)


@pytest.mark.parametrize("unpad,norm,mode", [(False, False, "bf16"), (True, True, "bf16"), (True, False, "autocast"),
                                             (False, True, "autocast")])
def test_served_layer(unpad, norm, mode, hip_device):
    from modeling.model_config import ModelConfig
    from modeling.moe_layer import MoELayer
    from modeling.zRMSNorm import ZeroCenteredRMSNorm

    torch.manual_seed(0)
    B, S, d = 2, 9, 128
    layer = MoELayer(ModelConfig(hidden_size=d, intermediate_size=64, n_experts=9, n_shared_experts=1, n_experts_per_token=2))
    layer = layer.to(hip_device)
    if mode == "bf16":
        layer = layer.bfloat16()
        layer.gate.expert_biases.data = layer.gate.expert_biases.data.float()
    served = layer.quantize_fp8()
    pre = ZeroCenteredRMSNorm(d).to(hip_device) if norm else None
    rows = torch.tensor([0, 1, 2, 4, 9, 10, 16], device=hip_device) if unpad else None
    h = torch.randn(B, S, d, generator=gen(1)).to(hip_device).to(BF if mode == "bf16" else torch.float32)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF, enabled=mode == "autocast"):
        out, idx = served(h, unpad_indices=rows, norm=pre)
        ref, ridx = layer(h, unpad_indices=rows, norm=pre)
    assert out.shape == ref.shape and out.dtype == ref.dtype and torch.equal(idx, ridx)
    assert float((out.float() - ref.float()).norm()) < 0.25 * float(ref.float().norm())
    if unpad:
        pad = torch.ones(B * S, dtype=torch.bool, device=hip_device).index_fill(0, rows, False)
        assert not out.view(B * S, d)[pad].any()
    layer.gate.weight.data.zero_()  # the served copy is its own
    with torch.no_grad(), torch.autocast("cuda", dtype=BF, enabled=mode == "autocast"):
        assert torch.equal(served(h, unpad_indices=rows, norm=pre)[0], out)
    with pytest.raises(RuntimeError):
        served(h.clone().requires_grad_(True))
    state = {n: t.clone() for n, t in served.state_dict().items()}
    served.load_state_dict(state)


def test_sublayer_served_and_captured(hip_device):
    """A block's MoE sublayer as a server runs it (norm, fp8 layer, norm_residual), eager and as replays of a graph."""
    from modeling.model_config import ModelConfig
    from modeling.moe_layer import MoELayer
    from modeling.zRMSNorm import NormResidual, ZeroCenteredRMSNorm

    torch.manual_seed(0)
    d = 256
    served = MoELayer(ModelConfig(hidden_size=d, intermediate_size=128, n_experts=17, n_shared_experts=1,
                                  n_experts_per_token=4)).to(hip_device).bfloat16().quantize_fp8()
    served.gate.expert_biases = served.gate.expert_biases.float()
    pre, step, nxt = ZeroCenteredRMSNorm(d), NormResidual(d, gate=True), ZeroCenteredRMSNorm(d)
    for m in (pre, step, nxt):
        m.to(hip_device).requires_grad_(False)
        m.weight.normal_(0, 0.2)

    def sublayer(h):
        with torch.no_grad():
            y, idx = served(h, norm=pre)
            return (*step(h, y, nxt), idx)

    h = torch.randn(4, 1, d, generator=gen(1)).to(BF).to(hip_device)
    sublayer(h)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sublayer(h)
    for seed in (2, 3, 4):
        new = torch.randn(4, 1, d, generator=gen(seed)).to(BF).to(hip_device)
        h.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, sublayer(new)):
            assert torch.equal(a, b)


def test_linear_train_captured(hip_device):
    from zmoe.functional import fp8_linear

    x = activations(50, 264, BF, 1, hip_device)
    W = weight((136, 264), 2, torch.float32, hip_device)
    dy = activations(50, 136, BF, 3, hip_device)

    def stepfn():
        xi, Wi = x.detach().requires_grad_(True), W.detach().requires_grad_(True)
        y = fp8_linear(xi, Wi)
        return (y.detach(), *torch.autograd.grad(y, (xi, Wi), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # also on another stream than the tensors' own
        first = stepfn()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, stepfn()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = stepfn()
    for seed in (4, 5, 6):
        x.copy_(activations(50, 264, BF, seed, hip_device))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, stepfn()))


def test_compiled(hip_device):
    """The ops are custom ops: compiled functions equal eager ones."""
    from zmoe import fp8
    from zmoe.functional import fp8_linear, norm_residual

    x = activations(40, 256, BF, 1, hip_device)
    q = fp8.quantize_weight(weight((256, 256), 2, BF, hip_device))
    w = weight((256,), 3, BF, hip_device)

    def fn(x, q, s):
        y = fp8_linear(x, fp8.Fp8Weight(q, s, 256))
        return norm_residual(x, y, w, w)

    with torch.no_grad():
        ref = fn(x, q.q, q.s)
        got = torch.compile(fn, fullgraph=True, backend="aot_eager")(x, q.q, q.s)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))

    W = weight((96, 256), 4, BF, hip_device)

    def train(x, W):
        y = fp8_linear(x, W)
        return y

    outs = []
    for f in (train, torch.compile(train, fullgraph=True, backend="aot_eager")):
        xi, Wi = x.clone().requires_grad_(True), W.clone().requires_grad_(True)
        y = f(xi, Wi)
        y.backward(torch.ones_like(y))
        outs.append((y.detach(), xi.grad, Wi.grad))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_refusals(hip_device):
    from scattermoe.mlp import GLUMLP, MLP
    from scattermoe.parallel_experts import ParallelExperts, flatten_sort_count, parallel_linear
    from zmoe import fp8, ops
    from zmoe.functional import fp8_linear

    x, W = activations(4, 64, BF, 1, hip_device), weight((32, 64), 2, BF, hip_device)
    q = fp8.quantize_weight(W)
    for bad in (lambda: fp8_linear(x[:, :60], W), lambda: fp8_linear(x, W[None]), lambda: fp8_linear(x[:, :60], q),
                lambda: fp8_linear(x.half(), W.half()), lambda: fp8_linear(x.cpu(), W), lambda: fp8.quantize_weight(W[:0]),
                lambda: ops.fp8_scatter2scatter(*ops.fp8_quantize_rows(x), q.q, q.s, 640),
                lambda: ops.fp8_scatter2scatter(*ops.fp8_quantize_rows(x), q.q, q.s, 64, out_dtype=torch.float16),
                lambda: ops.fp8_scatter2scatter(*ops.fp8_quantize_rows(x), q.q[None], q.s[None], 64),
                lambda: ops.fp8_quantize_rows(x, row_scale=torch.ones(3, device=hip_device)),
                lambda: ParallelExperts(2, 8, 8, bias=True, fp8=True), lambda: MLP(8, 8, 2, 1, bias=True, fp8=True),
                lambda: GLUMLP(8, 8, 2, 1, activation=nn.GELU()).to(hip_device).quantize_fp8(),
                lambda: GLUMLP(8, 8, 2, 1, bias=True).to(hip_device).quantize_fp8()):
        with pytest.raises(ValueError):
            bad()
    idx = random_topk(4, 2, 1, 1).to(hip_device)
    se, ss, off = flatten_sort_count(idx, 2)
    W3 = weight((2, 32, 64), 2, BF, hip_device).permute(0, 2, 1)
    for kw in (dict(expert_biases=torch.zeros(2, 32, device=hip_device)), dict(gates=torch.ones(4, 1, device=hip_device), grouped_out=True)):
        with pytest.raises(ValueError):
            parallel_linear(x, W3, 1, se, ss, off, fp8=True, **kw)
    with pytest.raises(ValueError):
        parallel_linear(x, W3, 2, se, ss, off, fp8=True)
