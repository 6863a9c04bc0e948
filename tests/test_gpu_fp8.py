"""Block-scaled e4m3 on the GPU against the format and the products in float64 (oracle.fp8_oracle).

Tolerances. Quantised values and scales are equal to the oracle's: v / s is exact. A product's terms are exact
(4-bit mantissas times 4-bit ones). The matrix unit adds them 128 at a time: in each group of 8 consecutive
depths it cuts every term off at 2^-13 of the power of two below the group's largest (measured: terms of 1.875 x
1.875 beside one of 2^16 keep bits down to 2^3), so a group loses less than 7 * 2^-13 of its largest term; the 16
group sums and the running sum are added to 24 bits or more, each cut off by less than 2^-23 of a partial sum, which is
at most S = sum |terms|. With G = sum over groups of the largest |term|:
|error| < 7 * 2^-13 G + 17 ceil(K / 128) 2^-23 S, plus half a step of the output, 2^-8 |y| in bf16, 2^-24 |y| in f32.
"""

import pytest
import torch

from helpers import gen, random_topk
from oracle import fp8_oracle as O

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def z():
    from zmoe import ops

    return ops


def same(a, b):
    """Equal, NaN in the same places."""
    return torch.equal(torch.nan_to_num(a.double(), nan=12345.0), torch.nan_to_num(b.double(), nan=12345.0))


def rows_values(q, s, K):
    """The values quantised rows stand for, and their exponents."""
    n, kp = q.shape
    c = s[:, :kp // 128].to(torch.int64) - 127
    v = q.to(torch.float32).double().view(n, kp // 128, 128) * O.two(c).unsqueeze(-1)
    return v.view(n, kp), c


def activations(n, K, dtype, seed, dev):
    g = gen(seed)
    x = torch.randn(n, K, generator=g) * torch.exp(torch.randn(K, generator=g))
    return x.to(dtype).to(dev)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,K", [(1, 1), (1, 128), (3, 127), (5, 129), (7, 510), (64, 512), (33, 2048), (0, 256)])
def test_quantize_rows(n, K, dtype, hip_device):
    x = activations(n, K, DT[dtype], n * K + 1, hip_device)
    q, s = z().fp8_quantize_rows(x)
    v, c = rows_values(q, s, K)
    ref, cref = O.quantize_rows(x)
    assert torch.equal(c, cref) and torch.equal(v[:, :K], ref)
    assert not v[:, K:].any()


def test_quantize_rows_at_the_borders(hip_device):
    """Zeros, the largest value on and next to 448 2^c, ties, f32 denormals and the largest f32, inf and NaN."""
    base = torch.zeros(12, 256)
    base[1, 5] = 448.0
    base[2, 5] = 448.0 + 2.0 ** -14
    base[3, :128] = torch.linspace(-448, 448, 128)
    base[4, :128] = (torch.arange(128) + 0.5) / 16 + 1      # ties of several binades
    base[4, 0] = 448.0
    base[5, 0], base[5, 1] = 2.0 ** -140, -2.0 ** -149
    base[6, 0], base[6, 1] = torch.finfo(torch.float32).max, 1.0
    base[7, 3], base[7, 4], base[7, 5] = float("inf"), 2.5, float("-inf")
    base[8, 3], base[8, 130] = float("nan"), 7.0
    base[9] = float("inf")
    base[10, 0], base[10, 1:40] = 448.0, torch.arange(1, 40) * 2.0 ** -10  # e4m3's own denormals
    base[11] = -0.0
    for x in (base, base.to(torch.bfloat16)):
        x = x.to(hip_device)
        q, s = z().fp8_quantize_rows(x)
        v, c = rows_values(q, s, 256)
        ref, cref = O.quantize_rows(x)
        assert torch.equal(c, cref) and same(v, ref)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_rows_views(dtype, hip_device):
    """Row strides and starts off 16 bytes, gathered and scaled rows, indices out of range."""
    big = activations(40, 301, DT[dtype], 5, hip_device)
    for x in (big[:, 1:258], big[::2, :256], big.t()[:, 3:], big[3:4, 2:]):
        q, s = z().fp8_quantize_rows(x)
        ref, cref = O.quantize_rows(x)
        v, c = rows_values(q, s, x.shape[1])
        assert torch.equal(c, cref) and torch.equal(v[:, :x.shape[1]], ref)
    x = big[:, :300]
    slots = torch.randperm(120, generator=gen(3)).to(hip_device)
    w = torch.rand(120, generator=gen(4)).to(hip_device)
    q, s = z().fp8_quantize_rows(x, rows=slots, row_div=3, row_scale=w)
    ref, cref = O.quantize_rows(x.float()[slots // 3] * w[slots].unsqueeze(1))
    v, c = rows_values(q, s, 300)
    assert torch.equal(c, cref) and torch.equal(v[:, :300], ref)
    bad = torch.tensor([0, -1, 119, 120, -120, 1 << 40], device=hip_device)
    q, s = z().fp8_quantize_rows(x, rows=bad, row_div=3, row_scale=w)
    v, _ = rows_values(q, s, 300)
    assert not v[[1, 3, 4, 5]].any() and v[0].any() and v[2].any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("E,N,K", [(1, 1, 1), (2, 128, 128), (3, 130, 257), (1, 510, 1030), (4, 96, 512)])
def test_quantize_weight(E, N, K, dtype, hip_device):
    W = (torch.randn(E, N, K, generator=gen(E * N + K)) * 0.05).to(DT[dtype]).to(hip_device)
    W[0, N // 2, K // 2] = float("nan")
    q, s, qt, st = z().fp8_quantize_weight(W, transposed=True)
    ref, cref = O.quantize_weight(W)
    nb, kb = -(-N // 128), -(-K // 128)

    def values(q, s, rows, cols):
        c = s[..., :-(-cols // 128)].to(torch.int64) - 127
        sc = O.two(c).repeat_interleave(128, 1)[:, :rows].repeat_interleave(128, 2)
        return q.to(torch.float32).double() * sc

    assert torch.equal(s[..., :kb].to(torch.int64) - 127, cref)
    assert torch.equal(st[..., :nb], s[..., :kb].transpose(1, 2))
    assert same(values(q, s, N, K)[..., :K], ref) and same(values(qt, st, K, N)[..., :N], ref.transpose(1, 2))
    assert not values(q, s, N, K)[..., K:].any() and not values(qt, st, K, N)[..., N:].any()
    q2, s2 = z().fp8_quantize_weight(W)
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2[..., :kb], s[..., :kb])


def check(got, ref, S, G, K, half=None):
    assert got.shape == ref.shape and not torch.isnan(got).any()
    half = half or (2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24)
    b = half * ref.abs() + 7 * 2.0 ** -13 * G + 17 * -(-K // 128) * 2.0 ** -23 * S
    err = (got.double() - ref).abs()
    worst = float((err / b.clamp(min=1e-300)).max()) if err.numel() else 0.0
    print(f"  worst |err| / bound {worst:.3f}", flush=True)
    assert worst <= 1.0, worst


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 1536, 2048), (3, 130, 127), (31, 256, 512), (33, 510, 1030),
                                   (200, 264, 640), (257, 1000, 384), (600, 770, 8200), (1025, 512, 128)])
def test_dense_product(M, N, K, out, hip_device):
    x = activations(M, K, torch.bfloat16, M + K, hip_device)
    W = (torch.randn(N, K, generator=gen(N)) * 0.1).to(torch.bfloat16).to(hip_device)
    W *= torch.exp2(torch.randint(-9, 9, (N, 1), generator=gen(1))).to(torch.bfloat16).to(hip_device)
    xr, wr = O.quantize_rows(x)[0], O.quantize_weight(W)[0]
    got = z().fp8_scatter2scatter(*z().fp8_quantize_rows(x), *z().fp8_quantize_weight(W), K, out_dtype=DT[out])
    check(got, *O.product(xr, wr), K)


@pytest.mark.parametrize("T,E,k,N,K,skew", [(1, 8, 2, 256, 256, 0.0), (40, 8, 2, 130, 200, 0.0), (300, 16, 4, 512, 512, 1.2),
                                            (500, 4, 2, 264, 384, 0.5), (1500, 5, 2, 770, 640, 1.5),
                                            (700, 130, 1, 96, 160, 1.0)])
@pytest.mark.parametrize("xg,yg", [(False, True), (True, False), (True, True), (False, False)])
def test_grouped_product(T, E, k, N, K, skew, xg, yg, hip_device):
    idx = random_topk(T, E, k, T + E, skew).to(hip_device)
    se, ss, off, inv = z().flatten_sort_count(idx, E)
    x = activations(T * k if xg else T, K, torch.bfloat16, T, hip_device)
    W = (torch.randn(E, N, K, generator=gen(N)) * 0.1).to(torch.bfloat16).to(hip_device)
    ref = O.grouped_product(O.quantize_rows(x)[0], O.quantize_weight(W)[0], ss, off, k, xg, yg)
    got = z().fp8_scatter2scatter(*z().fp8_quantize_rows(x), *z().fp8_quantize_weight(W), K, ss, off, 1 if xg else k, xg, yg)
    check(got, *ref, K)


def some(n, count, seed):
    """The first and last of n and some others, in order."""
    if n <= count:
        return torch.arange(n)
    mid = torch.randperm(n - 2, generator=gen(seed))[:count - 2] + 1
    return torch.cat([torch.tensor([0, n - 1]), mid]).sort().values


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(8, 4100, 1160), (16, 33, 8300), (17, 1030, 640), (32, 1500, 130), (40, 300, 8400),
                                   (500, 2000, 300), (1000, 1500, 640), (900, 4000, 512), (1100, 5100, 200),
                                   (4200, 2304, 384), (900, 9000, 8330), (1400, 9100, 300), (1400, 9100, 8330),
                                   (4200, 2050, 2100), (2100, 4100, 8330)])
def test_dense_product_tiles(M, N, K, out, hip_device):
    """Sizes for every tile (few rows, launches that fit on the CUs at once, long ones), sampled rows and columns."""
    from zmoe import _lib as L

    x = activations(M, K, torch.bfloat16, M + K, hip_device)
    W = (torch.randn(N, K, generator=gen(N)) * 0.1).to(torch.bfloat16).to(hip_device)
    Y = torch.full((M + 1, N + 3), 7.0, dtype=DT[out], device=hip_device)  # a stride of its own, a row behind
    (xq, xs), (wq, ws) = z().fp8_quantize_rows(x), z().fp8_quantize_weight(W)
    L.call("zmoe_fp8_scatter2scatter", xq.data_ptr(), xs.data_ptr(), M, wq.data_ptr(), ws.data_ptr(), None, None, K, N, 1,
           1, 1, 1, {"f32": L.DTYPE_F32, "bf16": L.DTYPE_BF16}[out], Y.data_ptr(), N + 3,
           torch.cuda.current_stream().cuda_stream)
    assert bool((Y[M] == 7.0).all()) and bool((Y[:, N:] == 7.0).all())
    ri, ci = some(M, 32, 1).to(hip_device), some(N, 96, 2).to(hip_device)
    got = Y[:M, :N][ri][:, ci]
    ref = O.product(O.quantize_rows(x)[0][ri], O.quantize_weight(W)[0][ci])
    check(got, *ref, K)


@pytest.mark.parametrize("T,E,k,N,K", [(700, 40, 1, 1500, 384), (60, 2, 2, 500, 200), (2000, 4, 2, 500, 300),
                                       (2600, 16, 2, 1100, 300), (4300, 4, 1, 770, 2050), (6000, 3, 1, 2304, 2100),
                                       (300, 64, 4, 600, 130), (9000, 8, 1, 1300, 300), (90, 40, 2, 1500, 8330)])
@pytest.mark.parametrize("out", ["bf16", "f32", "half"])
def test_grouped_product_tiles(T, E, k, N, K, out, hip_device):
    """The same by expert, bf16 and f32 rows and f16 ones with their scales (half a step is 2^-11 |y|, and at most 2^-39 of the
    largest of 64 columns: below the bound's S term, whose columns here differ by far less than 2^20)."""
    idx = random_topk(T, E, k, T + E, 0.0).to(hip_device)
    _, ss, off, _ = z().flatten_sort_count(idx, E)
    x = activations(T, K, torch.bfloat16, T, hip_device)
    W = (torch.randn(E, N, K, generator=gen(N)) * 0.1).to(torch.bfloat16).to(hip_device)
    q, w = z().fp8_quantize_rows(x), z().fp8_quantize_weight(W)
    ri, ci = some(T * k, 32, 1).to(hip_device), some(N, 96, 2).to(hip_device)
    slots = ss[ri]
    experts = idx.flatten()[slots]
    xr, wr = O.quantize_rows(x)[0][slots // k], O.quantize_weight(W)[0]
    parts = [O.product(xr[i:i + 1], wr[int(e)][ci]) for i, e in enumerate(experts)]
    ref = [torch.cat([p[j] for p in parts]) for j in range(len(parts[0]))]
    if out == "half":
        y, s = z().fp8_scatter2scatter_half(*q, *w, K, ss, off, k, False, False)
        cols = torch.arange(y.shape[1], device=hip_device)
        v = y.double() * torch.exp2(s.double()[:, cols // 64] - 127)  # (2^c exact in float64)
        check(v[slots][:, ci], *ref, K, half=2.0 ** -11)
    else:
        check(z().fp8_scatter2scatter(*q, *w, K, ss, off, k, False, False, DT[out])[slots][:, ci], *ref, K)


@pytest.mark.parametrize("E,T,empty", [(1, 300, 0.0), (2, 1, 0.0), (63, 40, 0.5), (64, 200, 0.9), (65, 3000, 0.0), (257, 700, 0.3),
                                       (1000, 5000, 0.98), (1024, 9000, 0.0), (1024, 2, 0.0)])
def test_every_expert_count(E, T, empty, hip_device):
    """Tiles are found among up to 1024 experts, many of them without a row (also the first and the last)."""
    N, K = 40, 130
    g = gen(E + T)
    some_e = (torch.rand(E, generator=g) >= empty).nonzero().flatten()
    if empty and len(some_e) > 2:
        some_e = some_e[(some_e != 0) & (some_e != E - 1)]
    idx = some_e[torch.randint(len(some_e), (T, 1), generator=g)].to(hip_device)
    idx[T // 2:] = idx[T // 2].clone()  # half the rows to one of them
    _, ss, off, _ = z().flatten_sort_count(idx, E)
    x = activations(T, K, torch.bfloat16, T, hip_device)
    W = (torch.randn(E, N, K, generator=g) * 0.1).to(torch.bfloat16).to(hip_device)
    q, w = z().fp8_quantize_rows(x), z().fp8_quantize_weight(W)
    got = z().fp8_scatter2scatter(*q, *w, K, ss, off, 1, False, False, torch.float32)
    xr, wr = O.quantize_rows(x)[0], O.quantize_weight(W)[0]
    for e in idx.unique().tolist()[:40] + [int(idx[-1])]:
        rows = (idx[:, 0] == e).nonzero().flatten()
        check(got[rows], *O.product(xr[rows], wr[e]), K)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_weight_views_and_values_not_finite(dtype, hip_device):
    """Rows that start on 16, 4 and 2 (or 4) bytes give the same bytes; inf and NaN become NaN beside the finite values."""
    E, N, K = 2, 140, 262
    base = (torch.randn(E, N, 300, generator=gen(3)) * 0.05).to(DT[dtype]).to(hip_device)
    base[0, 3, 20], base[1, 139, 140], base[1, 0, 130] = float("inf"), float("-inf"), float("nan")
    for at in (0, 2, 1):
        view = base[:, :, at:at + K]
        ref = z().fp8_quantize_weight(view.contiguous(), transposed=True)
        for a, b in zip(z().fp8_quantize_weight(view, transposed=True)[::2], ref[::2]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        q = ref[0].float()[..., :K]
        assert torch.equal(torch.isnan(q), ~torch.isfinite(view.float()))
        assert torch.equal(torch.isnan(ref[2].float()[..., :N]), ~torch.isfinite(view.float()).transpose(1, 2))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 8), (1, 1536, 2048), (3, 130, 136), (16, 40, 4104), (16, 1000, 1000), (5, 70, 16392),
                                   (9, 33, 512)])
def test_few_rows_quantised_in_the_product(M, N, K, dtype, hip_device):
    """The same, bit for bit, as quantising first: also rows with a stride, values that are not finite, zero blocks."""
    base = activations(M, K + 24, torch.float32, M + K, hip_device).to(DT[dtype])
    x = base[:, 8:8 + K]
    x[M // 2, K // 2], x[M - 1, :8] = float("nan"), 0.0
    if M > 2:
        x[1, K - 1], x[0] = float("-inf"), 0.0
    wq, ws = z().fp8_quantize_weight((torch.randn(N, K, generator=gen(N)) * 0.1).to(DT[dtype]).to(hip_device))
    got = z().fp8_linear(x, wq, ws)
    q, s = z().fp8_quantize_rows(x)
    assert same(got, z().fp8_scatter2scatter(q, s, wq, ws, K, out_dtype=DT[dtype]))
    ok = torch.isfinite(x.float()).all(1)
    assert torch.isnan(got[~ok]).all() and not torch.isnan(got[ok]).any()
    odd = base[:, 7:7 + K]  # off 16 bytes: quantised first
    assert same(z().fp8_linear(odd, wq, ws), z().fp8_linear(odd.clone(), wq, ws))


def test_dense_rows_past_two_gib(hip_device):
    """Rows in order have no limit on their span (gathered ones have); the last ones are right too."""
    M, N, K = 1100000, 40, 2048
    x = torch.empty(M, K, dtype=torch.bfloat16, device=hip_device).normal_(generator=torch.Generator(hip_device).manual_seed(1))
    w = z().fp8_quantize_weight((torch.randn(N, K, generator=gen(2)) * 0.05).to(hip_device))
    xq, xs = z().fp8_quantize_rows(x)
    y = z().fp8_scatter2scatter(xq, xs, *w, K)
    for rows in (slice(0, 40), slice(M // 2, M // 2 + 40), slice(M - 40, M)):
        a, wr = O.quantize_rows(x[rows])[0], rows_values(w[0], w[1].repeat_interleave(128, 0)[:N], K)[0]
        check(y[rows], *O.product(a, wr), K)
    ss, off = torch.arange(M, device=hip_device), torch.tensor([M], device=hip_device)
    with pytest.raises(Exception, match="2 GiB"):
        z().fp8_scatter2scatter(xq, xs, w[0][None], w[1][None], K, ss, off, 1, False, True)
