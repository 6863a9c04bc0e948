"""e4m3 calls past what one launch holds, and past what is added at float32's precision."""

import pytest
import torch

from helpers import gen, random_topk
from oracle import fp8_oracle as O
from test_gpu_fp8 import activations

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("listed", [False, True])
def test_rows_past_one_launch(listed, hip_device):
    """2^28 blocks and some of 16 threads each are 2^32 threads: every scale is that of its row's value, and the values
    around the border and at both ends those of calls on these rows."""
    from zmoe import ops

    n = (1 << 28) + 200
    g = torch.Generator(device=hip_device).manual_seed(4)
    x = torch.randn(n, 1, generator=g, device=hip_device, dtype=torch.bfloat16)
    rows = torch.arange(n - 1, -1, -1, device=hip_device) if listed else None
    scale = torch.rand(n, generator=g, device=hip_device) + 0.5
    q, s = ops.fp8_quantize_rows(x, rows, 1, scale)
    assert q.shape == (n, 128) and s.shape == (n, 4)
    for i0 in range(0, n, 1 << 26):
        i1 = min(n, i0 + (1 << 26))
        v = (x[:, 0].float() * scale).flip(0)[i0:i1] if listed else x[i0:i1, 0].float() * scale[i0:i1]
        bits = v.abs().view(torch.int32)  # |v| = 1.m 2^e <= 448 2^c
        code = (bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000).to(torch.int32)
        assert torch.equal(s[i0:i1, 0].to(torch.int32), code.clamp(min=0))
    for lo in (0, (1 << 28) - 100, n - 100):
        part = slice(lo, lo + 100)
        ref = ops.fp8_quantize_rows(x, rows[part], 1, scale)[0] if listed else ops.fp8_quantize_rows(x[part], None, 1, scale[part])[0]
        assert torch.equal(q[part].view(torch.uint8), ref.view(torch.uint8))


def bounds(x, w, d):
    """x w^T and how far the scaled matrix instruction's sums may be from it (test_gpu_fp8)."""
    v, S, G = O.product(x, w)
    return v, 7 * 2.0 ** -13 * G + 17 * -(-d // 128) * 2.0 ** -23 * S


@pytest.mark.parametrize("T,d,f,E,k", [(2100, 512, 1000, 1, 1), (1400, 512, 768, 32, 2), (700, 1000, 1500, 16, 2)])
def test_single_rows_past_the_exact_sums(T, d, f, E, k, hip_device):
    """Just above 2^21 activations, where the scaled matrix instruction adds: every activation, also of an expert's only row,
    is the e4m3 rounding, at its block's scale, of a value within D of the exact one (D as in test_gpu_fp8_layers'
    swiglu_check), so next to a border its neighbour at most. In a launch of its own, below 2^21, the same row's
    sums are f32's, and the same holds with 17 ceil(d / 128) 2^-23 S for each product's bound."""
    from zmoe import ops

    assert 1 << 21 < T * k * f < (1 << 21) * 1.03
    idx = random_topk(T, max(E - 1, 1), k, 5).to(hip_device)  # the last expert has one row
    if E > 1:
        idx[9, k - 1] = E - 1
    x = activations(T, d, torch.bfloat16, 6, hip_device)
    W1 = (torch.randn(2 * E, f, d, generator=gen(7)) * d ** -0.5).to(torch.bfloat16).to(hip_device)
    w = ops.fp8_quantize_weight(W1)
    wr, xr = O.quantize_weight(W1)[0], O.quantize_rows(x)[0]
    few = torch.tensor([0, 9, T - 1], device=hip_device)

    def run(tokens):
        _, ss, off, _ = ops.flatten_sort_count(idx[tokens], E)
        aq, as_ = ops.fp8_glu_w1_forward(*ops.fp8_quantize_rows(x[tokens]), *w, d, ss, off, k)
        out = torch.empty_like(aq, dtype=torch.float32), torch.empty_like(as_, dtype=torch.int64)
        out[0][ss], out[1][ss] = aq.float(), as_.long() - 127
        return out

    q, c = run(torch.arange(T, device=hip_device))
    alone = [run(few[i:i + 1]) for i in range(len(few))]
    for i, t in enumerate(few.tolist()):
        for j in range(k):
            e = int(idx[t, j])
            (u, eu), (g, eg) = bounds(xr[t:t + 1], wr[2 * e], d), bounds(xr[t:t + 1], wr[2 * e + 1], d)
            silu = g * torch.sigmoid(g)
            a = (silu * u)[0]
            for (qr, cr), exact in (((q[t * k + j], c[t * k + j]), False), ((alone[i][0][j], alone[i][1][j]), True)):
                if exact:
                    eu, eg = (17 * -(-d // 128) * 2.0 ** -23 * O.product(xr[t:t + 1], wr[2 * e + h])[1] for h in (0, 1))
                D = (silu.abs() * eu + 1.1 * (u.abs() + eu) * eg)[0] + 2.0 ** -18 * a.abs()
                for b in range(-(-f // 128)):
                    s = slice(128 * b, min(f, 128 * b + 128))
                    lo, hi = (O.scale_exponent(((a[s].abs() + sign * D[s]).clamp(min=0)).amax().view(1)) for sign in (-1, 1))
                    assert lo <= cr[b] <= hi
                    at = lambda v: O.e4m3((v * O.two(-cr[b])).clamp(-448, 448))  # noqa: E731
                    got = qr[s].double()
                    assert ((at(a[s] - D[s]) <= got) & (got <= at(a[s] + D[s]))).all(), (t, j, b, exact)
