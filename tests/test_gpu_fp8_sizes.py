"""e4m3 calls past what one launch holds."""

import pytest
import torch

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
