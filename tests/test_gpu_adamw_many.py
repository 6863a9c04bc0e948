"""zmoe.adamw.AdamW over more tensors than a launch's arguments hold, in every width and type: bit for bit what one call for each
tensor makes of the same clip."""

import pytest
import torch

from helpers import gen

pytestmark = pytest.mark.gpu

SIZES = [i % 9 * 130 + i % 4 for i in range(120)]  # empty ones, ends of blocks, starts off whole vectors


def tensors(dt, dev, seed, std=1.0):
    return [(torch.randn(n, generator=gen(seed + 7 * i)) * std).to(dt).to(dev) for i, n in enumerate(SIZES)]


@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("types", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("bits", [32, 8])
def test_many_are_one_by_one(bits, types, clip, hip_device):
    from zmoe import ops
    from zmoe.adamw import AdamW

    params = [p.requires_grad_(True) for dt in types for p in tensors(dt, hip_device, 1)]
    opt = AdamW(params, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1, state_bits=bits, max_grad_norm=clip)
    m, v = {32: (torch.float32,) * 2, 8: (torch.int8, torch.uint8)}[bits]
    alone = []
    for p in params:
        blocks = -(-p.numel() // 256)
        scales = [torch.zeros(blocks, device=hip_device) for _ in range(2)] if bits == 8 else []
        alone.append(([p.detach().clone()], [torch.zeros_like(p, dtype=m)], [torch.zeros_like(p, dtype=v)],
                      [[s] for s in scales] or [[], []], [torch.zeros((), device=hip_device)]))
    for t in range(3):
        grads = [g for dt in types for g in tensors(dt, hip_device, 1000 * t + 3, 0.1)]
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()
        factor = None if clip is None else ops.grad_norm(grads, clip)[1]
        for (p, a, b, s, n), g in zip(alone, grads):
            ops.adamw_(p, [g], a, b, *s, n, bits, 1e-2, 0.9, 0.95, 1e-8, 0.1, factor)
    values = opt.moments()
    for p, (q, a, b, s, n), (x, y) in zip(params, alone, values):
        st = opt.state[p]
        assert torch.equal(p, q[0]) and torch.equal(st["exp_avg"], a[0]) and torch.equal(st["exp_avg_sq"], b[0])
        assert torch.equal(st["step"], n[0]) and float(n[0]) == 3.0
        if bits == 8:
            assert torch.equal(st["exp_avg_scale"], s[0][0]) and torch.equal(st["exp_avg_sq_scale"], s[1][0])
            a, b = (ops.adamw_moments([c], [z[0]], [w])[0] for c, z, w in ((a[0], s[0], False), (b[0], s[1], True)))
            assert torch.equal(x, a) and torch.equal(y, b)  # (240 or 480 moments in one call, one in each of these)
        else:
            assert x is st["exp_avg"] and y is st["exp_avg_sq"]
