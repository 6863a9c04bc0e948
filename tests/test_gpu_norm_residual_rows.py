"""norm_residual where rows are none, many, too many for one launch or not finite, and a gate that broadcasts over them, by
the bounds of test_gpu_norm_residual."""

import pytest
import torch

from helpers import gen
from oracle import norm_residual_oracle as O
from test_gpu_norm_residual import EPS, check, close, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 2048, 4100, 8200, 16384])
def test_no_rows_give_zero_gradients(d, hip_device):
    """From a workspace full of NaN: what the sums over rows start from is the kernel's to write."""
    from zmoe import _lib as L

    lib, dev = L.load(), hip_device
    nbytes = lib.zmoe_norm_residual_backward_workspace_bytes(0, d)
    ws = torch.full((nbytes // 4,), float("nan"), device=dev)
    w1, w2, gate = (torch.ones(d, device=dev) for _ in range(3))
    scale = torch.ones(1, device=dev)
    dw1, dw2, dg, ds = (torch.full_like(t, float("nan")) for t in (w1, w2, gate, scale))
    p = lambda t: t.data_ptr()  # noqa: E731
    L.call("zmoe_norm_residual_backward", None, None, None, d, L.DTYPE_F32, None, d, L.DTYPE_F32, 0, d, p(w1), p(w2),
           L.DTYPE_F32, p(gate), 1, 0, L.DTYPE_F32, p(scale), 1.0, None, None, None, None, p(dw1), p(dw2), p(dg), p(ds),
           p(ws), nbytes, torch.cuda.current_stream().cuda_stream)
    for g in (dw1, dw2, dg, ds):
        assert (g == 0).all()
    t = make(0, d, "bf16", "bf16", "channel", True, True, True, dev)
    r, x, g = run(t)
    assert r.shape == x.shape == (0, d) and all((g[n] == 0).all() for n in ("w_post", "w_next", "gate", "scale"))


@pytest.mark.parametrize("gate", ["row", "full"])
def test_rows_past_one_launch(gate, hip_device):
    """2^26 rows and some of 64 threads each are 2^32 threads: the rows of a call on all of them are those of calls on
    parts."""
    from zmoe import ops

    n, d = (1 << 26) + 300, 4
    g = torch.Generator(device=hip_device).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device=hip_device, dtype=torch.bfloat16)  # noqa: E731
    r, y, w = rnd(n, d), rnd(n, d), rnd(d)
    kind = ops.GATE_ROW if gate == "row" else ops.GATE_FULL
    gt = rnd(n) if gate == "row" else rnd(n, d)
    whole = ops.norm_residual(r, y, w, w, gt, kind, None, 0.5, 1e-6)
    for lo, hi in ((0, n // 2), (n // 2, n)):
        part = ops.norm_residual(r[lo:hi], y[lo:hi], w, w, gt[lo:hi], kind, None, 0.5, 1e-6)
        assert all(torch.equal(a[lo:hi], b) for a, b in zip(whole, part))


@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("d", [96, 2048, 7168, 8200])
def test_residual_not_finite_and_no_grad_through_x(d, gate, hip_device):
    """Without a next norm, or with x unused, r' takes no part in its own gradient: what is finite by the formula stays
    finite where the residual is not."""
    for nxt in (False, True):
        t = make(5, d, "f32", "bf16", gate, True, nxt, False, hip_device)
        t["r"][1, 3], t["r"][2, 5], t["r"][3, 7] = float("inf"), -float("inf"), float("nan")
        _, _, g = run(t, use_dx=False)
        val, mag = O.backward(t["r"], t["y"], t["w_post"], None, t["gate"], 1.0, EPS, t["dr"], None)
        for name in ("r", "y", "w_post", "gate"):
            if name in g:
                rows = name == "w_post" or (name == "gate" and gate == "channel")
                close("d " + name, g[name], val[name].reshape(g[name].shape), mag[name].reshape(g[name].shape),
                      512 + (5 if rows else 0))
        assert not nxt or (g["w_next"] == 0).all()


@pytest.mark.parametrize("d", [96, 2048, 7168, 8200])
def test_rows_not_finite_without_their_norm(d, hip_device):
    """The same of y where it has no norm: dy = gate dr'."""
    for gate in ("none", "channel", "row", "full"):
        t = make(5, d, "f32", "bf16", gate, False, True, False, hip_device)
        t["y"][1, 3], t["y"][2, 5] = float("inf"), float("nan")
        _, _, g = run(t, use_dx=False)
        val, mag = O.backward(t["r"], t["y"], None, None, t["gate"], 1.0, EPS, t["dr"], None)
        for name in ("r", "y"):
            close("d " + name, g[name], val[name], mag[name], 512)
        assert (g["w_next"] == 0).all()


def test_gradient_of_a_gate_that_broadcasts(hip_device):
    """One gate a sequence, bf16: its gradient is rounded once, after the sum over the rows."""
    from zmoe.functional import norm_residual

    B, S, d = 3, 50, 264
    t = make(B * S, d, "bf16", "bf16", "none", True, True, False, hip_device)
    gate = torch.randn(B, 1, d, generator=gen(9)).to(torch.bfloat16).to(hip_device).requires_grad_(True)
    r, x = norm_residual(t["r"].view(B, S, d), t["y"].view(B, S, d), t["w_post"], t["w_next"], gate, None, EPS)
    torch.autograd.backward([r, x], [t["dr"].view(B, S, d), t["dx"].view(B, S, d)])
    full = gate.detach().expand(B, S, d).reshape(-1, d)
    val, mag = O.backward(t["r"], t["y"], t["w_post"], t["w_next"], full, 1.0, EPS, t["dr"], t["dx"])
    fold = lambda v: v.view(B, S, d).sum(1, keepdim=True)  # noqa: E731
    assert gate.grad.dtype == gate.dtype
    close("d gate", gate.grad, fold(val["gate"]), fold(mag["gate"]), 512 + S)


@pytest.mark.parametrize("n,d", [(2600, 200), (2100, 1024), (1030, 2048), (600, 4096), (520, 7168), (600, 8200), (520, 16384)])
@pytest.mark.parametrize("gate,post,nxt,use_dr,use_dx", [
    ("none", True, True, True, True), ("row", True, True, True, True), ("full", True, True, True, True),
    ("channel", True, False, True, True), ("row", False, True, True, True), ("full", False, True, True, True),
    ("none", False, True, True, True), ("none", True, True, True, False), ("channel", False, True, True, False),
    ("row", True, True, False, True)])
def test_blocks_of_many_rows(n, d, gate, post, nxt, use_dr, use_dx, hip_device):
    """More rows than the backward has blocks, in every form of a row's sums: one of the two, both, neither."""
    check(make(n, d, "bf16" if n % 200 else "f32", "bf16", gate, post, nxt, gate != "none", hip_device), use_dr, use_dx)
