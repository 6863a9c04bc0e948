"""Calls of the 8-bit products and of the norm around a block, as cases that can be timed and compared.

A case is a dict of plain values; ``kind`` names the public entry point it goes through:

* ``linear``   ``zmoe.functional.fp8_linear``: a dense product in e4m3 with a power-of-two scale for each block of
  128. Serving cases hold a weight that was quantised once, training cases a bf16 or fp32 weight that is
  quantised in the call, and return the gradients too.
* ``experts``  ``scattermoe.mlp.GLUMLP.quantize_fp8()``: the SwiGLU experts' products in e4m3 on given routing.
* ``grouped``  ``scattermoe.parallel_experts.parallel_linear(..., fp8=True)``: one grouped product, forward and
  backward, as an expert MLP's first: tokens' rows gathered, output rows sorted by expert.
* ``norm``     ``zmoe.functional.norm_residual``: the norm after a block, its gate, the scaled residual and the next
  block's norm.

Dimensions: T (tokens or rows), d (hidden), E (routed experts), k (experts per token), f (expert width), K and N
(a product's depth and columns). Widths are those of the package's tests and benchmark.

With ``own`` false, ``run`` computes the same from elementary torch operations in 32 bits; ``exact`` is the
definition in 64 bits.
"""

import math
import os
import sys

import torch

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = os.path.join(_ROOT, "architecture-zarelga-superposition_amd")

own = False

_BF16, _F32, _F64 = torch.bfloat16, torch.float32, torch.float64
_EPS = 1e-6


def _package():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)


# ------------------------------------------------------------------ the cases
def _linear(T, K, N, train, weight="bf16"):
    return {"kind": "linear", "T": T, "K": K, "N": N, "train": train, "weight": weight}


def _experts(T, d, E, k, f, skew):
    return {"kind": "experts", "T": T, "d": d, "E": E, "k": k, "f": f, "skew": skew}


def _grouped(T, K, N, E, k, skew):
    return {"kind": "grouped", "T": T, "K": K, "N": N, "E": E, "k": k, "skew": skew}


def _norm(T, d, stream, gate, post, nxt, scale, train):
    return {"kind": "norm", "T": T, "d": d, "stream": stream, "gate": gate, "post": post, "next": nxt,
            "scale": scale, "train": train}


def listed():
    cases = {
        # one decoding token through one projection: latency
        "linear_decode_1": _linear(1, 2048, 1536, False),
        # a training step of a narrow projection, ragged rows, a depth that is no whole number of blocks
        "linear_train_4097": _linear(4097, 1000, 1528, True, "f32"),
        # a long prompt through a wide projection
        "linear_prefill_8192": _linear(8192, 7168, 4096, False),
        # one decoding step of four sequences: some 30 experts' weights streamed
        "experts_decode_4": _experts(4, 2048, 128, 8, 768, 0.0),
        # a decoding batch with speculative tokens, or a short chunk of a prompt
        "experts_chunk_509": _experts(509, 2048, 128, 8, 768, 0.0),
        # the tokens of the package's benchmark as one prefill
        "experts_prefill_32768": _experts(32768, 2048, 128, 8, 768, 0.0),
        # a quarter (expert-parallel share) of 256 experts of a 7168-wide model, skewed routing
        "experts_skewed_8192": _experts(8192, 7168, 64, 2, 2048, 1.1),
        # a training step of one grouped product at widths that are not whole 16-byte chunks
        "grouped_train_4001": _grouped(4001, 510, 1030, 16, 2, 0.3),
        # the same at the benchmark's widths
        "grouped_train_16384": _grouped(16384, 2048, 1536, 64, 4, 0.0),
        # one decoding step of three sequences between two sublayers: latency
        "norm_decode_3": _norm(3, 2048, "bf16", "channel", True, True, False, False),
        # a training step, bf16 residual stream, a gate for each channel
        "norm_train_16383": _norm(16383, 2048, "bf16", "channel", True, True, False, True),
        # a wide model with an fp32 residual stream, a gate for each token and a learned residual scale
        "norm_train_4095": _norm(4095, 7168, "f32", "row", True, True, True, True),
    }
    return [dict(c, name=name) for name, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_WIDTHS = [(512, 32, 2, 160), (1024, 64, 8, 512), (2048, 128, 8, 768), (2048, 64, 4, 1024), (7168, 32, 2, 2048)]
_MOST_FLOPS = 2.4e12  # a drawn case costs no more than experts_prefill_32768


def draw(rng):
    """One more case of the listed ones' ranges."""
    case = _draw(rng)
    while work(case)["flops"] > _MOST_FLOPS:
        case["T"] = case["T"] // 2 + 1
    return case


def _draw(rng):
    kind = rng.choice(["linear", "linear", "experts", "experts", "grouped", "norm", "norm"])
    skew = round(rng.uniform(0.0, 1.2), 2)
    if kind == "linear":
        train = rng.random() < 0.5
        K, N = _log(rng, 250, 7168), _log(rng, 250, 7168)
        if rng.random() < 0.7:  # most widths are whole 16-byte chunks
            K, N = K // 8 * 8, N // 8 * 8
        return _linear(_log(rng, 64 if train else 1, 16384), K, N, train, rng.choice(["bf16", "f32"]))
    if kind == "experts":
        d, E, k, f = rng.choice(_WIDTHS)
        return _experts(_log(rng, 1, 32768), d, E, k, f, skew)
    if kind == "grouped":
        K, N = rng.randrange(250, 2060), rng.randrange(250, 2060)
        if rng.random() < 0.5:
            K, N = K // 8 * 8, N // 8 * 8
        return _grouped(_log(rng, 64, 16384), K, N, rng.choice([8, 16, 64]), rng.choice([1, 2, 4]), skew)
    d = rng.choice([510, 512, 1024, 2048, 4096, 7168])
    post, nxt = rng.choice([(True, True), (True, True), (True, False), (False, True)])
    return _norm(_log(rng, 1, 32768 if d <= 2048 else 8192), d, rng.choice(["bf16", "f32"]),
                 rng.choice(["none", "channel", "row", "full"]), post, nxt, rng.random() < 0.5, rng.random() < 0.6)


# ------------------------------------------------------------------ inputs, from the seed alone
def _rand(seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=_F32):
        return torch.randn(*shape, device=dev, generator=g, dtype=dtype).mul_(std)

    return g, normal


def _activations(normal, T, d):
    """Rows as a model has them: unit scale, some channels far above the others."""
    x = normal(T, d)
    x *= torch.exp(normal(d, std=0.7))
    return x.to(_BF16)


def _routing(case, g):
    """k distinct experts a token, drawn by popularity rank ** -skew (Gumbel top-k over a random
    ranking), and L1-normalised weights, as a sigmoid router gives them."""
    T, E, k = case["T"], case["E"], case["k"]
    dev = torch.device("cuda")
    rank = torch.randperm(E, device=dev, generator=g).add_(1).float()
    u = torch.rand(T, E, device=dev, generator=g).clamp_(1e-9, 1 - 1e-7)
    idx = torch.topk(-torch.log(-torch.log(u)) - case["skew"] * torch.log(rank), k, dim=-1).indices
    p = torch.rand(T, k, device=dev, generator=g) * 0.5 + 0.4
    return idx, p / p.sum(-1, keepdim=True)


def _inputs(case, seed):
    g, normal = _rand(seed)
    kind, T = case["kind"], case["T"]
    if kind == "linear":
        K, N = case["K"], case["N"]
        t = {"x": _activations(normal, T, K),
             "W": normal(N, K, std=K ** -0.5, dtype=_F32 if case["weight"] == "f32" else _BF16)}
        if case["train"]:
            t["dout"] = normal(T, N, dtype=_BF16)
        return t
    if kind == "experts":
        d, E, f = case["d"], case["E"], case["f"]
        t = {"x": _activations(normal, T, d), "W1": normal(E, 2 * f, d, std=d ** -0.5, dtype=_BF16),
             "W2": normal(E, d, f, std=f ** -0.5, dtype=_BF16)}
        t["idx"], t["p"] = _routing(case, g)
        return t
    if kind == "grouped":
        K, N, E = case["K"], case["N"], case["E"]
        t = {"x": _activations(normal, T, K), "W": normal(E, N, K, std=K ** -0.5, dtype=_BF16),
             "dout": normal(T * case["k"], N, dtype=_BF16)}
        t["idx"], _ = _routing(case, g)
        return t
    d = case["d"]
    stream = _F32 if case["stream"] == "f32" else _BF16
    t = {"r": normal(T, d, std=2.0, dtype=stream), "y": normal(T, d, std=0.5, dtype=_BF16)}
    if case["post"]:
        t["w1"] = normal(d, std=0.1, dtype=_BF16)
    if case["next"]:
        t["w2"] = normal(d, std=0.1, dtype=_BF16)
    shape = {"none": None, "channel": (d,), "row": (T, 1), "full": (T, d)}[case["gate"]]
    if shape is not None:
        t["gate"] = normal(*shape, std=0.5, dtype=_BF16)
    if case["scale"]:
        t["scale"] = torch.full((1,), 0.9, device="cuda") + normal(1, std=0.05)
    if case["train"]:
        t["dr"] = normal(T, d, dtype=stream)
        if case["next"]:
            t["dx"] = normal(T, d, dtype=_BF16)
    return t


def prepare(case, seed):
    """Inputs, and what a serving or training program keeps: a served weight quantised once, modules."""
    t = _inputs(case, seed)
    s = {"case": case, "own": own}
    serving = case["kind"] == "experts" or (case["kind"] == "linear" and not case["train"])
    if own:
        _package()
        if case["kind"] == "linear" and serving:
            from zmoe import fp8

            t["W"] = fp8.quantize_weight(t["W"])
        elif case["kind"] == "experts":
            from scattermoe.mlp import GLUMLP

            with torch.device("meta"):
                m = GLUMLP(case["d"], case["f"], case["E"], case["k"])
            m.load_state_dict({"experts.weight": t.pop("W1"), "output_experts.weight": t.pop("W2")}, assign=True)
            s["module"] = m.quantize_fp8()
    elif serving:
        # the values that the served weights stand for
        if case["kind"] == "linear":
            t["W"] = _dequantized_blocks(t["W"])
        else:
            E, f, d = case["E"], case["f"], case["d"]
            t["W1"] = _dequantized_blocks(t["W1"].view(2 * E, f, d)).view(E, 2 * f, d)
            t["W2"] = _dequantized_blocks(t["W2"])
    if case.get("train", case["kind"] == "grouped") and own:
        for n in ("x", "W", "r", "y", "w1", "w2", "gate", "scale"):
            if n in t:
                t[n].requires_grad_(True)
    s.update(t)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if s["own"] else _run_plain(s)


def _run_own(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "linear":
        from zmoe.functional import fp8_linear

        if not case["train"]:
            with torch.no_grad():
                return {"out": fp8_linear(s["x"], s["W"])}
        s["x"].grad = s["W"].grad = None
        out = fp8_linear(s["x"], s["W"])
        out.backward(s["dout"])
        return {"out": out.detach(), "d x": s["x"].grad, "d W": s["W"].grad}
    if kind == "experts":
        with torch.no_grad():
            return {"out": s["module"](s["x"], s["p"], s["idx"])}
    if kind == "grouped":
        from scattermoe.parallel_experts import flatten_sort_count, parallel_linear

        s["x"].grad = s["W"].grad = None
        se, ss, off = flatten_sort_count(s["idx"], case["E"])
        out = parallel_linear(s["x"], s["W"].permute(0, 2, 1), case["k"], se, ss, off, grouped_out=True, fp8=True)
        out.backward(s["dout"])
        return {"out": out.detach(), "d x": s["x"].grad, "d W": s["W"].grad}
    from zmoe.functional import norm_residual

    leaves = [n for n in ("r", "y", "w1", "w2", "gate", "scale") if n in s]
    args = dict(weight=s.get("w1"), next_weight=s.get("w2"), gate=s.get("gate"), residual_scale=s.get("scale"),
                eps=_EPS)
    if not case["train"]:
        with torch.no_grad():
            r, x = norm_residual(s["r"], s["y"], **args)
        return {"r": r} if x is None else {"r": r, "x": x}
    for n in leaves:
        s[n].grad = None
    r, x = norm_residual(s["r"], s["y"], **args)
    if x is None:
        r.backward(s["dr"])
        got = {"r": r.detach()}
    else:
        torch.autograd.backward([r, x], [s["dr"], s["dx"]])
        got = {"r": r.detach(), "x": x.detach()}
    got.update({"d " + n: s[n].grad for n in leaves})
    return got


# ------------------------------------------------------------------ the plain form, in 32 bits
def _e4m3(v, amax):
    """The values that v (blocks along its dims, their largest magnitudes amax) stands for in e4m3."""
    bits = amax.view(torch.int32)  # amax = 1.m 2^e; 448 = 1.75 * 2^8
    e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000).to(torch.int32)
    s = (e.clamp_(min=-126) + 127 << 23).view(_F32)
    return (v / s).to(torch.float8_e4m3fn).to(_F32) * s


def _quantized_rows(x):
    """Blocks of 128 along the last dim (a shorter last one)."""
    x = x.to(_F32)
    T, K = x.shape
    pad = -K % 128
    v = torch.nn.functional.pad(x, (0, pad)).view(T, -1, 128)
    return _e4m3(v, v.abs().amax(-1, keepdim=True)).view(T, K + pad)[:, :K]


def _dequantized_blocks(W):
    """Blocks of 128 x 128 of the last two dims (shorter ones at the edges), stack by stack."""
    lead, (N, K) = W.shape[:-2], W.shape[-2:]
    out = []
    for w in W.reshape(-1, N, K):
        v = torch.nn.functional.pad(w.to(_F32), (0, -K % 128, 0, -N % 128))
        n, kk = v.shape
        v = v.view(n // 128, 128, kk // 128, 128)
        out.append(_e4m3(v, v.abs().amax((1, 3), keepdim=True)).view(n, kk)[:N, :K])
    return torch.stack(out).view(*lead, N, K)


def _by_expert(idx, E):
    """Slots (t k + j) of each expert, in slot order."""
    order = torch.sort(idx.reshape(-1), stable=True).indices
    return torch.split(order, torch.bincount(idx.reshape(-1), minlength=E).tolist())


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "linear":
        x = _quantized_rows(s["x"])
        if not case["train"]:
            return {"out": (x @ s["W"].T).to(_BF16)}
        W = _dequantized_blocks(s["W"])
        dout = s["dout"].to(_F32)
        return {"out": (x @ W.T).to(_BF16), "d x": (_quantized_rows(s["dout"]) @ W).to(_BF16),
                "d W": (dout.T @ s["x"].to(_F32)).to(s["W"].dtype)}
    if kind in ("experts", "grouped"):
        T, k = s["idx"].shape
        x = _quantized_rows(s["x"])
        slots = _by_expert(s["idx"], case["E"])
    if kind == "experts":
        f, p = case["f"], s["p"].reshape(-1)
        Y = torch.empty(T * k, case["d"], device=x.device)
        for e, sl in enumerate(slots):
            if sl.numel():
                h = x[sl // k] @ s["W1"][e].T
                a = h[:, f:] / (1 + torch.exp(-h[:, f:])) * h[:, :f]
                Y[sl] = _quantized_rows(a) @ s["W2"][e].T
        return {"out": (Y * p.unsqueeze(1)).view(T, k, -1).sum(1).to(_BF16)}
    if kind == "grouped":
        W = _dequantized_blocks(s["W"])
        dout = s["dout"].to(_F32)
        dq, xf = _quantized_rows(s["dout"]), s["x"].to(_F32)
        out, dX = torch.empty_like(dout), torch.empty(T * k, case["K"], device=x.device)
        dW = torch.zeros_like(W)
        at = 0
        for e, sl in enumerate(slots):
            if sl.numel():
                rows = slice(at, at + sl.numel())
                out[rows] = x[sl // k] @ W[e].T
                dX[sl] = dq[rows] @ W[e]
                dW[e] = dout[rows].T @ xf[sl // k]
                at += sl.numel()
        return {"out": out.to(_BF16), "d x": dX.view(T, k, -1).sum(1).to(_BF16), "d W": dW.to(_BF16)}
    return _norm_plain(s)


def _norm_plain(s):
    case, d = s["case"], s["case"]["d"]
    f32 = {n: s[n].to(_F32) for n in ("r", "y", "w1", "w2", "gate", "scale", "dr", "dx") if n in s}
    r, y = f32["r"], f32["y"]
    u = y
    if case["post"]:
        rho1 = torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS)
        u = y * rho1 * (1 + f32["w1"])
    gate = f32.get("gate")
    gu = u if gate is None else gate * u
    h = (r * f32["scale"] if case["scale"] else r) + gu
    got = {"r": h.to(s["r"].dtype)}
    if case["next"]:
        rho2 = torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS)
        got["x"] = (h * rho2 * (1 + f32["w2"])).to(_BF16)
    if not case["train"]:
        return got
    t = f32["dr"]
    if case["next"]:
        gx = f32["dx"] * (1 + f32["w2"])
        t = t + rho2 * gx - h * (rho2 ** 3 / d) * (gx * h).sum(-1, keepdim=True)
        dw2 = (f32["dx"] * h * rho2).sum(0)
    du = t if gate is None else gate * t
    dy = du
    if case["post"]:
        gu = du * (1 + f32["w1"])
        dy = rho1 * gu - y * (rho1 ** 3 / d) * (gu * y).sum(-1, keepdim=True)
        dw1 = (du * y * rho1).sum(0)
    got["d r"] = (t * f32["scale"] if case["scale"] else t).to(s["r"].dtype)
    got["d y"] = dy.to(_BF16)
    if case["post"]:
        got["d w1"] = dw1.to(_BF16)
    if case["next"]:
        got["d w2"] = dw2.to(_BF16)
    if gate is not None:
        dg = t * u
        dg = {"channel": lambda: dg.sum(0), "row": lambda: dg.sum(-1, keepdim=True), "full": lambda: dg}[case["gate"]]()
        got["d gate"] = dg.to(_BF16)
    if case["scale"]:
        got["d scale"] = (t * r).sum().view(1)
    return got


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, T = case["kind"], case["T"]
    if kind == "linear":
        K, N = case["K"], case["N"]
        if not case["train"]:
            return {"bytes": 2 * T * K + N * K + 2 * T * N, "flops": 2 * T * K * N}
        w = 4 if case["weight"] == "f32" else 2
        return {"bytes": 4 * T * K + 2 * w * N * K + 4 * T * N, "flops": 6 * T * K * N}
    if kind == "experts":
        d, E, f, R = case["d"], case["E"], case["f"], T * case["k"]
        touched = E * (1 - (1 - case["k"] / E) ** T)
        return {"bytes": int(touched * 3 * d * f + 4 * T * d + 12 * R), "flops": 6 * R * d * f}
    if kind == "grouped":
        K, N, E, R = case["K"], case["N"], case["E"], T * case["k"]
        return {"bytes": 4 * T * K + 4 * E * K * N + 4 * R * N + 16 * R, "flops": 6 * R * K * N}
    d = case["d"]
    st = 4 if case["stream"] == "f32" else 2
    full = 2 if case["gate"] == "full" else 0
    fwd = T * d * (2 * st + 2 + full + (2 if case["next"] else 0))
    bwd = T * d * (3 * st + 4 + 2 * full + (2 if case["next"] else 0))
    return {"bytes": fwd + (bwd if case["train"] else 0) + 12 * d, "flops": T * d * (40 if case["train"] else 12)}


# ------------------------------------------------------------------ the definition, in 64 bits
def _two64(c):
    """2^c for whole numbers c, from the bits: a power function need not be exact."""
    return (c.to(torch.int64) + 1023 << 52).view(_F64)


def _floor_log64(a):
    """The whole e with 2^e <= a < 2^(e + 1), for a > 0."""
    e = torch.floor(torch.log2(a))
    e = torch.where(_two64(e) > a, e - 1, e)
    return torch.where(_two64(e + 1) <= a, e + 1, e)


def _grid64(v, c):
    """v 2^-c rounded to e4m3 (3 mantissa bits, exponents from -6, ties to even), times 2^c."""
    v = v * _two64(-c)
    step = _two64(_floor_log64(v.abs().clamp(min=2.0 ** -20)).clamp(min=-6.0) - 3)
    return torch.round(v / step) * step * _two64(c)


def _exponent64(a):
    """The least whole c with a <= 448 * 2^c."""
    a = a.clamp(min=2.0 ** -120)
    c = _floor_log64(a / 448)
    return torch.where(a > 448 * _two64(c), c + 1, c)


def _rows64(x):
    x = x.to(_F64)
    out = torch.empty_like(x)
    for b in range(0, x.shape[1], 128):
        v = x[:, b:b + 128]
        out[:, b:b + 128] = _grid64(v, _exponent64(v.abs().amax(1, keepdim=True)))
    return out


def _weight64(W):
    """One [N, K] weight."""
    W = W.to(_F64)
    N, K = W.shape
    a = W.abs()
    if N % 128:
        a = torch.cat([a, a.new_zeros(-N % 128, K)], 0)
    if K % 128:
        a = torch.cat([a, a.new_zeros(a.shape[0], -K % 128)], 1)
    a = a.unfold(0, 128, 128).unfold(1, 128, 128).flatten(2).amax(-1)
    c = _exponent64(a).repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return _grid64(W, c)


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    if kind == "linear":
        x, W = _rows64(t["x"]), _weight64(t["W"])
        got = {"out": x @ W.T}
        if case["train"]:
            got["d x"] = _rows64(t["dout"]) @ W
            got["d W"] = t["dout"].to(_F64).T @ t["x"].to(_F64)
        return got
    if kind == "norm":
        return _norm64(case, t)
    T, k = t["idx"].shape
    x = _rows64(t["x"])
    if kind == "experts":
        f, p = case["f"], t["p"].to(_F64)
        out = torch.zeros(T, case["d"], dtype=_F64, device=x.device)
        for e in range(case["E"]):
            rows, j = (t["idx"] == e).nonzero(as_tuple=True)
            if rows.numel():
                xe = x[rows]
                up, gt = xe @ _weight64(t["W1"][e, :f]).T, xe @ _weight64(t["W1"][e, f:]).T
                out.index_add_(0, rows, (_rows64(torch.sigmoid(gt) * gt * up) @ _weight64(t["W2"][e]).T)
                               * p[rows, j, None])
        return {"out": out}
    dx = torch.zeros(T, case["K"], dtype=_F64, device=x.device)
    dW = torch.zeros(t["W"].shape, dtype=_F64, device=x.device)
    dout, dq = t["dout"].to(_F64), _rows64(t["dout"])
    out, at = torch.zeros_like(dout), 0
    for e in range(case["E"]):
        rows = (t["idx"] == e).nonzero(as_tuple=True)[0]  # in token order, as the sort leaves them
        end = at + rows.numel()
        if rows.numel():
            W = _weight64(t["W"][e])
            out[at:end] = x[rows] @ W.T
            dx.index_add_(0, rows, dq[at:end] @ W)
            dW[e] = dout[at:end].T @ t["x"][rows].to(_F64)
        at = end
    return {"out": out, "d x": dx, "d W": dW}


def _norm64(case, t):
    """By autograd of the definition."""
    names = [n for n in ("r", "y", "w1", "w2", "gate", "scale") if n in t]
    v = {n: t[n].to(_F64).requires_grad_(case["train"]) for n in names}

    def norm(a, w):
        return a / torch.sqrt((a * a).mean(-1, keepdim=True) + _EPS) * (1 + w)

    u = norm(v["y"], v["w1"]) if case["post"] else v["y"]
    h = v["r"] * v.get("scale", 1.0) + (u * v["gate"] if "gate" in v else u)
    got = {"r": h.detach()}
    outs, grads = [h], [t.get("dr")]
    if case["next"]:
        x = norm(h, v["w2"])
        got["x"] = x.detach()
        outs.append(x)
        grads.append(t.get("dx"))
    if case["train"]:
        d = torch.autograd.grad(outs, [v[n] for n in names], [gr.to(_F64) for gr in grads])
        got.update({"d " + n: gv for n, gv in zip(names, d)})
    return got
