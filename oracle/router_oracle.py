"""Routing in its forms, the router's losses and their gradients in float64 by their formulas, with magnitudes for error
bounds: the sum of the magnitudes that a value is added up from (every subtraction taken as an addition)."""

import math

import torch

from .moe_oracle import sigmoid_f32

F64 = torch.float64


def probabilities(z, score):
    """float64 [T, E]; 0 in rows of -inf alone, for sigmoids of logits at or below -88.72283935546875 too."""
    z = z.detach().to(F64)
    if score == "sigmoid":
        p = 1 / (1 + torch.exp(-z))
        return torch.where(z <= -88.72283935546875, torch.zeros_like(p), p)
    top = z.amax(-1, keepdim=True)
    none = (z == -math.inf).all(-1, keepdim=True)
    e = torch.exp(z - torch.where(none, torch.zeros_like(top), top))
    return torch.where(none, torch.zeros_like(e), e / e.sum(-1, keepdim=True))


def complement(z):
    """1 - sigmoid(z) in float64, with all its digits where the sigmoid is near 1."""
    return 1 / (1 + torch.exp(z.detach().to(F64)))


def rounded(z, score):
    """The probabilities rounded once to float32 (those that the selection sees)."""
    if score == "sigmoid":
        return torch.from_numpy(sigmoid_f32(z.detach().float().cpu().numpy())).to(z.device)
    return probabilities(z, score).float()


def _order(s):
    """Places by (score descending, number ascending), NaN first."""
    s = torch.where(torch.isnan(s), torch.full_like(s, math.inf), s.clamp(max=torch.finfo(s.dtype).max))
    return torch.sort(s, dim=-1, descending=True, stable=True).indices


def select(z, k, bias, score, groups, top_groups, group_scores):
    """idx [T, k]."""
    p = rounded(z, score)
    s = p + bias.float() if bias is not None else z.detach().float()
    if groups > 1:
        T, E = z.shape
        by = s if bias is not None or group_scores == 1 else p
        best = torch.gather(by.view(T, groups, -1), 2, _order(by.view(T, groups, -1))[..., :group_scores])
        of_group = best[..., 0] if group_scores == 1 else best[..., 0] + best[..., 1]
        kept = _order(of_group)[:, :top_groups]
        out = torch.empty(T, k, dtype=torch.int64, device=z.device)
        for t in range(T):
            mine = torch.cat([torch.arange(g * (E // groups), (g + 1) * (E // groups)) for g in sorted(kept[t].tolist())])
            mine = mine.to(z.device)
            out[t] = mine[_order(s[t, mine])[:k]]
        return out
    return _order(s)[:, :k]


def weights(z, idx, score, renormalize, scale):
    p = probabilities(z, score).gather(1, idx)
    return scale * p / p.sum(1, keepdim=True).clamp(min=1e-12) if renormalize else scale * p


def weights_backward(z, idx, dw, score, renormalize, scale):
    """d logits and its magnitudes [T, E]."""
    full, dw = probabilities(z, score), dw.to(F64)
    p = full.gather(1, idx)
    c = abs(scale)
    dp, mp = scale * dw, c * dw.abs()
    if renormalize:
        S = p.sum(1, keepdim=True)
        free = S > 1e-12
        S = S.clamp(min=1e-12)
        dp = (dp - torch.where(free, (dp * p).sum(1, keepdim=True) / S, 0.0)) / S
        mp = (mp + torch.where(free, (mp * p).sum(1, keepdim=True) / S, 0.0)) / S
    if score == "sigmoid":
        at, slope = torch.zeros_like(full), p * complement(z).gather(1, idx)
        return at.scatter(1, idx, dp * slope), at.scatter(1, idx, mp * slope)
    at = torch.zeros_like(full)
    inner, minner = (dp * p).sum(1, keepdim=True), (mp * p).sum(1, keepdim=True)
    if renormalize:
        inner = torch.where(free, 0.0, inner)
        minner = torch.where(free, 0.0, minner)
    return full * (at.scatter(1, idx, dp) - inner), full * (at.scatter(1, idx, mp) + minner)


def _shares(z, score):
    """(ph, softmax, sigmoid, lse, whether the row has anything) of each token."""
    z = z.detach().to(F64)
    some = ~(z == -math.inf).all(-1, keepdim=True)
    soft, sig = probabilities(z, "softmax"), probabilities(z, "sigmoid")
    p = soft if score == "softmax" else sig
    total = p.sum(-1, keepdim=True)
    ph = torch.where(total == 0, torch.zeros_like(p), p / total)
    lse = torch.where(some[:, 0], torch.logsumexp(z, -1), torch.zeros((), dtype=F64, device=z.device))
    return ph, soft, sig, lse


def losses(z, idx, score, cu=None):
    """(balance, z loss, a [S, E], tokens): a is the balance loss's grad by a sequence's sums of shares."""
    T, E = z.shape
    k = idx.shape[1]
    cu = [0, T] if cu is None else cu.tolist()
    ph, _, _, lse = _shares(z, score)
    live = sum(b > a for a, b in zip(cu[:-1], cu[1:]))
    a = torch.zeros(len(cu) - 1, E, dtype=F64, device=z.device)
    balance = z2 = torch.zeros((), dtype=F64, device=z.device)
    n_all = 0
    for s, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
        n = hi - lo
        if n > 0:
            count = torch.bincount(idx[lo:hi].reshape(-1), minlength=E).to(F64)
            a[s] = E * count / (k * n * n * live)
            balance = balance + (a[s] * ph[lo:hi].sum(0)).sum()
            z2 = z2 + lse[lo:hi].square().sum()
            n_all += n
    return balance, z2 / max(n_all, 1), a, n_all


def losses_backward(z, idx, score, cu, g_balance, g_z):
    """d logits and its magnitudes [T, E]."""
    T, E = z.shape
    _, _, a, n_all = losses(z, idx, score, cu)
    cu = [0, T] if cu is None else cu.tolist()
    ph, soft, _, lse = _shares(z, score)
    val, mag = torch.zeros(T, E, dtype=F64, device=z.device), torch.zeros(T, E, dtype=F64, device=z.device)
    for s, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
        if hi <= lo:
            continue
        r = slice(lo, hi)
        dot = (ph[r] * a[s]).sum(-1, keepdim=True)
        f = ph[r] * complement(z[r]) if score == "sigmoid" else ph[r]
        zpart = 2 * g_z / n_all * lse[r].unsqueeze(1) * soft[r]
        val[r] = g_balance * f * (a[s] - dot) + zpart
        mag[r] = abs(g_balance) * f * (a[s] + dot) + zpart.abs()
    return val, mag
