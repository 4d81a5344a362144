"""The sequence operators from their definitions in 64 bits (torch, CPU), with the sums of absolute values that the
tests' tolerances are made of.  Test infrastructure only."""
import math

import torch

F64 = torch.float64


def attention(q, k, v, q_off, k_off, *, scale, causal=True, window=0, key_mask=None, k_len=None):
    """(out, lse, weight, spread): weight = sum_j p_j |v_j| per output, spread = max_j scale sum |q||k_j| per row and
    head over the visible keys.  Rows that belong to no series stay 0."""
    q, k, v = (x.detach().cpu().to(F64) for x in (q, k, v))
    R, H, D = q.shape
    rep = H // k.shape[1]
    out, weight = torch.zeros(R, H, D, dtype=F64), torch.zeros(R, H, D, dtype=F64)
    lse, spread = torch.zeros(R, H, dtype=F64), torch.zeros(R, H, dtype=F64)
    for s in range(len(q_off) - 1):
        a, b = q_off[s], q_off[s + 1]
        c, d = k_off[s], k_off[s + 1]
        nk = d - c
        if k_len is not None:
            nk = max(0, min(nk, int(k_len[s])))
        for i in range(a, b):
            end = (i - a) + nk - (b - a)
            see = torch.ones(nk, dtype=torch.bool)
            j = torch.arange(nk)
            if causal:
                see &= j <= end
            if window:
                see &= j > end - window
            if key_mask is not None:
                see &= key_mask[c:c + nk].cpu().bool()
            at = c + j[see]
            if len(at) == 0:
                lse[i] = -math.inf
                continue
            ks, vs = k[at].repeat_interleave(rep, 1), v[at].repeat_interleave(rep, 1)
            z = torch.einsum("hd,nhd->hn", q[i], ks) * scale
            p = torch.softmax(z, 1)
            lse[i] = torch.logsumexp(z, 1)
            out[i] = torch.einsum("hn,nhd->hd", p, vs)
            weight[i] = torch.einsum("hn,nhd->hd", p, vs.abs())
            spread[i] = (torch.einsum("hd,nhd->hn", q[i].abs(), ks.abs()) * scale).max(1)[0]
    return out, lse, weight, spread


def linear_attention(q, k, v, log_decay, offsets, *, scale, state=None):
    """(out, final, out_abs, final_abs): the last two with every product replaced by its absolute value."""
    q, k, v = (x.detach().cpu().to(F64) for x in (q, k, v))
    lam = torch.exp(log_decay.detach().cpu().to(F64).clamp(max=0))
    R, H, dk = q.shape
    dv, rep, n = v.shape[2], H // k.shape[1], len(offsets) - 1
    out, out_abs = torch.zeros(R, H, dv, dtype=F64), torch.zeros(R, H, dv, dtype=F64)
    S = torch.zeros(n, H, dk, dv, dtype=F64) if state is None else state.detach().cpu().to(F64).clone()
    A = S.abs()
    for s in range(n):
        for t in range(offsets[s], offsets[s + 1]):
            kk, vv = k[t].repeat_interleave(rep, 0), v[t].repeat_interleave(rep, 0)
            S[s] = lam[:, None, None] * S[s] + kk[:, :, None] * vv[:, None, :]
            A[s] = lam[:, None, None] * A[s] + kk.abs()[:, :, None] * vv.abs()[:, None, :]
            out[t] = scale * torch.einsum("hk,hkv->hv", q[t], S[s])
            out_abs[t] = abs(scale) * torch.einsum("hk,hkv->hv", q[t].abs(), A[s])
    return out, S, out_abs, A


ACT = {"linear": lambda x: x, "relu": lambda x: torch.where(x < 0, torch.zeros_like(x), x), "sigmoid": torch.sigmoid, "silu": lambda x: x * torch.sigmoid(x)}


def group_norm(x, groups, gamma, beta, offsets, *, eps, activation):
    """(y, size): size = the size of the terms that are summed before the activation."""
    x = x.detach().cpu().to(F64)
    C = x.shape[1]
    g = torch.ones(C, dtype=F64) if gamma is None else gamma.detach().cpu().to(F64)
    b = torch.zeros(C, dtype=F64) if beta is None else beta.detach().cpu().to(F64)
    y, size = torch.zeros_like(x), torch.zeros_like(x)
    for s in range(len(offsets) - 1):
        r = slice(offsets[s], offsets[s + 1])
        if offsets[s] == offsets[s + 1]:
            continue
        z = x[r].reshape(-1, groups, C // groups)
        mean = z.mean((0, 2), keepdim=True)
        std = torch.sqrt(((z - mean) ** 2).mean((0, 2), keepdim=True) + eps)
        w = ((z - mean) / std).reshape(-1, C)
        m = ((z.abs() + z.abs().mean((0, 2), keepdim=True)) / std).reshape(-1, C)
        y[r] = ACT[activation](w * g + b)
        size[r] = (m + w.abs()) * g.abs() + b.abs()
    return y, size
