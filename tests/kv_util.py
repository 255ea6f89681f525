"""The KV-cache operators in 64 bits, request by request and head by head, and
the bounds that their tests hold the kernels to."""

import math

import torch

U = 2.0**-24  # half a step of f32, relative


def dense(x, requests, heads, cap, hd):
    return x.view(requests, heads, cap, hd)


def attend(q, k, v, lens, new, pk=None, pv=None, scale=None):
    """q [R][n][H][hd]; k, v [R][G][cap][hd]; pk, pv [G][P][hd].  (out, bound,
    weights, weight bound, prefix weights, its bound): rows of tokens >= new
    are NaN in out.

    Bounds.  A score is a sum of hd products in f32 (or of f16 parts of q, off
    by 2^-22 of |q|): roundings of at most U of a partial sum, which is at most
    |q||k|, independent, so their sum stays within 6 sqrt(hd + 4) U |q||k|
    (6 sigma, sigma of one being under U), and 4 U of it for the parts.  A
    weight is off by that much of itself, 4 U for exp and the score's own
    rounding times its size, and the same once more through the sum it is
    divided by.  The sums over n keys add 6 sqrt(n) U of what their terms'
    sizes add up to."""
    R, n, H, hd = q.shape
    G, cap = k.shape[1], k.shape[2]
    rep = H // G
    P = 0 if pk is None else pk.shape[1]
    scale = hd**-0.5 if scale is None else scale
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    w = torch.zeros(R, G, cap, dtype=torch.float64, device=q.device)
    wt = torch.zeros_like(w)
    pw = torch.zeros(G, P, dtype=torch.float64, device=q.device)
    pwt = torch.zeros_like(pw)
    for b in range(R):
        L, t = int(lens[b]), int(new[b])
        if t == 0:
            continue
        for g in range(G):
            keys, vals = k[b, g, :L].double(), v[b, g, :L].double()
            if P:
                keys, vals = torch.cat([pk[g].double(), keys]), torch.cat([pv[g].double(), vals])
            qq = q[b, :t, g * rep : (g + 1) * rep].double()  # [t][rep][hd]
            s = (qq.reshape(t * rep, hd) @ keys.t().contiguous()).view(t, rep, P + L) * scale
            seen = torch.arange(P + L, device=q.device)[None] <= (P + L - t + torch.arange(t, device=q.device))[:, None]
            s = s.masked_fill(~seen[:, None], -math.inf)
            p = torch.softmax(s, 2)
            p0 = torch.where(seen[:, None], p, torch.zeros_like(p))
            o = torch.zeros_like(qq)
            size = torch.zeros_like(qq)
            for i in range(t):  # only what a row sees
                m = P + L - t + i + 1
                o[i] = p0[i, :, :m] @ vals[:m]
                size[i] = p0[i, :, :m] @ vals[:m].abs()
            kn = torch.where(seen, keys.norm(dim=1).expand(seen.shape), torch.zeros((), dtype=torch.float64, device=q.device)).amax(1)
            ds = (6 * math.sqrt(hd + 4) + 8) * U * scale * qq.norm(dim=2) * kn[:, None]
            ds = ds + 4 * U * (1 + s.masked_fill(~seen[:, None], 0).abs().amax(2))
            rel = 2 * ds + (12 * math.sqrt(P + L) + 16) * U
            out[b, :t, g * rep : (g + 1) * rep] = o
            tol[b, :t, g * rep : (g + 1) * rep] = rel[..., None] * size + 1e-37
            total, far = p0.sum((0, 1)), (p0 * rel[..., None]).sum((0, 1)) + 8 * U * p0.sum((0, 1)) + 1e-30
            w[b, g, :L], wt[b, g, :L] = total[P:], far[P:]
            pw[g] += total[:P]
            pwt[g] += far[:P]
    return out, tol, w, wt, pw, pwt


def select(scores, positions, n, keep, recent, sinks):
    """(from, to, m) of one head: rows of slots `from` move to slots `to`, m stay in use."""
    import numpy as np

    m = min(n, keep)
    if n <= keep:
        return [], [], m
    pos = positions[:n].astype(np.int64)
    s = scores[:n].astype(np.float64)
    s = np.where(np.isnan(s), -np.inf, s) + 0.0
    safe = (pos > pos.max() - recent) | (pos < sinks)
    best = np.lexsort((np.arange(n), -s, ~safe))[:m]
    kept = np.zeros(n, bool)
    kept[best] = True
    return (m + np.flatnonzero(kept[m:])).tolist(), np.flatnonzero(~kept[:m]).tolist(), m


def rotated(x, positions, gain, base, eps):
    """Normed (gain not None) and rotated heads x [..., heads, hd] at positions [...]."""
    x = x.double()
    hd = x.shape[-1]
    if gain is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * gain.double()
    f = torch.tensor(base, dtype=torch.float32).double().item() ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=x.device) / hd)
    a = positions.double()[..., None, None] * f
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack((e * a.cos() - o * a.sin(), e * a.sin() + o * a.cos()), -1).flatten(-2)
