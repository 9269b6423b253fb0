"""The cache operators' definitions in 64 bits, one sequence and head at a time,
with bounds for the kernels' rounding (test infrastructure).

Bounds.  The transform's exponent t (log2 units) is computed in fp32 from a score
s = q.k summed over D products: |ds| <= D 2^-24 sum |q||k|, and
|dt / ds| <= |n| c / ln 2 with c = scale b; log2, the product with n, the
subtraction of the running maximum or m and exp2 add one rounding each of values
below 32 in these tests (4 x 2^-19 = 2^-17).  A probability is then off by at
most ln 2 times twice that (itself and its normaliser), and before the product
with V it is rounded to the input type, by at most half a step.
"""

from __future__ import annotations

import math

import torch

LN2 = math.log(2.0)


def transform(s, n, b):
    """t = n sign(s) log2(1 + b |s|), of scaled scores."""
    return n * s.sign() * torch.log1p(b * s.abs()) / LN2


def t_slack(q, k, scale, n, b):
    """Bound of the exponent's error for one head's q [T, D] and k [L, D]."""
    if k.numel() == 0:
        return 2.0 ** -17
    most = float((q.abs() @ k.abs().t()).max())
    return 2.0 ** -17 + abs(n) * scale * b / LN2 * q.shape[1] * 2.0 ** -24 * most


def tree(q, k, v, lens, mask, scale, n, b):
    """(out, m, bound of out, bound of m) of every node, in float64."""
    B, Hq, T, D = q.shape
    G, cap = Hq // k.shape[1], k.shape[2]
    half = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    m = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=q.device)
    mtol = torch.zeros_like(m)
    for i in range(B):
        L = min(max(int(lens[i]), 0), cap)
        held = min(T, L)  # the tree's last `held` nodes are there
        rows = (mask[i] if mask.dim() == 3 else mask).bool()[:, T - held:]
        seen = torch.cat([torch.ones(T, L - held, dtype=torch.bool, device=q.device), rows], 1)
        for h in range(Hq):
            kh, vh, qh = k[i, h // G, :L].double(), v[i, h // G, :L].double(), q[i, h].double()
            # what a node does not see must not reach it, whatever it holds
            kz, vz = (torch.nan_to_num(x, 0.0, 0.0, 0.0) for x in (kh, vh))
            t = transform(scale * (qh @ kz.t()), n, b).masked_fill(~seen, -math.inf)
            top = t.amax(1, keepdim=True) if L else torch.full((T, 1), -math.inf, dtype=torch.float64, device=q.device)
            some = (top > -math.inf)[:, 0]
            p = torch.exp2(t - top.masked_fill(~some[:, None], 0.0))
            z = p.sum(1, keepdim=True)
            p = torch.where(some[:, None], p / z.clamp_min(1e-300), torch.zeros_like(p))
            out[i, h] = p @ vz
            m[i, h] = torch.where(some, (top + z.clamp_min(1e-300).log2())[:, 0], m[i, h])
            dt = t_slack(qh, kz, scale, n, b)
            weight = p @ vz.abs()
            tol[i, h] = half * out[i, h].abs() + (half + 2 * LN2 * dt) * 1.01 * weight + 2.0 ** -20 * weight + 1e-30
            mtol[i, h] = 2 * dt + 2.0 ** -22 * m[i, h].abs().nan_to_num(0.0, 0.0, 0.0)
    return out, m, tol, mtol


def key_weights(q, k, m, lens, weights, scale, n, b):
    """(weights, bound) after the queries' probabilities are added, in float64."""
    B, Hq, T, D = q.shape
    Hk, cap = k.shape[1], k.shape[2]
    G = Hq // Hk
    out = weights.double().clone()
    tol = torch.zeros_like(out)
    for i in range(B):
        L = min(max(int(lens[i]), 0), cap)
        pos = torch.arange(L - T, L, device=q.device)[:, None]
        seen = torch.arange(L, device=q.device)[None, :] <= pos
        for h in range(Hq):
            kh, qh, mh = k[i, h // G, :L].double(), q[i, h].double(), m[i, h].double()
            t = transform(scale * (qh @ kh.t()), n, b)
            p = torch.exp2(t - mh[:, None])
            p = torch.where(seen & (mh > -math.inf)[:, None], p, torch.zeros_like(p)).sum(0)
            out[i, h // G, :L] += p
            # G T sums of fp32, and the last one into the weight
            tol[i, h // G, :L] += p * (LN2 * t_slack(qh, kh, scale, n, b) * 1.01 + G * T * 2.0 ** -24)
        tol[i, :, :L] += out[i, :, :L].abs() * 2.0 ** -23 + 1e-30
    return out, tol


def evict(lens, weights, keep, sinks, recent):
    """(new lengths, new weights, kept) as lists and float32 / int32 tensors on the host."""
    B, Hk, cap = weights.shape
    w = weights.cpu()
    kept = torch.full((B, Hk, keep), -1, dtype=torch.int32)
    left = torch.zeros(B, Hk, cap)
    new = []
    for i in range(B):
        L = min(max(int(lens[i]), 0), cap)
        new.append(min(L, keep))
        for h in range(Hk):
            rows = list(range(L))
            if L > keep:
                must = set(range(sinks)) | set(range(L - recent, L))
                free = [r for r in rows if r not in must]
                rank = lambda r: (not math.isnan(w[i, h, r]), float(w[i, h, r].nan_to_num(0.0, math.inf, -math.inf)))  # noqa: E731
                free.sort(key=lambda r: (rank(r), -r), reverse=True)
                rows = sorted(must | set(free[:keep - len(must)]))
            kept[i, h, :len(rows)] = torch.tensor(rows, dtype=torch.int32)
            left[i, h, :len(rows)] = w[i, h, rows]
    return new, left, kept
