"""Masked attention of some rows of one long sequence, restated in 64 bits, with the bound its
kernels are held to."""
import math

import torch

from block_ref import F64, rounding, unit


def attention_rows(q, k, v, rows, scale, softcap=0.0, window=(-1, -1), prefix=0, doc_q=None, doc_k=None, slopes=None,
                   rel_bias=None):
    """(out, bound) of the query rows `rows` (places as in the whole sequence).

    A score is off by its product's fp32 sum (2^-23 of the magnitudes a term) and a few fp32
    operations (2^-21 of the score each: scale, cap whatever its size, bias), which moves every weight
    by a factor of at most e^(2d).  The sums over the n keys that a row sees are fp32 (n 2^-23 of the
    magnitudes), weights and output are rounded to the type."""
    dtype, u = q.dtype, unit(q.dtype)
    n, m, group = q.shape[0], k.shape[0], q.shape[1] // k.shape[1]
    rows = torch.as_tensor(rows)
    q, k, v = q.detach().cpu()[rows].to(F64), k.detach().cpu().to(F64), v.detach().cpu().to(F64)
    place = rows[:, None] + m - n
    away = torch.arange(m)[None] - place
    seen = torch.ones(len(rows), m, dtype=torch.bool)
    if window[0] >= 0:
        seen &= away >= -window[0]
    if window[1] >= 0:
        seen &= away <= window[1]
    seen |= torch.arange(m)[None] < prefix
    if doc_q is not None:
        a = torch.as_tensor(doc_q).cpu()[rows, None]
        seen &= (a == torch.as_tensor(doc_k).cpu()[None]) & (a >= 0)
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(q.shape[1]):
        ks, vs = k[:, h // group], v[:, h // group]
        t = scale * (q[:, h] @ ks.T)
        err = 2.0 ** -23 * (q.shape[2] + 4) * abs(scale) * (q[:, h].abs() @ ks.abs().T) + 2.0 ** -21 * t.abs()
        if softcap:
            t = softcap * torch.tanh(t / softcap)
            err = err + 2.0 ** -21 * t.abs()
        if slopes is not None:
            b = -slopes[h].cpu().to(F64) * away.abs()
            t, err = t + b, err + 2.0 ** -21 * (b.abs() + t.abs())
        if rel_bias is not None:
            r = rel_bias.shape[1] // 2
            b = rel_bias[h].cpu().to(F64)[away.clamp(-r, r) + r]
            t, err = t + b, err + 2.0 ** -21 * (b.abs() + t.abs())
        t = t.masked_fill(~seen, -math.inf)
        top = t.amax(-1, keepdim=True)
        p = torch.exp(t - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        p = p / torch.where(total > 0, total, 1.0)
        # (keys far below the maximum have no weight, and no error to give)
        d = torch.where(p > 2.0 ** -60, err, 0.0).amax(-1, keepdim=True)
        out[:, h] = p @ vs
        sums = 2.0 ** -23 * (p > 2.0 ** -60).sum(-1, keepdim=True) + 2.0 ** -20
        tiny = 2.0 ** -24 * vs.abs().amax()
        tol[:, h] = rounding(dtype, out[:, h]) + (u + torch.expm1(2 * d) + sums) * (p @ vs.abs()) * (1 + u) + tiny
    return out, tol
