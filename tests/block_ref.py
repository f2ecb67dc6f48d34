"""64-bit restatements of the attention block's operators, and the bounds their kernels are
held to.

A rounding to a type is off by at most u = eps / 2 of the value.  Sums are fp32: a sum of n
products is off by at most n 2^-23 of the sum of their magnitudes (the tensor cores may
truncate where the ALUs round)."""
import math

import torch

F64 = torch.float64


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rounding(dtype, x):
    """How far rounding to `dtype` may move x: half a step.  A step is eps of the value down to the
    type's least normal number 2^e and stays eps 2^e below it (fp16: 2^-24, so half is 2^-25)."""
    return unit(dtype) * x.abs().clamp(min=torch.finfo(dtype).smallest_normal)


# ------------------------------------------------------------------ attention
def attention(q, k, v, lens_q, lens_k, scale, softcap=0.0, window=(-1, -1), prefix=None, doc_q=None, doc_k=None,
              slopes=None, rel_bias=None):
    """(out, bound) in 64 bits on the CPU; rows of no sequence are NaN in both.

    The bound: the output's rounding, the weights' rounding (each weight times |v|), and the
    scores' error d, which moves every weight by a factor of at most e^(2d)."""
    dtype, u = q.dtype, unit(q.dtype)
    q, k, v = (x.detach().cpu().to(F64) for x in (q, k, v))
    host = [None if x is None else x.detach().cpu() for x in (prefix, doc_q, doc_k, slopes, rel_bias)]
    prefix, doc_q, doc_k, slopes, rel_bias = host
    group = q.shape[1] // k.shape[1]
    out = torch.full_like(q, float("nan"))
    tol = torch.full_like(q, float("nan"))
    at_q = at_k = 0
    for s, (n, m) in enumerate(zip(lens_q, lens_k)):
        place = torch.arange(n)[:, None] + m - n
        away = torch.arange(m)[None] - place
        seen = torch.ones(n, m, dtype=torch.bool)
        if window[0] >= 0:
            seen &= away >= -window[0]
        if window[1] >= 0:
            seen &= away <= window[1]
        if prefix is not None:
            seen |= torch.arange(m)[None] < int(prefix[s])
        if doc_q is not None:
            a, b = doc_q[at_q : at_q + n, None], doc_k[None, at_k : at_k + m]
            seen &= (a == b) & (a >= 0)
        for h in range(q.shape[1]):
            qs, ks, vs = q[at_q : at_q + n, h], k[at_k : at_k + m, h // group], v[at_k : at_k + m, h // group]
            # hidden keys have no part: what they hold is taken out before any product
            used = seen.any(0)
            ks, vs = torch.where(used[:, None], ks, 0.0), torch.where(used[:, None], vs, 0.0)
            t = scale * (qs @ ks.T)
            size = abs(scale) * (qs.abs() @ ks.abs().T)
            err = 2.0 ** -23 * (q.shape[2] + 4) * size + 2.0 ** -21 * t.abs()
            if softcap:
                t = softcap * torch.tanh(t / softcap)
                err = err + 2.0 ** -21 * t.abs() + 2.0 ** -22 * softcap
            if slopes is not None:
                b = -slopes[h].to(F64) * away.abs()
                t, err = t + b, err + 2.0 ** -22 * (b.abs() + t.abs())
            if rel_bias is not None:
                r = rel_bias.shape[1] // 2
                b = rel_bias[h].to(F64)[away.clamp(-r, r) + r]
                t, err = t + b, err + 2.0 ** -22 * torch.where(b.isfinite(), b.abs().clamp(max=1e4) + t.abs().clamp(max=1e4), 0.0)
            t = t.masked_fill(~seen, -math.inf)
            top = t.amax(-1, keepdim=True) if m else torch.zeros(n, 1, dtype=F64)
            top = torch.where(top == -math.inf, 0.0, top)
            p = torch.exp(t - top)
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total > 0, total, 1.0)
            # each row's own keys: 0 times what a key hidden from the row holds is not a product
            o = torch.stack([(p[i, seen[i], None] * vs[seen[i]]).sum(0) for i in range(n)]) if n else qs
            size = torch.stack([(p[i, seen[i], None] * vs[seen[i]].abs()).sum(0) for i in range(n)]) if n else qs
            # 2^-20: exponentials, running rescales and the division, fp32
            near = torch.where(seen & (p > 0), err, 0.0)
            d = near.amax(-1, keepdim=True) if m else torch.zeros(n, 1, dtype=F64)
            tiny = 2.0 ** -24 * (vs.abs().amax() if m else 0.0)  # weights below the type's least step
            out[at_q : at_q + n, h] = o
            tol[at_q : at_q + n, h] = rounding(dtype, o) + (u + torch.expm1(2 * d) + 2.0 ** -20) * size * (1 + u) + tiny
        at_q, at_k = at_q + n, at_k + m
    return out, tol


def check(got, ref, tol):
    """`got` is within `tol` of `ref` wherever `ref` is a number, and NaN or infinite alike elsewhere."""
    got = got.detach().cpu().to(F64)
    fine = ref.isfinite()
    bad = (got[fine] - ref[fine]).abs() > tol[fine]
    bad |= ~got[fine].isfinite()
    assert not bad.any(), (int(bad.sum()), float(((got[fine] - ref[fine]).abs() / tol[fine].clamp(min=1e-30)).max()))


# ------------------------------------------------------------------ rotary positions
def frequencies(rot, theta=10000.0, scaling="none", factor=1.0, context=0, beta_fast=32.0, beta_slow=1.0):
    i = torch.arange(rot // 2, dtype=F64)
    if scaling == "ntk":
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** (-2 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        at = [rot * math.log(context / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (beta_fast, beta_slow)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        g = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        return f / factor * g + f * (1 - g), 0.1 * math.log(factor) + 1
    return f, 1.0


def rope(x, positions, rot, interleaved, freq, stretch):
    """(out, bound): sin and cos of a 64-bit angle reduced to fp32 (off by 2^-22), three fp32
    operations on each value, the output's rounding."""
    dtype = x.dtype
    x = x.detach().cpu().to(F64)
    ang = positions.cpu().to(F64)[:, None] * freq
    c, s = (torch.cos(ang) * stretch)[:, None], (torch.sin(ang) * stretch)[:, None]
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    out, size = x.clone(), torch.zeros_like(x)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., a] * s + x[..., b] * c
    size[..., a] = size[..., b] = (x[..., a].abs() + x[..., b].abs()) * stretch
    return out, rounding(dtype, out) + 2.0 ** -20 * size


# ------------------------------------------------------------------ the linear layer
def activation(t, act):
    if act == "relu":
        return t.clamp(min=0)
    if act == "silu":
        return t / (1 + torch.exp(-t))
    if act == "gelu":
        return 0.5 * t * (1 + torch.erf(t / math.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3)))
    return t


def linear(x, w, bias, act, residual, out_dtype, weights_rounded):
    """(out, bound): the products' sums, the weights' rounding to fp16 where they are stored as
    blocks, the activation (slope up to 1.13, approximations of 2^-20), the output's rounding."""
    x, w = x.detach().cpu().to(F64), torch.as_tensor(w).to(F64)
    t, size = x @ w.T, x.abs() @ w.abs().T
    err = (2.0 ** -23 * x.shape[1] + (2.0 ** -11 if weights_rounded else 0.0)) * size
    if bias is not None:
        t = t + bias.cpu().to(F64)
    y = activation(t, act)
    tol = 1.13 * err + 2.0 ** -20 * (y.abs() + t.abs())
    if residual is not None:
        r = residual.cpu().to(F64)
        y, tol = y + r, tol + 2.0 ** -23 * (r.abs() + y.abs())
    return y, tol + rounding(out_dtype, y.abs() + tol)
