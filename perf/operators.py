"""The operators of an encoder's attention block, and the calls that are timed of them.

Three operators, in the order in which a block runs them on its packed rows (sequences one
behind the other, offsets in cu_seqlens):

rope       rotary positions.  Pair i of a head turns by the angle p f_i, with p the row's
           position and f_i = theta^(-2i/r) for r rotated values a head; "half" pairs the values
           i and i + r/2, "interleaved" 2i and 2i + 1; the head's values behind r stay.  For long
           contexts f_i is divided by a factor ("linear"), taken from a larger theta ("ntk"), or
           mixed of both by a ramp over i ("yarn", which also stretches cos and sin).
attention  out_i = sum_j p_ij v_j with p_i the softmax over the keys that row i may see of
           c tanh(scale q_i.k_j / c) + bias(j - i), c the cap (none: the plain product).  The bias
           is -slope |j - i| of the head, or a table by the clamped distance.  Row i of n sees key
           j of m by its place i + m - n: a window around it, a prefix of the keys that every row
           sees, and equal document numbers.  A row that sees nothing gets zeros.
linear     act(x W^T + bias) + residual, with W stored as fp16 or as blocks of 32 8-bit
           numbers and a scale each.

`run` computes them as elementary torch operations in 32 bits (angles in 64), or, where `own` is
true, by the calls a program makes of this package.
"""
import math
import random

import numpy as np
import torch

own = False

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}


# ------------------------------------------------------------------------------ the cases
def _rope(name, **kw):
    c = dict(op="rope", dtype="fp16", heads=24, head_dim=64, rot=64, layout="half", theta=10000.0, scaling="none",
             factor=1.0, context=0, spare=0, positions="own", seqs=1, shortest=1, longest=1)
    return dict(c, **kw, name=name) if name else dict(c, **kw)


def _attn(name, **kw):
    c = dict(op="attention", dtype="fp16", heads=12, kv_heads=12, head_dim=64, fused=True, seqs=1, shortest=1,
             longest=1, rows=0, left=-1, right=-1, cap=0.0, bias="none", radius=0, prefix=0.0, docs=0)
    return dict(c, **kw, name=name) if name else dict(c, **kw)


def _linear(name, **kw):
    c = dict(op="linear", weight="fp16", k=768, n=768, m=1, bias=True, act="none", residual="fp16", out="fp16", spare=0)
    return dict(c, **kw, name=name) if name else dict(c, **kw)


def listed():
    return [
        # one token of a block of 12 heads: its query and key, the smallest call
        _rope("rope one token", positions="given"),
        # the queries and keys of a batch of 256 texts, in the rows that the QKV product wrote
        _rope("rope batch", seqs=256, shortest=32, longest=512, spare=12 * 64),
        # long documents with grouped heads, half of each head rotated, past the trained context
        _rope("rope long", dtype="bf16", heads=10, head_dim=128, rot=64, layout="interleaved", theta=500000.0,
              scaling="yarn", factor=16.0, context=8192, seqs=2, shortest=30001, longest=65536),
        # the last token of 32 texts against all keys before it
        _attn("attention one token", dtype="bf16", heads=16, kv_heads=4, head_dim=128, fused=False, seqs=32,
              shortest=500, longest=4096, rows=1, right=0, cap=50.0),
        # a batch of texts with a bias that falls with the distance on both sides
        _attn("attention slopes", seqs=256, shortest=32, longest=512, bias="slopes"),
        # narrow heads with a learned bias for each distance, a short batch
        _attn("attention table", head_dim=32, seqs=37, shortest=1, longest=400, bias="table", radius=128),
        # long texts, capped scores, each token with the 1024 before it, grouped heads
        _attn("attention capped window", dtype="bf16", heads=8, kv_heads=2, head_dim=128, fused=False, seqs=2,
              shortest=6001, longest=8192, left=1024, right=0, cap=30.0),
        # one packed row of 24 documents, each read by itself
        _attn("attention documents", seqs=1, shortest=8000, longest=8000, docs=24),
        # causal texts whose first part is read in both directions
        _attn("attention prefix", dtype="bf16", heads=16, kv_heads=16, head_dim=80, fused=False, seqs=6, shortest=1000,
              longest=2100, right=0, prefix=0.3),
        # the output product of one token
        _linear("linear one token", weight="q8_0", act="silu"),
        # the output product of the batch of 256 texts, added to the residual stream
        _linear("linear batch", m=70825),
        # a wider block's up product, with 32-bit rows to add to
        _linear("linear wide", weight="q8_0", k=1024, n=1536, m=33001, act="gelu_tanh", residual="fp32", spare=64),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("rope", "attention", "attention", "linear"))
    if op == "rope":
        hd = 8 * rng.randint(4, 16)
        rot = hd if rng.random() < 0.5 else 2 * rng.randint(2, hd // 2)
        longest = _spread(rng, 1, 16384)
        scaling = rng.choice(("none", "none", "linear", "ntk", "yarn"))
        return _rope(None, dtype=rng.choice(("fp16", "bf16", "fp32")), heads=rng.randint(1, 32), head_dim=hd, rot=rot,
                     layout=rng.choice(("half", "interleaved")), theta=rng.choice((1e4, 1e5, 5e5)), scaling=scaling,
                     factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 16.0)),
                     context=rng.choice((2048, 8192)) if scaling == "yarn" else 0, spare=8 * rng.randint(0, 100),
                     positions=rng.choice(("own", "given")), seqs=_spread(rng, 1, max(1, 32768 // longest)),
                     shortest=rng.randint(1, longest), longest=longest)
    if op == "attention":
        kv = rng.choice((1, 2, 3, 4, 8, 12))
        group = rng.choice((1, 1, 2, 3, 4)) if kv < 12 else 1
        longest = _spread(rng, 1, 4096)
        hd = 8 * rng.randint(2, 16)
        bias = rng.choice(("none", "none", "slopes", "table"))
        right = rng.choice((-1, -1, 0, 100))
        left = rng.choice((-1, -1, _spread(rng, 1, 1000)))
        return _attn(None, dtype=rng.choice(("fp16", "bf16")), heads=kv * group, kv_heads=kv, head_dim=hd,
                     fused=rng.random() < 0.5, seqs=_spread(rng, 1, max(1, min(128, (1 << 24) // (longest * longest)))),
                     shortest=rng.randint(1, longest), longest=longest, rows=rng.choice((0, 0, 0, 1, rng.randint(2, 40))),
                     left=left, right=right, cap=rng.choice((0.0, 0.0, 20.0, 50.0)), bias=bias,
                     radius=_spread(rng, 1, 600) if bias == "table" else 0,
                     prefix=rng.choice((0.0, 0.0, rng.random())), docs=rng.choice((0, 0, rng.randint(1, 12))))
    weight = rng.choice(("fp16", "q8_0"))
    return _linear(None, weight=weight, k=64 * rng.randint(2, 24), n=128 * rng.randint(1, 12), m=_spread(rng, 1, 30000),
                   bias=rng.random() < 0.7, act=rng.choice(("none", "relu", "silu", "gelu", "gelu_tanh")),
                   residual="fp16" if weight == "q8_0" else rng.choice(("none", "fp16", "bf16", "fp32")),
                   out=rng.choice(("fp16", "bf16")) if weight == "q8_0" else rng.choice(("fp16", "bf16", "fp32")),
                   spare=8 * rng.randint(0, 20))


def _lengths(case):
    """(rows, keys) of each sequence: the keys spread evenly over the case's range, in an order of their own."""
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    keys = [b - (b - a) * i // max(1, n - 1) for i in range(n)]
    random.Random(n * 7919 + a * 31 + b).shuffle(keys)
    rows = case.get("rows", 0)
    return [min(rows, x) if rows else x for x in keys], keys


def _prefix(case, keys):
    return [int(case["prefix"] * x) for x in keys]


def _documents(case, n):
    """The document number of each of n packed keys: runs of uneven lengths."""
    r = random.Random(n + case["docs"])
    cuts = np.array(sorted(r.randrange(n) for _ in range(case["docs"] - 1)), dtype=np.int64)
    return np.searchsorted(cuts, np.arange(n), side="right").astype(np.int32)


# ------------------------------------------------------------------------------ what a pass needs
def _span(case, rows, keys):
    """First and last + 1 key of the window of each row of one sequence."""
    place = np.arange(rows, dtype=np.int64) + keys - rows
    lo = np.zeros(rows, dtype=np.int64) if case["left"] < 0 else np.maximum(place - case["left"], 0)
    hi = np.full(rows, keys, dtype=np.int64) if case["right"] < 0 else np.minimum(place + case["right"] + 1, keys)
    return np.minimum(lo, hi), hi


def _pairs(case):
    """The (row, key) pairs that see each other, over all sequences."""
    total, at = 0, 0
    rows, keys = _lengths(case)
    docs = _documents(case, sum(keys)) if case["docs"] else None
    for n, m, p in zip(rows, keys, _prefix(case, keys)):
        lo, hi = _span(case, n, m)
        if docs is None:
            total += int((hi - lo + np.minimum(p, lo) + np.maximum(p - np.maximum(hi, lo), 0)).sum())
        else:
            d = docs[at : at + m]
            first, last = np.searchsorted(d, d[m - n :], "left"), np.searchsorted(d, d[m - n :], "right")
            inside = np.maximum(np.minimum(hi, last) - np.maximum(lo, first), 0)
            ahead = np.maximum(np.minimum(np.minimum(p, lo), last) - first, 0)
            behind = np.maximum(np.minimum(p, last) - np.maximum(np.maximum(hi, lo), first), 0)
            total += int((inside + ahead + behind).sum())
        at += m
    return total


def work(case):
    if case["op"] == "rope":
        rows = sum(_lengths(case)[1])
        values = rows * case["heads"] * case["head_dim"]
        return {"bytes": 2 * values * SIZE[case["dtype"]], "flops": 3 * rows * case["heads"] * case["rot"]}
    if case["op"] == "attention":
        rows, keys = (sum(x) for x in _lengths(case))
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        return {"bytes": 2 * d * (2 * rows * h + 2 * keys * kv), "flops": 4 * d * h * _pairs(case)}
    m, n, k = case["m"], case["n"], case["k"]
    w = n * k * (2 if case["weight"] == "fp16" else 34 / 32)
    moved = m * k * 2 + m * n * SIZE[case["out"]] + m * n * SIZE.get(case["residual"], 0)
    return {"bytes": w + moved + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------ inputs
def _offsets(lens):
    return torch.tensor([0] + np.cumsum(lens).tolist(), dtype=torch.int32, device="cuda")


def _frequencies(case):
    """f_i of the case in 64 bits, and what cos and sin are stretched by."""
    r, theta, s = case["rot"], case["theta"], case["factor"]
    i = np.arange(r // 2, dtype=np.float64)
    f = theta ** (-2.0 * i / r)
    if case["scaling"] == "linear":
        return f / s, 1.0
    if case["scaling"] == "ntk":
        return (theta * s ** (r / (r - 2.0))) ** (-2.0 * i / r), 1.0
    if case["scaling"] == "yarn":
        # the pair that turns b times within the trained context lies at this i
        at = [r * math.log(case["context"] / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), r - 1)
        ramp = np.clip((i - low) / max(high - low, 1e-3), 0.0, 1.0)
        return f / s * ramp + f * (1.0 - ramp), 0.1 * math.log(s) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype="fp16"):
        return torch.randn(shape, generator=g, device="cuda").to(DT[dtype])

    s = dict(case=case)
    if case["op"] == "rope":
        _, lens = _lengths(case)
        rows, width = sum(lens), case["heads"] * case["head_dim"]
        s["x"] = normal(rows, width + case["spare"], dtype=case["dtype"])[:, :width].view(rows, case["heads"], -1)
        s["cu"] = _offsets(lens)
        s["positions"] = torch.from_numpy(np.concatenate([np.arange(n, dtype=np.int32) for n in lens])).cuda()
        if case["positions"] == "given":  # each text goes on where an earlier part of it ended
            s["positions"] += torch.randint(0, 4096, (1,), generator=g, device="cuda").int()
        s["freq"], s["stretch"] = _frequencies(case)
        if own:
            from crispembed_b200 import binding

            s["rope"] = binding.Rope(case["rot"], case["theta"], scaling=case["scaling"], factor=case["factor"],
                                     context=case["context"])
        return s
    if case["op"] == "attention":
        rows, keys = _lengths(case)
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        if case["fused"] and rows == keys:  # the rows that a QKV product wrote
            x = normal(sum(rows), (h + 2 * kv) * d, dtype=case["dtype"]).view(sum(rows), h + 2 * kv, d)
            s["q"], s["k"], s["v"] = x[:, :h], x[:, h : h + kv], x[:, h + kv :]
        else:
            s["q"] = normal(sum(rows), h, d, dtype=case["dtype"])
            s["k"], s["v"] = (normal(sum(keys), kv, d, dtype=case["dtype"]) for _ in "kv")
        s["cu_q"], s["cu_k"] = _offsets(rows), _offsets(keys)
        s["max_q"], s["max_k"] = max(rows), max(keys)
        s["scale"] = 1.5 / math.sqrt(d)
        s["slopes"] = s["table"] = s["prefix"] = s["doc_q"] = s["doc_k"] = None
        if case["bias"] == "slopes":
            s["slopes"] = torch.rand(h, generator=g, device="cuda") * 0.1
        if case["bias"] == "table":
            s["table"] = normal(h, 2 * case["radius"] + 1, dtype="fp32")
        if case["prefix"] > 0:
            s["prefix"] = torch.tensor(_prefix(case, keys), dtype=torch.int32, device="cuda")
        if case["docs"]:
            docs = _documents(case, sum(keys))
            at = np.concatenate([e - n + np.arange(n) for n, e in zip(rows, np.cumsum(keys))])
            s["doc_k"], s["doc_q"] = torch.from_numpy(docs).cuda(), torch.from_numpy(docs[at]).cuda()
        return s
    m, n, k = case["m"], case["n"], case["k"]
    s["x"] = normal(m, k + case["spare"])[:, :k]
    w = torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k)
    if case["weight"] == "fp16":
        s["w"] = w.half()
        raw = s["w"].cpu().numpy().view(np.uint8)
    else:  # a row's blocks: the scale as fp16, then 32 whole numbers of [-127, 127]
        b = w.view(n, k // 32, 32)
        scale = (b.abs().amax(-1, keepdim=True) / 127).half()
        q = torch.clamp(torch.round(b / scale.float()), -127, 127).to(torch.int8)
        s["w"] = (q.float() * scale.float()).view(n, k)
        raw = torch.cat([scale.view(torch.uint8), q.view(torch.uint8)], -1).cpu().numpy()
    s["bias"] = normal(n, dtype="fp32") if case["bias"] else None
    s["residual"] = None
    if case["residual"] != "none":
        s["residual"] = normal(m, n + case["spare"], dtype=case["residual"])[:, :n]
    if own:
        from crispembed_b200 import binding

        kind = binding.TYPE_F16 if case["weight"] == "fp16" else binding.TYPE_Q8_0
        s["linear"] = binding.Linear(kind, raw, n, k)
    return s


# ------------------------------------------------------------------------------ one pass
def run(s):
    if own:
        return {"rope": _call_rope, "attention": _call_attention, "linear": _call_linear}[s["case"]["op"]](s)
    return {"rope": _plain_rope, "attention": _plain_attention, "linear": _plain_linear}[s["case"]["op"]](s)


def _call_rope(s):
    c = s["case"]
    where = dict(positions=s["positions"]) if c["positions"] == "given" else dict(cu_seqlens=s["cu"])
    return s["rope"](s["x"], interleaved=c["layout"] == "interleaved", **where)


def _call_attention(s):
    from crispembed_b200 import binding

    c = s["case"]
    return binding.attention_masked(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["max_q"], s["max_k"],
                                    scale=s["scale"], softcap=c["cap"], window=(c["left"], c["right"]),
                                    prefix=s["prefix"], doc_q=s["doc_q"], doc_k=s["doc_k"], slopes=s["slopes"],
                                    rel_bias=s["table"])


def _call_linear(s):
    c = s["case"]
    return s["linear"].fused(s["x"], bias=s["bias"], act=c["act"], residual=s["residual"], out_dtype=DT[c["out"]])


def _plain_rope(s):
    c, x = s["case"], s["x"]
    r = c["rot"]
    angle = s["positions"].double()[:, None] * torch.from_numpy(s["freq"]).cuda()
    cos, sin = ((f(angle) * s["stretch"]).float()[:, None] for f in (torch.cos, torch.sin))
    out = x.float()
    a, b = (out[..., : r // 2], out[..., r // 2 : r]) if c["layout"] == "half" else (out[..., 0:r:2], out[..., 1:r:2])
    turned = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat(turned, -1) if c["layout"] == "half" else torch.stack(turned, -1).flatten(-2)
    return torch.cat([turned, out[..., r:]], -1).to(x.dtype)


def _padded(x, cu, longest):
    """[rows, heads, d] as [sequences, heads, longest, d] in 32 bits, zeros behind each sequence; and which rows are one."""
    at = torch.arange(longest, device="cuda")
    there = at < (cu[1:] - cu[:-1])[:, None]
    rows = torch.where(there, cu[:-1, None] + at, 0)
    return torch.where(there[..., None, None], x[rows].float(), 0.0).transpose(1, 2), there, rows


def _plain_attention(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    q, q_there, q_rows = _padded(s["q"], s["cu_q"], s["max_q"])
    k, k_there, k_rows = _padded(s["k"], s["cu_k"], s["max_k"])
    v = _padded(s["v"], s["cu_k"], s["max_k"])[0]
    k, v = (x.repeat_interleave(group, dim=1) for x in (k, v))
    score = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    if c["cap"] > 0:
        score = c["cap"] * torch.tanh(score / c["cap"])
    n, m = s["cu_q"][1:] - s["cu_q"][:-1], s["cu_k"][1:] - s["cu_k"][:-1]
    i = torch.arange(s["max_q"], device="cuda") + (m - n)[:, None]
    j = torch.arange(s["max_k"], device="cuda")
    distance = j - i[..., None]  # [sequences, rows, keys]
    if s["slopes"] is not None:
        score = score - s["slopes"][:, None, None] * distance.abs()[:, None]
    if s["table"] is not None:
        at = torch.clamp(distance, -c["radius"], c["radius"]) + c["radius"]
        score = score + s["table"][:, at].transpose(0, 1)
    seen = torch.ones_like(distance, dtype=torch.bool)
    if c["left"] >= 0:
        seen &= distance >= -c["left"]
    if c["right"] >= 0:
        seen &= distance <= c["right"]
    if s["prefix"] is not None:
        seen |= j < s["prefix"][:, None, None]
    if c["docs"]:
        seen &= s["doc_q"][q_rows][..., None] == s["doc_k"][k_rows][:, None]
    seen &= k_there[:, None]
    score = torch.where(seen[:, None], score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return out.transpose(1, 2)[q_there].to(s["q"].dtype)


def _plain_linear(s):
    c = s["case"]
    y = torch.matmul(s["x"].float(), s["w"].float().t())
    if s["bias"] is not None:
        y = y + s["bias"]
    if c["act"] == "relu":
        y = torch.clamp(y, min=0.0)
    elif c["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y / math.sqrt(2.0)))
    elif c["act"] == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(DT[c["out"]])


# ------------------------------------------------------------------------------ in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attention": _exact_attention, "linear": _exact_linear}[case["op"]](case, s)


def _exact_rope(case, s):
    r, x = case["rot"], s["x"].double()
    f = torch.tensor(s["freq"], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(f, s["stretch"]).expand(len(x), -1), torch.outer(s["positions"].double(), f))
    first = torch.arange(r // 2, device="cuda") * (2 if case["layout"] == "interleaved" else 1)
    second = first + (1 if case["layout"] == "interleaved" else r // 2)
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _exact_attention(case, s):
    rows, keys = _lengths(case)
    group, c = case["heads"] // case["kv_heads"], case["cap"]
    out, at_q, at_k = [], 0, 0
    for n, m, p in zip(rows, keys, _prefix(case, keys)):
        q = s["q"][at_q : at_q + n].double()
        k, v = (s[x][at_k : at_k + m].double() for x in "kv")
        lo, hi = (torch.from_numpy(x).cuda()[:, None] for x in _span(case, n, m))
        j = torch.arange(m, device="cuda")[None]
        hidden = ~(((j >= lo) & (j < hi)) | (j < p))
        if case["docs"]:
            hidden |= s["doc_q"][at_q : at_q + n, None] != s["doc_k"][None, at_k : at_k + m]
        away = j - (torch.arange(n, device="cuda")[:, None] + m - n)
        heads = []
        for h in range(case["heads"]):
            t = s["scale"] * (q[:, h] @ k[:, h // group].t())
            if c > 0:
                t = c * torch.tanh(t / c)
            if case["bias"] == "slopes":
                t = t - s["slopes"][h].double() * away.abs()
            if case["bias"] == "table":
                t = t + s["table"][h].double()[away.clamp(-case["radius"], case["radius"]) + case["radius"]]
            t = torch.softmax(t.masked_fill(hidden, float("-inf")), -1)
            heads.append(torch.nan_to_num(t, nan=0.0) @ v[:, h // group])
        out.append(torch.stack(heads, 1))
        at_q, at_k = at_q + n, at_k + m
    return torch.cat(out)


def _exact_linear(case, s):
    y = torch.nn.functional.linear(s["x"].double(), s["w"].double(), s["bias"].double() if case["bias"] else None)
    act = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
           "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["act"]]
    y = act(y)
    return y if s["residual"] is None else y + s["residual"].double()
