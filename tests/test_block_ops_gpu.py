"""Masked attention, rotary positions and the fused linear layer against 64-bit restatements
(block_ref.py, where the tolerances are derived)."""
import math

import numpy as np
import pytest
import torch

import block_ref as R
from crispembed_b200 import binding, quant
from crispembed_b200.gguf_io import GGML_F16, GGML_Q4_K, GGML_Q8_0

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(6)


def _cu(lens, dev):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=dev)


def _qkv(dev, dtype, rows, keys, heads, kv, hd, seed=0):
    g = torch.Generator().manual_seed(seed + rows + 31 * keys + 7 * heads + hd)
    mk = lambda *s: torch.randn(s, generator=g).to(dtype).to(dev)  # noqa: E731
    return mk(rows, heads, hd), mk(keys, kv, hd), mk(keys, kv, hd)


def _attend(q, k, v, lens_q, lens_k, scale=None, **kw):
    dev = q.device
    out = binding.attention_masked(q, k, v, _cu(lens_q, dev), _cu(lens_k, dev), max(lens_q), max(lens_k), scale=scale,
                                   **kw)
    binding.sync_check()
    ref, tol = R.attention(q, k, v, lens_q, lens_k, q.shape[2] ** -0.5 if scale is None else scale, **kw)
    R.check(out, ref, tol)
    return out


LENS = [[1], [1, 2, 3], [17, 64, 31], [127, 128, 129], [200, 1, 257], [0, 40, 0], [513]]


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("lens", LENS)
def test_attention_open(cuda, lens, dtype):
    _attend(*_qkv(cuda, dtype, sum(lens), sum(lens), 3, 3, 64), lens, lens)


@pytest.mark.parametrize("hd", [8, 16, 24, 32, 40, 56, 64, 72, 80, 96, 104, 120, 128])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_attention_head_dims(cuda, hd, dtype):
    lens = [33, 150]
    _attend(*_qkv(cuda, dtype, 183, 183, 2, 2, hd), lens, lens)


@pytest.mark.parametrize("heads,kv", [(4, 1), (6, 2), (5, 1), (7, 1), (12, 4), (33, 1), (128, 1), (130, 2)])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_shared_heads(cuda, heads, kv, hd):
    lens = [3, 70, 140]
    _attend(*_qkv(cuda, BF, 213, 213, heads, kv, hd), lens, lens, window=(50, 0))


MASKS = [
    dict(window=(-1, 0)), dict(window=(0, 0)), dict(window=(7, 0)), dict(window=(0, -1)), dict(window=(100, 30)),
    dict(window=(-1, 129)), dict(window=(300, -1)), dict(window=(2**31 - 1, 2**31 - 1)),
]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("hd", [64, 80])
def test_attention_windows(cuda, mask, hd):
    lens = [5, 300, 131]
    _attend(*_qkv(cuda, HF, 436, 436, 2, 2, hd), lens, lens, **mask)


@pytest.mark.parametrize("lens_q,lens_k", [
    ([1, 1, 1], [1, 300, 77]),          # one token against the keys before it
    ([3, 20, 1], [130, 20, 513]),
    ([200, 5, 9], [40, 5, 1]),          # more rows than keys: the first rows see nothing when causal
    ([4, 7], [0, 9]),                   # no keys at all
    ([0, 6], [50, 6]),
])
@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (16, 0), (3, 3)])
def test_attention_unequal_lengths(cuda, lens_q, lens_k, window):
    q, k, v = _qkv(cuda, BF, sum(lens_q), sum(lens_k), 4, 2, 64)
    out = _attend(q, k, v, lens_q, lens_k, window=window)
    if lens_q == [200, 5, 9] and window[1] == 0:
        assert (out[:160] == 0).all()
    if lens_k == [0, 9]:
        assert (out[:4] == 0).all()


@pytest.mark.parametrize("prefix", [[0, 0, 0], [5, 100, 1], [1000, 64, -3], [128, 200, 7]])
@pytest.mark.parametrize("window", [(-1, 0), (20, 0), (4, 9)])
def test_attention_prefix(cuda, prefix, window):
    lens = [129, 400, 64]
    _attend(*_qkv(cuda, HF, sum(lens), sum(lens), 2, 1, 64), lens, lens, window=window,
            prefix=torch.tensor(prefix, dtype=torch.int32, device=cuda))


@pytest.mark.parametrize("kind", ["runs", "shuffled", "negative", "disjoint"])
@pytest.mark.parametrize("window", [(-1, -1), (60, 0)])
def test_attention_documents(cuda, kind, window):
    lens = [300, 40, 257]
    n = sum(lens)
    rng = np.random.default_rng(3)
    doc = np.sort(rng.integers(0, 5, n)).astype(np.int32)
    if kind == "shuffled":
        rng.shuffle(doc)
    if kind == "negative":
        doc[100:180] = -1
    doc_q = torch.from_numpy(doc).to(cuda)
    doc_k = doc_q + 100 if kind == "disjoint" else doc_q
    out = _attend(*_qkv(cuda, BF, n, n, 2, 2, 64), lens, lens, window=window, doc_q=doc_q, doc_k=doc_k,
                  prefix=torch.tensor([10, 0, 3], dtype=torch.int32, device=cuda))
    if kind == "negative":
        assert (out[100:180] == 0).all()
    if kind == "disjoint":
        assert (out == 0).all()


@pytest.mark.parametrize("cap", [1.0, 5.0, 50.0])
@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_capped(cuda, cap, dtype, hd):
    lens = [70, 260]
    _attend(*_qkv(cuda, dtype, 330, 330, 4, 2, hd), lens, lens, softcap=cap, scale=0.7, window=(-1, 0))


@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (40, 9)])
@pytest.mark.parametrize("cap", [0.0, 4.0])
def test_attention_slopes(cuda, window, cap):
    lens = [1, 300, 140]
    slopes = torch.tensor([0.5, 0.0, -0.02, 0.004], device=cuda)
    _attend(*_qkv(cuda, HF, sum(lens), sum(lens), 4, 2, 64), lens, lens, slopes=slopes, window=window, softcap=cap)


@pytest.mark.parametrize("radius", [0, 1, 32, 500])
@pytest.mark.parametrize("heads,kv", [(3, 3), (6, 2)])
def test_attention_bias_table(cuda, radius, heads, kv):
    lens = [2, 290, 129]
    g = torch.Generator().manual_seed(radius)
    table = torch.randn(heads, 2 * radius + 1, generator=g).to(cuda)
    _attend(*_qkv(cuda, HF, sum(lens), sum(lens), heads, kv, 32), lens, lens, rel_bias=table)


@pytest.mark.parametrize("low", [-math.inf, torch.finfo(torch.float32).min, -1e30])
@pytest.mark.parametrize("lens_q,lens_k", [([260], [260]), ([1, 30], [140, 30])])
def test_attention_bias_as_mask(cuda, low, lens_q, lens_k):
    """Bias entries of the type's lowest value or -inf: they hide keys, a row that has nothing else
    averages its keys (lowest value: all scores are equal) or gets zeros (-inf)."""
    table = torch.zeros(2, 81)
    table[0, :30] = low    # keys more than 10 before the row
    table[1, :] = low
    out = _attend(*_qkv(cuda, BF, sum(lens_q), sum(lens_k), 2, 2, 64), lens_q, lens_k, rel_bias=table.to(cuda))
    if low == -math.inf:
        assert (out[:, 1] == 0).all()


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("hd", [64, 104])
def test_attention_hidden_keys_hold_anything(cuda, poison, hd):
    """Keys behind a window, of another document, of no sequence: what they hold has no part."""
    lens = [100, 301]
    q, k, v = _qkv(cuda, HF, 430, 430, 2, 2, hd)
    doc = torch.zeros(430, dtype=torch.int32, device=cuda)
    doc[140:150] = 5  # ten keys that only their own rows see
    for t in (q, k, v):
        t[401:] = poison   # behind the last sequence
    k[140:150], v[140:150] = poison, poison
    v[60] = poison         # hidden from the rows in front of it
    cu = _cu(lens, cuda)
    out = binding.attention_masked(q, k, v, cu, cu, 301, 301, window=(-1, 0), doc_q=doc, out=torch.full_like(q, 7.0))
    binding.sync_check()
    ref, tol = R.attention(q[:401], k[:401], v[:401], lens, lens, hd ** -0.5, window=(-1, 0), doc_q=doc[:401],
                           doc_k=doc[:401])
    assert (out[401:] == 7.0).all()
    clean = torch.ones(401, dtype=torch.bool)
    clean[60:100] = clean[140:150] = False
    R.check(out[:401][clean], ref[clean], tol[clean])
    assert not torch.isfinite(out[60:100]).any() and not torch.isfinite(out[140:150]).any()


def test_attention_strides(cuda):
    """Heads before rows, rows of a fused projection, an output of its own layout."""
    lens, n, h, d = [77, 130], 207, 4, 64
    q, k, v = _qkv(cuda, BF, n, n, h, h, d)
    ref = _attend(q, k, v, lens, lens)
    qt, kt, vt = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    out = torch.zeros(h, n + 3, d + 8, dtype=BF, device=cuda)
    view = out.transpose(0, 1)[:n, :, :d]
    cu = _cu(lens, cuda)
    binding.attention_masked(qt, kt, vt, cu, cu, 130, 130, out=view)
    assert torch.equal(view, ref) and (out[:, n:] == 0).all() and (out[:, :, d:] == 0).all()
    fused = torch.cat([q, k, v], 1)
    assert torch.equal(binding.attention_masked(fused[:, :h], fused[:, h:2 * h], fused[:, 2 * h:], cu), ref)


def test_attention_rows_of_no_sequence(cuda):
    q, k, v = _qkv(cuda, HF, 300, 300, 2, 2, 64)
    cu = torch.tensor([10, 60, 60, 200], dtype=torch.int32, device=cuda)
    out = binding.attention_masked(q, k, v, cu, cu, 140, 140, out=torch.full_like(q, 3.0))
    binding.sync_check()
    ref, tol = R.attention(q[10:200], k[10:200], v[10:200], [50, 0, 140], [50, 0, 140], 0.125)
    R.check(out[10:200], ref, tol)
    assert (out[:10] == 3.0).all() and (out[200:] == 3.0).all()


def test_attention_no_key_rows(cuda):
    q = torch.randn(5, 2, 64, device=cuda).half()
    k = torch.empty(0, 2, 64, device=cuda).half()
    doc = torch.zeros(5, dtype=torch.int32, device=cuda)
    for kw in ({}, dict(doc_q=doc, doc_k=doc[:0])):
        for rows in (5, 1):
            out = binding.attention_masked(q, k, k, _cu([rows], cuda), _cu([0], cuda), rows, 0, out=torch.ones_like(q), **kw)
            binding.sync_check()
            assert (out[:rows] == 0).all() and (out[rows:] == 1).all()


@pytest.mark.parametrize("cu_q,cu_k,max_q,max_k", [
    ([0, 64], [0, 64], 32, 64), ([0, 64], [0, 64], 64, 32), ([0, 40, 100], [0, 40, 64], 64, 64),
    ([0, 40, 64], [0, 70, 64], 64, 64), ([-4, 20], [0, 64], 64, 64), ([0, 64], [10, 2], 64, 64),
])
def test_attention_bad_offsets(cuda, cu_q, cu_k, max_q, max_k):
    q, k, v = _qkv(cuda, HF, 64, 64, 2, 2, 64)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    binding.attention_masked(q, k, v, t(cu_q), t(cu_k), max_q, max_k)
    with pytest.raises(binding.CrispEmbedError, match=r"\(5\).*0x106"):
        binding.sync_check()
    binding.sync_check()
    _attend(q, k, v, [64], [64])


def test_attention_far_offsets(cuda):
    """Rows whose element offsets pass 2^31 in a long cache."""
    rows, step = 40000, 57344  # 2.3e9 elements from the first key row to the last
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    cache = torch.empty(rows * step, dtype=HF, device=cuda)
    view = cache.as_strided((rows, 2, 64), (step, 64, 1))
    q, k, v = _qkv(cuda, HF, 70, 300, 2, 1, 64)
    view[rows - 300:, :1], view[rows - 300:, 1:] = k, v
    cu_k = torch.tensor([rows - 300, rows], dtype=torch.int32, device=cuda)
    out = binding.attention_masked(q, view[:, :1], view[:, 1:], _cu([70], cuda), cu_k, 70, 300, window=(-1, 0))
    binding.sync_check()
    ref, tol = R.attention(q, k, v, [70], [300], 0.125, window=(-1, 0))
    R.check(out, ref, tol)


def test_attention_long_single_token(cuda):
    """One row per sequence against thousands of keys: the keys' sums are split and joined."""
    lens_k = [5000, 1, 12345, 127]
    q, k, v = _qkv(cuda, BF, 4, sum(lens_k), 8, 2, 128)
    _attend(q, k, v, [1] * 4, lens_k, window=(-1, 0), softcap=30.0)


FEW = [dict(slopes=[0.1, 0.0, -0.02, 0.3]), dict(radius=40), dict(radius=700, softcap=3.0), dict(prefix=[7, 0, 64, 5]),
       dict(docs=True), dict(softcap=2.0, scale=1.0), dict(scale=-0.2), dict(radius=9, low=True)]


@pytest.mark.parametrize("kw", FEW)
@pytest.mark.parametrize("hd", [40, 64, 128])
@pytest.mark.parametrize("kv,most", [(4, 1), (1, 4), (2, 8)])
def test_attention_few_rows(cuda, kw, hd, kv, most):
    """Up to 16 rows a key head run on a kernel of their own: every mask and bias, keys that end inside
    a step, sequences without rows or keys."""
    lens_q, lens_k = [most, 1, 0, most], [333, 1, 64, 1030]
    q, k, v = _qkv(cuda, BF if hd == 64 else HF, sum(lens_q), sum(lens_k), 4, kv, hd)
    kw, n = dict(kw), sum(lens_k)
    radius, docs, low = kw.pop("radius", None), kw.pop("docs", False), kw.pop("low", False)
    if "slopes" in kw:
        kw["slopes"] = torch.tensor(kw["slopes"], device=cuda)
    if "prefix" in kw:
        kw.update(prefix=torch.tensor(kw["prefix"], dtype=torch.int32, device=cuda), window=(30, 0))
    if radius:
        kw["rel_bias"] = torch.randn(4, 2 * radius + 1, device=cuda)
        if low:
            kw["rel_bias"][1] = -math.inf
            kw["rel_bias"][2] = torch.finfo(FP).min
    if docs:
        kw["doc_k"] = torch.randint(-1, 3, (n,), device=cuda).int()
        kw["doc_q"] = torch.randint(-1, 3, (sum(lens_q),), device=cuda).int()
    _attend(q, k, v, lens_q, lens_k, **kw)


@pytest.mark.parametrize("poison", [math.nan, math.inf])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_few_rows_hidden_keys(cuda, poison, hd):
    lens_q, lens_k = [1, 3], [100, 4000]
    q, k, v = _qkv(cuda, BF, 4, 4140, 4, 2, hd)
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    for t in (k2, v2):
        t[100 + 3000:100 + 3100] = poison  # hidden by the window
        t[4100:] = poison                  # behind the last sequence
    cu = _cu(lens_q, cuda), _cu(lens_k, cuda)
    kw = dict(window=(500, 0))
    out = binding.attention_masked(q2, k2, v2, *cu, 3, 4000, **kw)
    binding.sync_check()
    ref, tol = R.attention(q, k[:4100], v[:4100], lens_q, lens_k, hd ** -0.5, **kw)
    R.check(out, ref, tol)
    v2[100 + 3990] = poison                # seen by the second text's rows
    out = binding.attention_masked(q2, k2, v2, *cu, 3, 4000, **kw)
    R.check(out[:1], ref[:1], tol[:1])
    assert not torch.isfinite(out[1:]).any()


def test_attention_few_rows_bad_offsets(cuda):
    q, k, v = _qkv(cuda, HF, 2, 64, 2, 2, 64)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    for cu_k in ([0, 70, 64], [0, 30, 80], [-1, 30, 64]):
        binding.attention_masked(q, k, v, t([0, 1, 2]), t(cu_k), 1, 64)
        with pytest.raises(binding.CrispEmbedError, match=r"\(5\).*0x106"):
            binding.sync_check()


def test_first_call_of_a_process_is_captured(cuda):
    """The library's device words may be made while the caller's stream is being captured."""
    import subprocess
    import sys
    code = """
import torch
from crispembed_b200 import binding
q = torch.randn(70, 2, 64, device="cuda").half()
cu = torch.tensor([0, 70], dtype=torch.int32, device="cuda")
out = torch.zeros_like(q)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    binding.attention_masked(q, q, q, cu, cu, 70, 70, out=out)
assert (out == 0).all()
g.replay()
ref = binding.attention_masked(q, q, q, cu, cu, 70, 70)
binding.sync_check()
assert torch.equal(out, ref) and (out != 0).any()
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_attention_repeats_overlaps_and_replays(cuda):
    """The same bits again; on two streams at once; captured by two graphs on one stream and
    replayed on two."""
    lens = [300, 511, 64, 200, 17]
    cu = _cu(lens, cuda)
    sets = [_qkv(cuda, BF, sum(lens), sum(lens), 8, 2, 64, seed=s) for s in (1, 2)]
    call = lambda t, **kw: binding.attention_masked(*t, cu, cu, 511, 511, window=(-1, 0), **kw)  # noqa: E731
    ref = [call(t) for t in sets]
    torch.cuda.synchronize()
    assert all(torch.equal(call(t), r) for t, r in zip(sets, ref))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(sets[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref[i]) for i in (0, 1) for o in got[i])
    outs = [torch.empty_like(r) for r in ref]
    graphs = []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(sets[i], out=outs[i])
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, r) for o, r in zip(outs, ref))
    binding.sync_check()


# ------------------------------------------------------------------ rotary positions
ROPES = [  # rot, head_dim
    (64, 64), (32, 64), (128, 128), (2, 8), (6, 8), (34, 40), (50, 80), (80, 80), (20, 24), (256, 256),
]


@pytest.mark.parametrize("dtype", [HF, BF, FP])
@pytest.mark.parametrize("rot,hd", ROPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_layouts(cuda, rot, hd, dtype, interleaved):
    g = torch.Generator().manual_seed(rot + hd)
    x = torch.randn(37, 5, hd, generator=g).to(dtype).to(cuda)
    pos = torch.randint(0, 5000, (37,), generator=g).int()
    rope = binding.Rope(rot)
    out = rope(x, positions=pos.to(cuda), interleaved=interleaved)
    ref, tol = R.rope(x, pos, rot, interleaved, *R.frequencies(rot))
    R.check(out, ref, tol)
    assert torch.equal(out[..., rot:], x[..., rot:])
    y = x.clone()
    assert rope(y, out=y, positions=pos.to(cuda), interleaved=interleaved) is y and torch.equal(y, out)


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=8.0), dict(scaling="ntk", factor=4.0),
                                dict(scaling="yarn", factor=16.0, context=4096),
                                dict(scaling="yarn", factor=2.0, context=512, beta_fast=20.0, beta_slow=2.0),
                                dict(theta=1e6)])
@pytest.mark.parametrize("rot", [64, 96])
def test_rope_scaled_far_positions(cuda, kw, rot):
    x = torch.randn(9, 3, 96, device=cuda)
    pos = torch.tensor([0, 1, -7, 4095, 131071, 1000003, 16777217, 2**31 - 1, -2**31], dtype=torch.int32)
    out = binding.Rope(rot, **kw)(x, positions=pos.to(cuda))
    ref, tol = R.rope(x, pos, rot, False, *R.frequencies(rot, **kw))
    # the 64-bit turns of both sides: 2^31 (f_i off by 2^-51) is off by 2^-20 rad
    R.check(out, ref, tol + pos.double().abs()[:, None, None] * 2.0 ** -50 * x.abs().amax().item())


@pytest.mark.parametrize("lens", [[1], [0, 3, 0, 0, 9], list(range(80)), [700, 1, 1300]])
def test_rope_positions_of_sequences(cuda, lens):
    """Positions are places in the sequences; rows of none stay as they were."""
    n = sum(lens)
    x = torch.randn(n + 9, 4, 64, device=cuda).half()
    cu = _cu(lens, cuda) + 4
    rope = binding.Rope(64)
    pos = torch.tensor(sum((list(range(m)) for m in lens), []), dtype=torch.int32) + 2
    out = rope(x, out=torch.full_like(x, 9.0), cu_seqlens=cu, pos_offset=2)
    ref, tol = R.rope(x[4:n + 4], pos, 64, False, *R.frequencies(64))
    R.check(out[4:n + 4], ref, tol)
    assert (out[:4] == 9.0).all() and (out[n + 4:] == 9.0).all()


@pytest.mark.parametrize("step,heads", [(64 * 7, 64), (64 * 7 + 1, 64), (64 * 7 + 2, 66), (450, 65)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strides(cuda, step, heads, interleaved):
    """Rows and heads at odd distances: narrower accesses, the same numbers."""
    buf = torch.randn(step * 33 + 7, device=cuda).half()
    for shift in (0, 1):
        x = buf[shift:].as_strided((33, 5, 64), (step, heads, 1))
        pos = torch.arange(33, dtype=torch.int32)
        out = binding.Rope(64)(x, positions=pos.to(cuda), interleaved=interleaved)
        ref, tol = R.rope(x, pos, 64, interleaved, *R.frequencies(64))
        R.check(out, ref, tol)


def test_rope_refuses(cuda):
    x = torch.zeros(8, 4, 64, device=cuda).half()
    pos = torch.zeros(8, dtype=torch.int32, device=cuda)
    rope = binding.Rope(64)
    with pytest.raises(binding.CrispEmbedError, match="positions"):
        rope(x)
    with pytest.raises(binding.CrispEmbedError, match="below rot_dim"):
        rope(x[..., :32], positions=pos)
    with pytest.raises(binding.CrispEmbedError, match="positions"):
        rope(x, positions=pos[:7])
    with pytest.raises(binding.CrispEmbedError, match="overlaps"):
        rope(x[:, :2], out=x[:, 1:3], positions=pos)
    with pytest.raises(binding.CrispEmbedError, match="apart"):
        rope(x.as_strided((8, 4, 64), (64, 64, 1)), positions=pos)
    with pytest.raises(binding.CrispEmbedError, match="type"):
        rope(x, out=x.float(), positions=pos)
    assert rope(x[:0], positions=pos[:0]).shape == (0, 4, 64)


# ------------------------------------------------------------------ linear layer
def _linear(dev, wtype, n, k, seed=0):
    rng = np.random.default_rng(seed + n + k)
    raw = quant.quantize((rng.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32), wtype)
    w = binding.gguf_dequantize(wtype, raw, n, k)
    return binding.Linear(wtype, raw, n, k), w, wtype != GGML_F16


def _fused(lin, x, out_dtype, bias=None, act="none", residual=None, **kw):
    layer, w, rounded = lin
    out = layer.fused(x, bias=bias, act=act, residual=residual, out_dtype=out_dtype, **kw)
    binding.sync_check()
    assert out.dtype == out_dtype
    return out, R.linear(x, w, bias, act, residual, out_dtype, rounded)


@pytest.mark.parametrize("wtype", [GGML_F16, GGML_Q8_0, GGML_Q4_K])
@pytest.mark.parametrize("n,k", [(128, 256), (256, 256), (768, 768), (384, 512)])
@pytest.mark.parametrize("m", [1, 2, 7, 33, 130, 300, 1409])
def test_linear_fused_sizes(cuda, wtype, n, k, m):
    g = torch.Generator().manual_seed(m)
    lin = _linear(cuda, wtype, n, k)
    x = torch.randn(m, k, generator=g).half().to(cuda)
    bias, res = torch.randn(n, generator=g).to(cuda), torch.randn(m, n, generator=g).half().to(cuda)
    got, want = _fused(lin, x, HF, bias, "silu", res)
    R.check(got, *want)


@pytest.mark.parametrize("act", list(binding.ACTIVATIONS))
@pytest.mark.parametrize("out_dtype", [HF, BF, FP])
@pytest.mark.parametrize("res_dtype", [None, HF, BF, FP])
@pytest.mark.parametrize("n,m", [(256, 3), (128, 45), (256, 300), (256, 1301), (128, 2500)])
def test_linear_fused_epilogues(cuda, act, out_dtype, res_dtype, n, m):
    g = torch.Generator().manual_seed(m)
    lin = _linear(cuda, GGML_F16, n, 128)
    x = 3 * torch.randn(m, 128, generator=g).half().to(cuda)
    res = None if res_dtype is None else torch.randn(m, n, generator=g).to(res_dtype).to(cuda)
    for bias in (None, torch.randn(n, generator=g).to(cuda)):
        got, want = _fused(lin, x, out_dtype, bias, act, res)
        R.check(got, *want)


@pytest.mark.parametrize("m", [300, 3000])
def test_linear_fused_beside_forward(cuda, m):
    """Without residual and with the activations that ceb_linear_forward has: the same function, held to
    the same bound (few rows run on another kernel, whose sums have another order); where both
    run the tcgen05 kernel, the same bits."""
    layer, w, rounded = _linear(cuda, GGML_Q8_0, 256, 256)
    x = torch.randn(m, 256, device=cuda).half()
    bias = torch.randn(256, device=cuda)
    for gelu in (False, True):
        for dt in (HF, FP):
            act = "gelu" if gelu else "none"
            a, b = layer.fused(x, bias=bias, act=act, out_dtype=dt), layer(x, bias=bias, gelu=gelu, out_f16=dt == HF)
            for y in (a, b):
                R.check(y, *R.linear(x, w, bias, act, None, dt, rounded))
            assert m == 300 or torch.equal(a, b)


@pytest.mark.parametrize("n", [128, 256])
@pytest.mark.parametrize("m", [1, 5, 77, 300, 2391])
@pytest.mark.parametrize("dtype", [HF, FP])
def test_linear_fused_strides_and_in_place(cuda, n, m, dtype):
    lin = _linear(cuda, GGML_F16, n, 192)
    g = torch.Generator().manual_seed(n + m)
    x = torch.randn(m, 200, generator=g).half().to(cuda)[:, :192]
    wide = torch.randn(m, n + 24, generator=g).to(dtype).to(cuda)
    keep = wide.clone()
    res = wide[:, 8:n + 8]
    bias = torch.randn(n + 1, generator=g).to(cuda)[1:]
    got, want = _fused(lin, x, dtype, bias, "gelu", res.clone())
    R.check(got, *want)
    assert lin[0].fused(x, bias=bias, act="gelu", residual=res, out=res) is res
    assert torch.equal(res, got)
    assert torch.equal(wide[:, :8], keep[:, :8]) and torch.equal(wide[:, n + 8:], keep[:, n + 8:])
    # a longer buffer's rows behind m stay
    tall = torch.full((m + 40, n), 5.0, dtype=dtype, device=cuda)
    lin[0].fused(x, bias=bias, act="gelu", residual=keep[:, 8:n + 8], out=tall[:m])
    assert torch.equal(tall[:m], got) and (tall[m:] == 5.0).all()


def test_linear_fused_infinities(cuda):
    """A row that holds NaN or infinities keeps them to itself."""
    lin = _linear(cuda, GGML_F16, 256, 128)
    x = torch.randn(40, 128, device=cuda).half()
    ref = lin[0].fused(x, act="silu", residual=torch.zeros(40, 256, device=cuda), out_dtype=FP)
    y = x.clone()
    y[7], y[9, 3] = math.nan, math.inf
    got = lin[0].fused(y, act="silu", residual=torch.zeros(40, 256, device=cuda), out_dtype=FP)
    assert torch.isnan(got[7]).all() and not torch.isfinite(got[9]).all()
    same = torch.ones(40, dtype=torch.bool)
    same[7] = same[9] = False
    assert torch.equal(got[same], ref[same])


def test_linear_fused_refuses(cuda):
    layer, _, _ = _linear(cuda, GGML_F16, 128, 128)
    x = torch.zeros(8, 128, device=cuda).half()
    big = torch.zeros(20, 128, device=cuda).half()
    bad = lambda match: pytest.raises(binding.CrispEmbedError, match=match)  # noqa: E731
    with bad("activation"):
        layer.fused(x, act="tanh")
    with bad("fp16"):
        layer.fused(x.float())
    with bad("fp16"):
        layer.fused(x[:, :64])
    with bad("residual"):
        layer.fused(x, residual=big)
    with bad("bias"):
        layer.fused(x, bias=torch.zeros(127, device=cuda))
    with bad("overlaps"):
        layer.fused(x, out=x)
    with bad("overlaps"):
        layer.fused(x, residual=big[:8], out=big[1:9])
    with bad("overlaps"):
        layer.fused(x, residual=big[:8], out=big.view(BF)[:8])
    with bad("strides"):
        layer.fused(x, out=torch.zeros(8, 131, device=cuda).half()[:, :128])
    with bad("aligned"):
        layer.fused(x, out=torch.zeros(8 * 128 + 4, device=cuda).half()[4:].view(8, 128))
    assert layer.fused(x[:0]).shape == (0, 128)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("captured", [False, True])
def test_block_of_an_encoder(cuda, captured):
    """QKV product, rotation of Q and K in place, attention, output product added to the residual
    stream in place: each stage against 64 bits on the stage's own inputs, eager and captured."""
    h, d, lens = 4, 64, [130, 1, 77, 300]
    w = h * d
    n = sum(lens)
    cu = _cu(lens, cuda)
    qkv_l, o_l = _linear(cuda, GGML_Q8_0, 3 * w, w, 1), _linear(cuda, GGML_Q8_0, w, w, 2)
    rope = binding.Rope(d, scaling="linear", factor=2.0)
    stream = torch.randn(n, w, device=cuda)
    x = stream.half()
    bias = torch.randn(3 * w, device=cuda)
    slopes = torch.tensor([0.1, 0.05, 0.02, 0.01], device=cuda)

    def block(stream):
        qkv = qkv_l[0].fused(x, bias=bias, out_dtype=HF)
        qk = qkv.view(n, 3 * h, d)[:, :2 * h]
        before = qk.clone()
        rope(qk, out=qk, cu_seqlens=cu)
        t = qkv.view(n, 3 * h, d)
        att = binding.attention_masked(t[:, :h], t[:, h:2 * h], t[:, 2 * h:], cu, cu, 300, 300, slopes=slopes)
        o_l[0].fused(att.view(n, w), residual=stream, out=stream)
        return qkv, before, att

    out = stream.clone()
    if captured:
        block(out)  # (the library's device words exist from here on)
        torch.cuda.synchronize()
        out.copy_(stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            qkv, before, att = block(out)
        g.replay()
    else:
        qkv, before, att = block(out)
    binding.sync_check()
    t = qkv.view(n, 3 * h, d)
    ref, tol = R.linear(x, qkv_l[1], bias, "none", None, HF, True)
    R.check(torch.cat([before, t[:, 2 * h:]], 1).reshape(n, 3 * w), ref, tol)
    pos = torch.tensor(sum((list(range(m)) for m in lens), []), dtype=torch.int32)
    R.check(t[:, :2 * h], *R.rope(before, pos, d, False, *R.frequencies(d, scaling="linear", factor=2.0)))
    R.check(att, *R.attention(t[:, :h], t[:, h:2 * h], t[:, 2 * h:], lens, lens, 0.125, slopes=slopes))
    R.check(out, *R.linear(att.view(n, w), o_l[1], None, "none", stream, FP, True))
