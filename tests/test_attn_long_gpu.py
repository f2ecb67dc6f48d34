"""Masked attention over long sequences: documents on more chunks of keys than the loading warp's
cache of ranges has slots (256; chunks of 64 or 96 keys)."""
import pytest
import torch

import block_ref as R
from block_rows_ref import attention_rows
from crispembed_b200 import binding
from docs_search import documents

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _attend(dev, dtype, rows, keys, heads, kv, hd, kind, **kw):
    """One sequence in documents; every 97th row against 64 bits."""
    g = torch.Generator().manual_seed(rows + 3 * keys + hd)
    mk = lambda *s: torch.randn(s, generator=g).to(dtype).to(dev)  # noqa: E731
    q, k, v = mk(rows, heads, hd), mk(keys, kv, hd), mk(keys, kv, hd)
    doc = torch.from_numpy(documents(keys, kind)).int()
    doc_q = doc[-rows:] if rows > 1000 else doc[torch.linspace(0, keys - 1, rows).long()]
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (rows, keys))
    call = dict(kw, doc_q=doc_q.contiguous().to(dev), doc_k=doc.to(dev))
    ref = dict(kw)
    if "prefix" in kw:
        call["prefix"] = torch.tensor([kw["prefix"]], dtype=torch.int32, device=dev)
    out = binding.attention_masked(q, k, v, cu_q, cu_k, rows, keys, **call)
    binding.sync_check()
    some = torch.arange(0, rows, 97 if rows > 1000 else 3)
    R.check(out[some.to(dev)], *attention_rows(q, k, v, some, hd ** -0.5, doc_q=doc_q, doc_k=doc, **ref))


@pytest.mark.parametrize("dtype,hd,heads,kv,keys,kw", [
    (HF, 64, 2, 1, 33000, {}),                       # 96 keys a chunk
    (BF, 128, 2, 2, 20000, {}),                      # 64
    (HF, 40, 3, 1, 20000, dict(softcap=20.0)),
    (HF, 128, 1, 1, 40000, dict(window=(-1, 0))),
])
@pytest.mark.parametrize("kind", ["runs", "far", "gaps"])
def test_documents_of_long_rows(cuda, dtype, hd, heads, kv, keys, kw, kind):
    _attend(cuda, dtype, keys, keys, heads, kv, hd, kind, **kw)


@pytest.mark.parametrize("dtype,hd,keys,bias,kw", [
    (HF, 64, 17000, "slopes", {}),
    (BF, 128, 18000, "table", {}),
    (HF, 128, 33500, "slopes", dict(window=(-1, 0))),
    (BF, 64, 20000, None, dict(window=(1024, 0), prefix=1000)),   # 96 keys a chunk: the positions jump
    (HF, 96, 20000, None, dict(window=(1024, 0), prefix=100)),
    (HF, 64, 20000, "table", dict(window=(300, 300), prefix=9000)),
])
def test_documents_where_positions_jump(cuda, dtype, hd, keys, bias, kw):
    """The chunk near a row comes first where there is a bias, and windows lie behind a prefix."""
    g = torch.Generator().manual_seed(keys)
    if bias == "slopes":
        kw = dict(kw, slopes=torch.tensor([0.01, 0.0002], device=cuda))
    if bias == "table":
        kw = dict(kw, rel_bias=torch.randn(2, 201, generator=g).to(cuda))
    for kind in ("runs", "far"):
        _attend(cuda, dtype, keys, keys, 2, 1, hd, kind, **kw)


@pytest.mark.parametrize("kind", ["runs", "far"])
def test_documents_of_few_rows_and_many_keys(cuda, kind):
    """The keys of a tile divided among a cluster's blocks, more than 256 chunks each."""
    _attend(cuda, HF, 200, 140000, 1, 1, 128, kind)


def test_rows_of_a_long_text_computed_again(cuda):
    """A hidden key that holds NaN: rows of 200,000 keys are computed again one by one, for longer than
    the block's other warps wait for anything else, and the block has another text to do."""
    n, keys, short = 600, 200000, 100
    g = torch.Generator(device=cuda).manual_seed(2)
    total = keys + (n - 1) * short
    q = torch.randn(n, 32, 64, generator=g, device=cuda).half()
    k, v = (torch.randn(total, 1, 64, generator=g, device=cuda).half() for _ in "kv")
    doc_q = torch.zeros(n, dtype=torch.int32, device=cuda)
    doc_k = torch.zeros(total, dtype=torch.int32, device=cuda)
    doc_k[keys // 2] = -1
    cu_q = torch.arange(n + 1, dtype=torch.int32, device=cuda)
    cu_k = torch.cat([torch.zeros(1), keys + short * torch.arange(n)]).int().to(cuda)
    ref = binding.attention_masked(q, k, v, cu_q, cu_k, 1, keys, doc_q=doc_q, doc_k=doc_k)
    binding.sync_check()
    v[keys // 2] = float("nan")
    out = binding.attention_masked(q, k, v, cu_q, cu_k, 1, keys, doc_q=doc_q, doc_k=doc_k)
    binding.sync_check()
    assert torch.equal(out[1:], ref[1:])
    v[keys // 2] = 0
    want = attention_rows(q[:1], k[:keys], v[:keys], torch.arange(1), 0.125, doc_q=doc_q[:1], doc_k=doc_k[:keys])
    R.check(ref[:1], *want)
    R.check(out[:1], *want)
