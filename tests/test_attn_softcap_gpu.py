"""Capped scores of masked attention where the cap is far above them, or only some of them: the
capped score has the bits of a score, whatever the cap (block_rows_ref.py has the bound, without a
term in the cap)."""
import pytest
import torch

import block_ref as R
from block_rows_ref import attention_rows
from crispembed_b200 import binding

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
CAPS = [3.0, 64.0, 65.0, 1e3, 1e4, 1e5, 1e6, 1e9, 1e30]


def _attend(dev, dtype, rows, keys, heads, kv, hd, loud=None, **kw):
    g = torch.Generator().manual_seed(rows + 3 * keys + hd)
    mk = lambda *s: torch.randn(s, generator=g).to(dtype).to(dev)  # noqa: E731
    q, k, v = mk(rows, heads, hd), mk(keys, kv, hd), mk(keys, kv, hd)
    if loud:  # rows whose scores pass the cap, next to rows whose scores are far below it
        q[1::5] *= loud
    kw = {n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (rows, keys))
    out = binding.attention_masked(q, k, v, cu_q, cu_k, rows, keys, **kw)
    binding.sync_check()
    scale = kw.pop("scale", hd ** -0.5)
    R.check(out, *attention_rows(q, k, v, torch.arange(rows), scale, **kw))


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("dtype,hd", [(HF, 64), (BF, 128), (HF, 40)])
@pytest.mark.parametrize("rows,heads,kv", [(1, 4, 1), (4, 4, 2), (16, 2, 2)])
def test_few_rows(cuda, cap, dtype, hd, rows, heads, kv):
    _attend(cuda, dtype, rows, 700, heads, kv, hd, softcap=cap)


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("dtype,hd", [(HF, 64), (BF, 128)])
@pytest.mark.parametrize("kind", ["cap", "slopes", "table", "negative"])
def test_tiles(cuda, cap, dtype, hd, kind):
    """Scores in registers (cap alone) and prepared ones (cap with a bias, scales below zero)."""
    g = torch.Generator().manual_seed(5)
    kw = {"cap": {}, "slopes": dict(slopes=torch.tensor([0.01, 0.2])), "negative": dict(scale=-0.2),
          "table": dict(rel_bias=torch.randn(2, 81, generator=g))}[kind]
    _attend(cuda, dtype, 200, 300, 2, 1, hd, softcap=cap, window=(-1, 0), **kw)


@pytest.mark.parametrize("cap,loud", [(2.0, 8.0), (50.0, 64.0), (1e3, 1024.0), (4e3, 8192.0)])
@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("slopes", [False, True])
def test_scores_on_both_sides_of_the_cap(cuda, cap, loud, rows, slopes):
    kw = dict(slopes=torch.tensor([0.01, 0.2])) if slopes else {}
    for dtype, hd in ((HF, 64), (BF, 128)):
        _attend(cuda, dtype, rows, 500, 2, 1, hd, loud=loud, softcap=cap, **kw)
