"""What has no part in a row's result has none in its bits either: finite values of keys that the
row does not see, rows of other sequences, what shared memory held before."""
import pytest
import torch

from crispembed_b200 import binding

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
KINDS = [{}, dict(softcap=20.0), dict(slopes=True), dict(table=True), dict(softcap=20.0, slopes=True)]


def _inputs(dev, dtype, rows, heads, kv, hd):
    g = torch.Generator().manual_seed(rows + heads + hd)
    mk = lambda *s: torch.randn(s, generator=g).to(dtype).to(dev)  # noqa: E731
    return mk(rows, heads, hd), mk(rows, kv, hd), mk(rows, kv, hd)


def _call(t, lens, heads, kind, longest=None, **kw):
    dev = t[0].device
    kind = dict(kind)
    if kind.pop("slopes", False):
        kw["slopes"] = torch.linspace(0.001, 0.05, heads, device=dev)
    if kind.pop("table", False):
        kw["rel_bias"] = torch.linspace(-1, 1, heads * 41, device=dev).view(heads, 41)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    out = binding.attention_masked(*t, cu, cu, longest or max(lens), longest or max(lens), **kw, **kind)
    binding.sync_check()
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,hd", [(HF, 64), (BF, 128)])
@pytest.mark.parametrize("heads,kv", [(2, 2), (3, 1), (5, 1), (4, 1), (24, 2)])
def test_hidden_keys_and_other_texts(cuda, kind, dtype, hd, heads, kv):
    lens = [200, 90, 180]
    t = _inputs(cuda, dtype, sum(lens), heads, kv, hd)
    ref = _call(t, lens, heads, kind, window=(-1, 0))
    # the last 50 keys of the first text grow: the rows in front of them do not see that
    q, k, v = (x.clone() for x in t)
    k[150:200] *= 8
    v[150:200] += 3
    got = _call((q, k, v), lens, heads, kind, window=(-1, 0))
    assert torch.equal(got[:150], ref[:150]) and torch.equal(got[200:], ref[200:])
    assert not torch.equal(got[150:200], ref[150:200])
    # another text's queries and keys
    q, k, v = (x.clone() for x in t)
    q[200:290] *= 40
    k[200:290] *= 5
    got = _call((q, k, v), lens, heads, kind, window=(-1, 0))
    assert torch.equal(got[:200], ref[:200]) and torch.equal(got[290:], ref[290:])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv", [(3, 1), (5, 1), (12, 1), (4, 2)])
def test_a_text_alone_and_among_others(cuda, kind, heads, kv):
    """(At lengths whose keys are not divided among blocks, and with the same longest length.)"""
    lens = [77, 200, 33, 130]
    t = _inputs(cuda, HF, sum(lens), heads, kv, 64)
    ref = _call(t, lens, heads, kind)
    at = 0
    for n in lens:
        alone = tuple(x[at : at + n].clone() for x in t)
        assert torch.equal(_call(alone, [n], heads, kind, longest=200), ref[at : at + n]), n
        at += n


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv", [(3, 1), (5, 1), (12, 1)])
def test_what_ran_before(cuda, kind, heads, kv):
    """Groups that do not divide a tile leave rows of it to what shared memory holds."""
    lens = [70, 200, 150]
    t = _inputs(cuda, HF, sum(lens), heads, kv, 64)
    ref = _call(t, lens, heads, kind)
    loud = tuple((60000 * torch.rand_like(x)) for x in _inputs(cuda, HF, 4000, 8, 8, 64))
    for _ in range(3):
        _call(loud, [200] * 20, 8, {})
        assert torch.equal(_call(t, lens, heads, kind), ref)
