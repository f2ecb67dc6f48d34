"""Numbers that the C entries' 32 bits do not hold are refused by the wrappers, not cut."""
import pytest
import torch

from crispembed_b200 import binding


@pytest.mark.parametrize("kw", [dict(rot_dim=2**32 + 64), dict(rot_dim=64, context=2**32 + 4096, scaling="yarn", factor=2.0),
                                dict(rot_dim=64, context=-2**31 - 1)])
def test_rope_plan(kw):
    with pytest.raises(binding.CrispEmbedError, match="32-bit"):
        binding.Rope(**kw)


@pytest.mark.parametrize("offset", [2**31, 2**32, 2**32 + 3, -2**31 - 1])
def test_rope_offset(offset):
    rope = object.__new__(binding.Rope)  # (a plan needs a device; the call is refused before it is looked at)
    rope._h = None
    with pytest.raises(binding.CrispEmbedError, match="pos_offset"):
        rope(torch.zeros(2, 1, 64), cu_seqlens=torch.tensor([0, 2], dtype=torch.int32), pos_offset=offset)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(window=(2**31, 0)), dict(window=(0, 2**40)), dict(max_q=2**32 + 4), dict(max_k=2**31),
                                dict(scale=1e39), dict(softcap=1e39)])
def test_attention(cuda, kw):
    q = torch.zeros(4, 2, 64, dtype=torch.float16, device=cuda)
    cu = torch.tensor([0, 4], dtype=torch.int32, device=cuda)
    with pytest.raises(binding.CrispEmbedError, match="32 bits|scale beyond|softcap must"):
        binding.attention_masked(q, q, q, cu, **{**dict(max_q=4, max_k=4), **kw})
    out = binding.attention_masked(q, q, q, cu, max_q=4, max_k=4, window=(2**31 - 1, 0))
    binding.sync_check()
    assert (out == 0).all()
