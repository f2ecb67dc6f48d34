"""Refusals of the attention block's operators that need no device: bad arguments are
reported with status 1 or 2 before anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

from crispembed_b200 import binding


@pytest.fixture(scope="module")
def lib():
    return binding.load_library()


P = 1 << 20  # an aligned address that no refused call may touch


def _attn(**kw):
    d = dict(dtype=binding.ACT_F16, n_head=4, n_head_kv=2, head_dim=64, n_seqs=1, q_rows=8, k_rows=8, max_q=8, max_k=8,
             q_row_stride=256, q_head_stride=64, k_row_stride=128, k_head_stride=64, v_row_stride=128,
             v_head_stride=64, out_row_stride=256, out_head_stride=64, d_cu_q=P, d_cu_k=P, scale=0.125, softcap=0.0,
             window_left=-1, window_right=-1)
    assert not set(kw) - {n for n, _ in binding._AttnParams._fields_}
    return binding._AttnParams(**{**d, **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=binding.ACT_F32), 1),
    (dict(dtype=7), 1),
    (dict(n_head=0), 1),
    (dict(n_head_kv=0), 1),
    (dict(n_head_kv=3), 1),
    (dict(n_head=258, n_head_kv=2), 1),
    (dict(head_dim=4), 2),
    (dict(head_dim=60), 2),
    (dict(head_dim=136), 2),
    (dict(n_seqs=-1), 1),
    (dict(q_rows=-1), 1),
    (dict(max_k=-1), 1),
    (dict(scale=float("nan")), 1),
    (dict(scale=float("inf")), 1),
    (dict(softcap=-1.0), 1),
    (dict(softcap=float("inf")), 1),
    (dict(softcap=1e-16), 1),
    (dict(softcap=2e30), 1),
    (dict(scale=-2e15), 1),
    (dict(window_left=-2), 1),
    (dict(window_right=-2), 1),
    (dict(d_doc_q=P), 1),
    (dict(d_doc_k=P), 1),
    (dict(d_slopes=P, d_rel_bias=P), 1),
    (dict(d_rel_bias=P, rel_bias_radius=-1), 1),
    (dict(d_rel_bias=P, rel_bias_radius=1 << 25), 1),
    (dict(d_cu_q=None), 1),
    (dict(d_cu_k=None), 1),
    (dict(q_row_stride=252), 1),
    (dict(k_head_stride=60), 1),
    (dict(v_row_stride=64), 1),      # rows run into the next row's heads
    (dict(out_row_stride=128), 1),
    (dict(q_head_stride=0), 1),
    (dict(k_row_stride=-128), 1),
    (dict(k_row_stride=1 << 42), 1),
])
def test_attention_masked_refuses(lib, kw, status):
    p = _attn(**kw)
    assert lib.ceb_attention_masked(ctypes.byref(p), P, P + (1 << 21), P + (1 << 22), P + (1 << 23), None) == status
    assert "attention_masked" in binding.last_error()


def test_attention_masked_refuses_pointers(lib):
    q, k, v, o = (P + (i << 20) for i in range(4))
    call = lambda *t, p=_attn(): lib.ceb_attention_masked(ctypes.byref(p), *t, None)  # noqa: E731
    assert lib.ceb_attention_masked(None, q, k, v, o, None) == 1
    for t in ((None, k, v, o), (q, None, v, o), (q, k, None, o), (q, k, v, None), (q + 8, k, v, o), (q, k + 2, v, o),
              (q, k, v + 8, o), (q, k, v, o + 4)):
        assert call(*t) == 1
    # out overlapping an input, whole or in part
    for t in ((q, k, v, q), (q, k, v, k), (q, k, v, v + 16), (q, k, v, q + 16)):
        assert call(*t) == 1
        assert "overlaps" in binding.last_error()


@pytest.mark.parametrize("kw", [dict(n_seqs=0), dict(q_rows=0), dict(max_q=0)])
def test_attention_masked_nothing_to_do(lib, kw):
    p = _attn(**kw)
    assert lib.ceb_attention_masked(ctypes.byref(p), None, None, None, None, None) == 0


@pytest.mark.parametrize("args", [
    (0, 1e4, 0, 1.0, 0, 32.0, 1.0),
    (63, 1e4, 0, 1.0, 0, 32.0, 1.0),
    (258, 1e4, 0, 1.0, 0, 32.0, 1.0),
    (64, 1.0, 0, 1.0, 0, 32.0, 1.0),
    (64, float("nan"), 0, 1.0, 0, 32.0, 1.0),
    (64, 1e4, 4, 1.0, 0, 32.0, 1.0),
    (64, 1e4, -1, 1.0, 0, 32.0, 1.0),
    (64, 1e4, 1, 0.5, 0, 32.0, 1.0),
    (64, 1e4, 1, float("inf"), 0, 32.0, 1.0),
    (2, 1e4, 2, 2.0, 0, 32.0, 1.0),
    (64, 1e4, 3, 2.0, 0, 32.0, 1.0),
    (64, 1e4, 3, 2.0, 2048, 1.0, 1.0),
    (64, 1e4, 3, 2.0, 2048, 32.0, 0.0),
])
def test_rope_create_refuses(lib, args):
    assert lib.ceb_rope_create(*args) is None
    assert "rope_create" in binding.last_error()


def test_null_handles(lib):
    assert lib.ceb_rope_forward(None, P, P, 0, 1, 1, 64, 64, 64, 64, 64, 0, P, None, 0, 0, None) == 1
    assert lib.ceb_linear_fused(None, P, 64, 1, None, 0, None, 0, 0, 0, P, 64, None) == 1
    lib.ceb_rope_free(None)
    lib.ceb_linear_free(None)


def test_params_layout():
    """The ctypes structure has the size a C compiler gives ceb_attn_params: 9 ints padded to 40
    bytes, 8 strides, 2 pointers, 4 four-byte values, 5 pointers, an int padded to 8."""
    assert ctypes.sizeof(binding._AttnParams) == 40 + 64 + 16 + 16 + 40 + 8


def test_wrappers_refuse_host_tensors_and_bad_types():
    q = torch.zeros(4, 2, 64, dtype=torch.float16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(binding.CrispEmbedError, match="CUDA"):
        binding.attention_masked(q, q, q, cu)
    with pytest.raises(binding.CrispEmbedError, match="fp16 or bf16"):
        binding.attention_masked(q.float(), q.float(), q.float(), cu)
    with pytest.raises(binding.CrispEmbedError, match="fp16 or bf16"):
        binding.attention_masked(q, q.bfloat16(), q, cu)
    with pytest.raises(binding.CrispEmbedError, match="expected"):
        binding.attention_masked(q, q[..., :32], q, cu)
    with pytest.raises(binding.CrispEmbedError, match="contiguous"):
        binding.attention_masked(q.transpose(1, 2), q.transpose(1, 2), q.transpose(1, 2), cu)
    with pytest.raises(binding.CrispEmbedError, match="scaling"):
        binding.Rope(64, scaling="cubic")


def test_frequencies_restated():
    """The test oracle's frequencies: hand-computed values of every scaling."""
    from block_ref import frequencies
    f, s = frequencies(4, theta=100.0)
    assert np.allclose(f, [1.0, 0.1]) and s == 1.0
    assert np.allclose(frequencies(4, 100.0, "linear", 4.0)[0], [0.25, 0.025])
    assert np.allclose(frequencies(4, 100.0, "ntk", 4.0)[0], [1.0, 1 / 40])  # theta 100 * 4^2
    f, s = frequencies(64, 10000.0, "yarn", 4.0, 4096)
    plain = frequencies(64)[0]
    assert np.allclose(f[0], plain[0]) and np.allclose(f[-1], plain[-1] / 4) and np.isclose(s, 1 + 0.1 * np.log(4.0))
    assert ((f <= plain + 1e-15) & (f >= plain / 4 - 1e-15)).all()
