"""ctypes binding of libcrispembed.so (include/crispembed.h, include/ceb_ops.h).

``CrispEmbed`` mirrors the reference's Python class (python/crispembed/_binding.py:
``CrispEmbed(model_path, n_threads).encode(texts)``) for the embedding entry
points this library implements, plus ``encode_ids`` for token-id input.  The
operator-level wrappers (``MoELayer``, ``matmul``, ``pool_l2``) take torch CUDA
tensors purely as device buffers.

There is no CPU fallback: if the CUDA library is missing this module raises.
"""
from __future__ import annotations

import ctypes
import os
import struct
from typing import List, Optional, Sequence, Union

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libcrispembed.so")

TYPE_F32, TYPE_F16, TYPE_Q8_0, TYPE_Q4_K = 0, 1, 8, 12
ACT_F32, ACT_BF16, ACT_F16 = 0, 1, 2

_lib = None


class CrispEmbedError(RuntimeError):
    pass


class _Hparams(ctypes.Structure):
    _fields_ = [
        ("n_vocab", ctypes.c_int32), ("n_max_tokens", ctypes.c_int32), ("n_embd", ctypes.c_int32),
        ("n_head", ctypes.c_int32), ("n_layer", ctypes.c_int32), ("n_intermediate", ctypes.c_int32),
        ("n_output", ctypes.c_int32), ("layer_norm_eps", ctypes.c_float), ("n_experts", ctypes.c_int32),
        ("n_experts_per_tok", ctypes.c_int32),
    ]


class _AttnParams(ctypes.Structure):
    _fields_ = (
        [(n, ctypes.c_int) for n in ("dtype", "n_head", "n_head_kv", "head_dim", "n_seqs", "q_rows", "k_rows", "max_q",
                                     "max_k")]
        + [(n, ctypes.c_int64) for n in ("q_row_stride", "q_head_stride", "k_row_stride", "k_head_stride",
                                         "v_row_stride", "v_head_stride", "out_row_stride", "out_head_stride")]
        + [("d_cu_q", ctypes.c_void_p), ("d_cu_k", ctypes.c_void_p), ("scale", ctypes.c_float),
           ("softcap", ctypes.c_float), ("window_left", ctypes.c_int), ("window_right", ctypes.c_int)]
        + [(n, ctypes.c_void_p) for n in ("d_prefix", "d_doc_q", "d_doc_k", "d_slopes", "d_rel_bias")]
        + [("rel_bias_radius", ctypes.c_int)])


# ceb_attn_params as bytes (the same layout; packing is quicker than filling the structure)
_ATTN_PARAMS = struct.Struct("@9i4x8q2P2f2i5Pi4x")


def load_library(path: Optional[str] = None):
    """Load (never build) the shared library; raises if it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    path = path or os.environ.get("CRISPEMBED_LIB") or LIB_PATH
    if not os.path.exists(path):
        raise CrispEmbedError(f"{path} not found: build it with `python -m crispembed_b200.build`")
    L = ctypes.CDLL(path)
    vp, cp, ip, fp = ctypes.c_void_p, ctypes.c_char_p, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_float)
    i32p = ctypes.POINTER(ctypes.c_int32)
    sig = {
        "crispembed_init": ([cp, ctypes.c_int], vp),
        "ceb_init_ex": ([cp, ctypes.c_int, ctypes.c_int], vp),
        "crispembed_free": ([vp], None),
        "crispembed_set_dim": ([vp, ctypes.c_int], None),
        "crispembed_set_prefix": ([vp, cp], None),
        "crispembed_get_prefix": ([vp], cp),
        "crispembed_set_gpu_backend": ([cp], None),
        "crispembed_get_hparams": ([vp], ctypes.POINTER(_Hparams)),
        "crispembed_encode": ([vp, cp, ip], fp),
        "crispembed_encode_batch": ([vp, ctypes.POINTER(cp), ctypes.c_int, ip], fp),
        "crispembed_encode_ids_batch": ([vp, i32p, i32p, ctypes.c_int, ip], fp),
        "crispembed_encode_ids_device": ([vp, vp, i32p, ctypes.c_int, vp, ip, vp], ctypes.c_int),
        "crispembed_stream": ([vp], vp),
        "ceb_encode_ids_routes": ([vp, i32p, i32p, ctypes.c_int, vp, vp, vp], ctypes.c_int),
        "ceb_moe_block_count": ([vp], ctypes.c_int),
        "crispembed_has_sparse": ([vp], ctypes.c_int),
        "crispembed_has_colbert": ([vp], ctypes.c_int),
        "crispembed_is_reranker": ([vp], ctypes.c_int),
        "ceb_moe_layer_create": ([ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, vp,
                                  ctypes.c_int, vp, vp, vp], vp),
        "ceb_moe_layer_free": ([vp], None),
        "ceb_moe_workspace_size": ([vp, ctypes.c_int], ctypes.c_size_t),
        "ceb_moe_ffn": ([vp, vp, ctypes.c_int, ctypes.c_int, vp, vp, vp, vp, vp, vp, ctypes.c_size_t, vp],
                        ctypes.c_int),
        "ceb_moe_ffn_static": ([vp, vp, ctypes.c_int, ctypes.c_int, vp, vp], ctypes.c_int),
        "ceb_moe_workspace_routing": ([vp, ctypes.c_int, vp, ctypes.POINTER(vp), ctypes.POINTER(vp),
                                       ctypes.POINTER(vp), ctypes.POINTER(vp)], ctypes.c_int),
        "ceb_gguf_dequantize": ([ctypes.c_int, vp, ctypes.c_int64, ctypes.c_int64, vp], ctypes.c_int),
        "ceb_ep_create": ([ctypes.c_int] * 7, vp),
        "ceb_ep_ipc_handle": ([vp, vp], ctypes.c_int),
        "ceb_ep_connect": ([vp, vp], ctypes.c_int),
        "ceb_ep_set_timeout_ms": ([vp, ctypes.c_int], None),
        "ceb_ep_free": ([vp], None),
        "ceb_ep_attach": ([vp, vp], ctypes.c_int),
        "ceb_moe_ffn_ep": ([vp, vp, vp, ctypes.c_int, ctypes.c_int, vp, vp, ctypes.c_size_t, vp], ctypes.c_int),
        "ceb_moe_route_ln": ([vp, vp, vp, ctypes.c_int, vp, vp, ctypes.c_float, vp, vp, vp, vp, vp, vp,
                              ctypes.c_size_t, vp], ctypes.c_int),
        "ceb_pool_l2": ([vp, vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, vp, vp], ctypes.c_int),
        "ceb_tokenizer_load": ([ctypes.c_char_p, ctypes.c_int], vp),
        "ceb_tokenizer_encode": ([vp, ctypes.c_char_p, vp, ctypes.c_int], ctypes.c_int),
        "ceb_tokenizer_kind_of": ([vp], ctypes.c_int),
        "ceb_tokenizer_free": ([vp], None),
        "crispembed_encode_tokens": ([vp, ctypes.c_char_p, vp, vp], vp),
        "crispembed_encode_tokens_raw": ([vp, ctypes.c_char_p, vp, vp], vp),
        "crispembed_last_token_ids": ([vp], vp),
        "crispembed_token_str": ([vp, ctypes.c_int32], ctypes.c_char_p),
        "crispembed_tokenizer_kind": ([vp], ctypes.c_int),
        "ceb_attention_forward": ([vp, ctypes.c_int, vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, vp, vp],
                                  ctypes.c_int),
        "ceb_matmul": ([ctypes.c_int, vp, ctypes.c_int, ctypes.c_int, vp, ctypes.c_int, vp, ctypes.c_int,
                        ctypes.c_int, vp, vp], ctypes.c_int),
        "ceb_linear_create": ([ctypes.c_int, vp, ctypes.c_int, ctypes.c_int], vp),
        "ceb_linear_forward": ([vp, vp, ctypes.c_int, vp, ctypes.c_int, ctypes.c_int, vp, vp], ctypes.c_int),
        "ceb_linear_fused": ([vp, vp, ctypes.c_int64, ctypes.c_int, vp, ctypes.c_int, vp, ctypes.c_int, ctypes.c_int64,
                              ctypes.c_int, vp, ctypes.c_int64, vp], ctypes.c_int),
        "ceb_linear_free": ([vp], None),
        "ceb_attention_masked": ([vp, vp, vp, vp, vp, vp], ctypes.c_int),
        "ceb_rope_create": ([ctypes.c_int, ctypes.c_double, ctypes.c_int, ctypes.c_double, ctypes.c_int,
                             ctypes.c_double, ctypes.c_double], vp),
        "ceb_rope_forward": ([vp, vp, vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int64,
                              ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, vp, vp, ctypes.c_int,
                              ctypes.c_int, vp], ctypes.c_int),
        "ceb_rope_free": ([vp], None),
        "ceb_launch_count": ([], ctypes.c_longlong),
        "ceb_profile_enable": ([ctypes.c_int], None),
        "ceb_profile_read": ([ctypes.POINTER(ctypes.c_longlong), ctypes.POINTER(ctypes.c_double),
                              ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double), ctypes.c_int],
                             ctypes.c_int),
        "ceb_last_error": ([], cp),
        "ceb_sync_check": ([vp], ctypes.c_int),
    }
    for name, (args, res) in sig.items():
        f = getattr(L, name)
        f.argtypes = args
        f.restype = res
    _lib = L
    return L


def last_error() -> str:
    m = load_library().ceb_last_error()
    return m.decode() if m else ""


def _check(rc: int, what: str):
    if rc != 0:
        raise CrispEmbedError(f"{what} failed ({rc}): {last_error()}")


def _stream_ptr(stream) -> Optional[int]:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return int(stream)


def _ptr(t) -> Optional[int]:
    return None if t is None else t.data_ptr()


# The operators of the attention block are called once a layer and token: their wrappers test
# plain conditions and build messages only to raise them.
_block = None


def _block_state():
    """(torch, {dtype: CEB_ACT_*}, library), looked up once."""
    global _block
    if _block is None:
        import torch
        _block = (torch, {torch.float32: ACT_F32, torch.bfloat16: ACT_BF16, torch.float16: ACT_F16}, load_library())
    return _block


def _same_device(what: str, x, tensors):
    """The device index of `x`, on which every other tensor (None allowed) must lie too."""
    dev = x.get_device()
    if dev < 0:
        raise CrispEmbedError(f"{what}: CUDA tensors expected")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise CrispEmbedError(f"{what}: a tensor on {t.device}, not on {x.device}")
    return dev


def _vector(t, dtype, n: int, what: str):
    """`t` (None allowed) is a contiguous vector of n values of `dtype`."""
    if t is not None and (t.dtype != dtype or t.numel() != n or not t.is_contiguous()):
        raise CrispEmbedError(f"{what}: {n} contiguous values of {dtype} expected")


def _c_int(what: str, value: int) -> int:
    """`value`, which a C int must hold: ctypes passes the lower 32 bits of any number."""
    if not -(1 << 31) <= value < 1 << 31:
        raise CrispEmbedError(f"{what}: {value} is not a 32-bit number")
    return value


def _raw_stream(torch, dev: int) -> int:
    """The current stream of device `dev` as a pointer (the quick form where torch has it)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(dev) if raw is not None else torch.cuda.current_stream(dev).cuda_stream


def _call_on(torch, dev: int, stream, fn, *args) -> int:
    """fn(*args, stream pointer) with device `dev` current, on its current stream unless one is given."""
    st = _raw_stream(torch, dev) if stream is None else int(stream)
    if torch.cuda.current_device() == dev:
        return fn(*args, st)
    with torch.cuda.device(dev):
        return fn(*args, st)


class CrispEmbed:
    """Text/ids -> L2-normalised embeddings through libcrispembed.so."""

    def __init__(self, model_path: str, n_threads: int = 4, lib_path: Optional[str] = None,
                 reference_arithmetic: bool = False):
        """reference_arithmetic: encode in the reference's CPU arithmetic bit for bit
        (ceb_init_ex with CEB_INIT_REFERENCE_ARITHMETIC; CUDA cores, slow)."""
        self._lib = load_library(lib_path)
        if reference_arithmetic:
            self._ctx = self._lib.ceb_init_ex(model_path.encode(), n_threads, 1)
        else:
            self._ctx = self._lib.crispembed_init(model_path.encode(), n_threads)
        if not self._ctx:
            raise CrispEmbedError(f"Failed to load model: {model_path}: {last_error()}")

    def close(self):
        if getattr(self, "_ctx", None):
            self._lib.crispembed_free(self._ctx)
            self._ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def hparams(self) -> _Hparams:
        return self._lib.crispembed_get_hparams(self._ctx).contents

    @property
    def n_moe_blocks(self) -> int:
        return int(self._lib.ceb_moe_block_count(self._ctx))

    @property
    def dim(self) -> int:
        h = self.hparams
        return h.n_output if h.n_output > 0 else h.n_embd

    def set_prefix(self, prefix: Optional[str]):
        self._lib.crispembed_set_prefix(self._ctx, (prefix or "").encode())

    def set_dim(self, dim: int):
        self._lib.crispembed_set_dim(self._ctx, int(dim))

    def encode(self, texts: Union[str, List[str]], matryoshka_dim: Optional[int] = None) -> np.ndarray:
        if matryoshka_dim is not None:
            self.set_dim(matryoshka_dim)
        single = isinstance(texts, str)
        if single:
            texts = [texts]
        try:
            dim = ctypes.c_int(0)
            if len(texts) == 1:
                ptr = self._lib.crispembed_encode(self._ctx, texts[0].encode(), ctypes.byref(dim))
            else:
                arr = (ctypes.c_char_p * len(texts))(*(t.encode() for t in texts))
                ptr = self._lib.crispembed_encode_batch(self._ctx, arr, len(texts), ctypes.byref(dim))
            if not ptr:
                raise CrispEmbedError(f"encoding failed: {last_error()}")
            out = np.ctypeslib.as_array(ptr, shape=(len(texts) * dim.value,)).copy().reshape(len(texts), dim.value)
            return out[0] if single else out
        finally:
            if matryoshka_dim is not None:
                self.set_dim(0)

    def encode_tokens(self, text: str, raw: bool = False):
        """Per-token final hidden states [n_tokens, n_embd] (L2-normalised unless raw) and their ids."""
        n = ctypes.c_int(0)
        dim = ctypes.c_int(0)
        fn = self._lib.crispembed_encode_tokens_raw if raw else self._lib.crispembed_encode_tokens
        ptr = fn(self._ctx, text.encode("utf-8"), ctypes.byref(n), ctypes.byref(dim))
        if not ptr:
            raise CrispEmbedError(f"encode_tokens failed: {last_error()}")
        vec = np.ctypeslib.as_array(ctypes.cast(ptr, ctypes.POINTER(ctypes.c_float)),
                                    shape=(n.value * dim.value,)).copy().reshape(n.value, dim.value)
        ids_ptr = ctypes.cast(self._lib.crispembed_last_token_ids(self._ctx), ctypes.POINTER(ctypes.c_int32))
        ids = np.ctypeslib.as_array(ids_ptr, shape=(n.value,)).copy()
        return vec, ids

    def token_str(self, token_id: int) -> str:
        r = self._lib.crispembed_token_str(self._ctx, int(token_id))
        return r.decode("utf-8", "replace") if r is not None else ""

    @property
    def tokenizer_kind(self) -> int:
        return self._lib.crispembed_tokenizer_kind(self._ctx)

    def attach_ep(self, ep: "ExpertParallel"):
        """Route every MoE block through `ep` (this context keeps only ep's experts)."""
        _check(self._lib.ceb_ep_attach(self._ctx, ep._h), "ceb_ep_attach")
        self._ep = ep  # the exchange must outlive the context's use of it

    def encode_ids(self, ids: np.ndarray, lens: Sequence[int]) -> np.ndarray:
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        lens = np.ascontiguousarray(lens, dtype=np.int32)
        dim = ctypes.c_int(0)
        i32p = ctypes.POINTER(ctypes.c_int32)
        ptr = self._lib.crispembed_encode_ids_batch(self._ctx, ids.ctypes.data_as(i32p), lens.ctypes.data_as(i32p),
                                                    len(lens), ctypes.byref(dim))
        if not ptr:
            raise CrispEmbedError(f"encode_ids failed: {last_error()}")
        return np.ctypeslib.as_array(ptr, shape=(len(lens) * dim.value,)).copy().reshape(len(lens), dim.value)

    def encode_ids_routes(self, ids: np.ndarray, lens: Sequence[int]):
        """(embeddings [n_seqs, dim], expert ids [n_moe, M, top_k], router logits
        [n_moe, M, n_experts]) of one synchronous encode (ceb_encode_ids_routes)."""
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        lens = np.ascontiguousarray(lens, dtype=np.int32)
        hp = self.hparams
        M, E, K = int(lens.sum()), int(hp.n_experts), int(hp.n_experts_per_tok)
        n_moe = self.n_moe_blocks
        emb = np.empty((len(lens), self.dim), dtype=np.float32)
        rid = np.empty((n_moe, M, max(K, 1)), dtype=np.int32)
        lg = np.empty((n_moe, M, max(E, 1)), dtype=np.float32)
        i32p = ctypes.POINTER(ctypes.c_int32)
        rc = self._lib.ceb_encode_ids_routes(self._ctx, ids.ctypes.data_as(i32p), lens.ctypes.data_as(i32p), len(lens),
                                             emb.ctypes.data, rid.ctypes.data, lg.ctypes.data)
        _check(rc, "encode_ids_routes")
        return emb, rid, lg

    def encode_ids_device(self, d_ids, lens: np.ndarray, d_out, stream=None) -> int:
        """d_ids: int32 CUDA tensor, d_out: float32 CUDA tensor [n_seqs, dim]."""
        lens = np.ascontiguousarray(lens, dtype=np.int32)
        dim = ctypes.c_int(0)
        rc = self._lib.crispembed_encode_ids_device(self._ctx, d_ids.data_ptr(),
                                                    lens.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), len(lens),
                                                    d_out.data_ptr(), ctypes.byref(dim), _stream_ptr(stream))
        _check(rc, "encode_ids_device")
        return dim.value


class MoELayer:
    """One MoE feed-forward block on the device (ceb_moe_layer_create / ceb_moe_ffn)."""

    def __init__(self, d: int, n_experts: int, top_k: int, ffn: int, router_type: int, router_raw: np.ndarray,
                 expert_type: int, fc1_raw: np.ndarray, fc2_raw: np.ndarray, bias: Optional[np.ndarray] = None):
        self._lib = load_library()
        self.d, self.n_experts, self.top_k, self.ffn = d, n_experts, top_k, ffn
        keep = [np.ascontiguousarray(router_raw), np.ascontiguousarray(fc1_raw), np.ascontiguousarray(fc2_raw)]
        b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        self._h = self._lib.ceb_moe_layer_create(d, n_experts, top_k, ffn, router_type, keep[0].ctypes.data,
                                                 expert_type, keep[1].ctypes.data, keep[2].ctypes.data,
                                                 None if b is None else b.ctypes.data)
        if not self._h:
            raise CrispEmbedError(f"ceb_moe_layer_create failed: {last_error()}")

    def close(self):
        if getattr(self, "_h", None):
            self._lib.ceb_moe_layer_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def forward_static(self, x, y, stream=None):
        """ceb_moe_ffn_static: the library's own fixed scratch, no device allocation."""
        import torch
        act = {torch.float32: ACT_F32, torch.bfloat16: ACT_BF16, torch.float16: ACT_F16}[x.dtype]
        _check(self._lib.ceb_moe_ffn_static(self._h, x.data_ptr(), act, x.shape[0], y.data_ptr(), _stream_ptr(stream)),
               "ceb_moe_ffn_static")

    def routing(self, workspace, n_tokens: int):
        """(ids, weights, slot_pos, offsets) of the last call on `workspace` (a uint8
        CUDA tensor), as host numpy arrays (ceb_moe_workspace_routing)."""
        import torch
        ptrs = [ctypes.c_void_p() for _ in range(4)]
        _check(self._lib.ceb_moe_workspace_routing(self._h, n_tokens, workspace.data_ptr(),
                                                   *[ctypes.byref(p) for p in ptrs]), "ceb_moe_workspace_routing")
        K, E = self.top_k, self.n_experts
        out = []
        for p, n, dt in ((ptrs[0], n_tokens * K, torch.int32), (ptrs[1], n_tokens * K, torch.float32),
                         (ptrs[2], n_tokens * K, torch.int32), (ptrs[3], E + 1, torch.int32)):
            off = p.value - workspace.data_ptr()
            out.append(workspace[off:off + 4 * n].view(dt).cpu().numpy())
        ids, w, sp, offsets = out
        return ids.reshape(n_tokens, K), w.reshape(n_tokens, K), sp.reshape(n_tokens, K), offsets

    def workspace_size(self, n_tokens: int) -> int:
        return int(self._lib.ceb_moe_workspace_size(self._h, n_tokens))

    def forward(self, x, y, workspace, ids=None, weights=None, counts=None, logits=None, stream=None):
        import torch
        act = {torch.float32: ACT_F32, torch.bfloat16: ACT_BF16, torch.float16: ACT_F16}[x.dtype]
        rc = self._lib.ceb_moe_ffn(self._h, x.data_ptr(), act, x.shape[0], y.data_ptr(), _ptr(ids), _ptr(weights),
                                   _ptr(counts), _ptr(logits), workspace.data_ptr(), workspace.numel(),
                                   _stream_ptr(stream))
        _check(rc, "ceb_moe_ffn")

    def forward_ep(self, ep: "ExpertParallel", x, y, workspace, stream=None):
        """ceb_moe_ffn_ep: this rank's tokens through the expert-parallel exchange."""
        import torch
        act = {torch.float32: ACT_F32, torch.bfloat16: ACT_BF16, torch.float16: ACT_F16}[x.dtype]
        rc = self._lib.ceb_moe_ffn_ep(self._h, ep._h, x.data_ptr(), act, x.shape[0], y.data_ptr(),
                                      workspace.data_ptr(), workspace.numel(), _stream_ptr(stream))
        _check(rc, "ceb_moe_ffn_ep")

    def route_ln(self, res, y, out, workspace, gamma=None, beta=None, eps=1e-5, out16=None, ids=None, weights=None,
                 logits=None, stream=None):
        """ceb_moe_route_ln: out = LN(res + y), and the router on the normalised rows in the same pass."""
        rc = self._lib.ceb_moe_route_ln(self._h, res.data_ptr(), y.data_ptr(), res.shape[0], _ptr(gamma), _ptr(beta),
                                        float(eps), out.data_ptr(), _ptr(out16), _ptr(ids), _ptr(weights),
                                        _ptr(logits), workspace.data_ptr(), workspace.numel(), _stream_ptr(stream))
        _check(rc, "ceb_moe_route_ln")


EP_HANDLE_BYTES = 64


class ExpertParallel:
    """Expert-parallel exchange of one rank (ceb_ep_create / _ipc_handle / _connect).

    `connect(handles)` takes every rank's handle bytes in rank order; see
    crispembed_b200.dist.connect_expert_parallel for the torch.distributed form."""

    def __init__(self, rank: int, world: int, n_experts: int, top_k: int, d: int, ffn: int, max_local_tokens: int):
        self._lib = load_library()
        self.rank, self.world = rank, world
        self._h = self._lib.ceb_ep_create(rank, world, n_experts, top_k, d, ffn, max_local_tokens)
        if not self._h:
            raise CrispEmbedError(f"ceb_ep_create failed: {last_error()}")

    def handle(self) -> bytes:
        buf = ctypes.create_string_buffer(EP_HANDLE_BYTES)
        _check(self._lib.ceb_ep_ipc_handle(self._h, buf), "ceb_ep_ipc_handle")
        return buf.raw

    def connect(self, handles: Sequence[bytes]):
        if len(handles) != self.world or any(len(h) != EP_HANDLE_BYTES for h in handles):
            raise CrispEmbedError("connect: one handle of EP_HANDLE_BYTES per rank expected")
        blob = ctypes.create_string_buffer(b"".join(handles), EP_HANDLE_BYTES * self.world)
        _check(self._lib.ceb_ep_connect(self._h, blob), "ceb_ep_connect")

    def set_timeout_ms(self, ms: int):
        self._lib.ceb_ep_set_timeout_ms(self._h, int(ms))

    def close(self):
        if getattr(self, "_h", None):
            self._lib.ceb_ep_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


class Linear:
    """Device-resident linear layer (ceb_linear_create / ceb_linear_forward)."""

    def __init__(self, w_type: int, w_raw: np.ndarray, n_out: int, k: int):
        self._lib = load_library()
        self.n_out, self.k = n_out, k
        w_raw = np.ascontiguousarray(w_raw)
        self._h = self._lib.ceb_linear_create(w_type, w_raw.ctypes.data, n_out, k)
        if not self._h:
            raise CrispEmbedError(f"ceb_linear_create failed: {last_error()}")

    def __call__(self, x, out=None, bias=None, gelu=False, out_f16=False, stream=None):
        import torch
        if out is None:
            out = torch.empty((x.shape[0], self.n_out), dtype=torch.float16 if out_f16 else torch.float32,
                              device=x.device)
        _check(self._lib.ceb_linear_forward(self._h, x.data_ptr(), x.shape[0], _ptr(bias), int(gelu), int(out_f16),
                                            out.data_ptr(), _stream_ptr(stream)), "ceb_linear_forward")
        return out

    def fused(self, x, bias=None, act: str = "none", residual=None, out=None, out_dtype=None, stream=None):
        """act(x W^T + bias) + residual (ceb_linear_fused), rounded once to the output's type.

        x: [m, k] fp16; residual, out: [m, n_out] in fp32, fp16 or bf16; rows may be strided.
        act: "none", "relu", "silu", "gelu" or "gelu_tanh".  out (default: new, of out_dtype or
        fp16) may be the residual.  Runs on x's device and its current stream."""
        torch, types, lib = _block_state()
        m, n = x.shape[0], self.n_out
        if act not in ACTIVATIONS:
            raise CrispEmbedError(f"fused: activation {act!r}: one of {', '.join(ACTIVATIONS)}")
        if x.dim() != 2 or x.shape[1] != self.k or x.dtype != torch.float16 or x.stride(1) != 1:
            raise CrispEmbedError(f"fused: x must be fp16 [rows, {self.k}] with contiguous rows")
        dev = _same_device("fused", x, (bias, residual, out))
        _vector(bias, torch.float32, n, "fused: bias")
        if out is None:
            out = x.new_empty((m, n), dtype=out_dtype or torch.float16)
        elif out_dtype is not None and out.dtype != out_dtype:
            raise CrispEmbedError("fused: out is not of out_dtype")
        for t in (out,) if residual is None else (out, residual):
            if t.dtype not in types or t.shape != (m, n) or t.stride(1) != 1:
                raise CrispEmbedError(f"fused: residual and out must be [{m}, {n}] in fp32, fp16 or bf16 with contiguous rows")
        res = (None, 0, 0) if residual is None else (residual.data_ptr(), types[residual.dtype], residual.stride(0))
        rc = _call_on(torch, dev, stream, lib.ceb_linear_fused, self._h, x.data_ptr(), x.stride(0), m,
                      None if bias is None else bias.data_ptr(), ACTIVATIONS[act], *res, types[out.dtype],
                      out.data_ptr(), out.stride(0))
        if rc:
            _check(rc, "ceb_linear_fused")
        return out

    def close(self):
        if getattr(self, "_h", None):
            self._lib.ceb_linear_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def matmul(w_type: int, w_raw: np.ndarray, n_out: int, k: int, x, bias=None, gelu=False, out_f16=False, stream=None):
    import torch
    lib = load_library()
    out = torch.empty((x.shape[0], n_out), dtype=torch.float16 if out_f16 else torch.float32, device=x.device)
    w_raw = np.ascontiguousarray(w_raw)
    rc = lib.ceb_matmul(w_type, w_raw.ctypes.data, n_out, k, x.data_ptr(), x.shape[0], _ptr(bias), int(gelu),
                        int(out_f16), out.data_ptr(), _stream_ptr(stream))
    _check(rc, "ceb_matmul")
    return out


def pool_l2(hidden, cu_seqlens, out_dim: Optional[int] = None, stream=None):
    import torch
    lib = load_library()
    n = cu_seqlens.numel() - 1
    d = hidden.shape[1]
    od = out_dim or d
    out = torch.empty((n, od), dtype=torch.float32, device=hidden.device)
    _check(lib.ceb_pool_l2(hidden.data_ptr(), cu_seqlens.data_ptr(), n, d, od, out.data_ptr(), _stream_ptr(stream)),
           "ceb_pool_l2")
    return out


def attention(qkv, cu_seqlens, n_head: int, max_len: Optional[int] = None, stream=None):
    """softmax(Q K^T / sqrt(64)) V per sequence and head; qkv [rows, 3d] fp16 on the device."""
    import torch
    lib = load_library()
    rows, d3 = qkv.shape
    d = d3 // 3
    n = cu_seqlens.numel() - 1
    if max_len is None:
        max_len = int((cu_seqlens[1:] - cu_seqlens[:-1]).max().item()) if n else 0
    out = torch.empty((rows, d), dtype=torch.float16, device=qkv.device)
    _check(lib.ceb_attention_forward(qkv.data_ptr(), rows, cu_seqlens.data_ptr(), n, max_len, d, n_head,
                                     out.data_ptr(), _stream_ptr(stream)), "ceb_attention_forward")
    return out


def attention_masked(q, k, v, cu_q, cu_k=None, max_q: Optional[int] = None, max_k: Optional[int] = None, *,
                     scale: Optional[float] = None, softcap: float = 0.0, window=(-1, -1), prefix=None, doc_q=None,
                     doc_k=None, slopes=None, rel_bias=None, out=None, stream=None):
    """Packed attention with shared key heads, a capped score, a bias by distance and masks
    (ceb_attention_masked, whose header has the formulas).

    q: [q_rows, n_head, head_dim], k / v: [k_rows, n_head_kv, head_dim], fp16 or bf16, any row and
    head strides that are multiples of 8 values; cu_q / cu_k (default: cu_q) int32 row offsets;
    max_q / max_k: the longest sequence (default: read from the offsets, which waits for the
    device).  scale: default 1/sqrt(head_dim).  window: (left, right) keys around a row's place,
    -1 open; (-1, 0) is causal.  prefix: int32 [n_seqs] keys that every row sees.  doc_q / doc_k:
    int32 document numbers (doc_k default: doc_q).  slopes: fp32 [n_head], or rel_bias: fp32
    [n_head, 2 R + 1].  Returns out, [q_rows, n_head, head_dim]; rows of no sequence are not
    written.  Runs on q's device and its current stream."""
    torch, types, lib = _block_state()
    dtype = q.dtype
    if dtype not in types or dtype == torch.float32 or k.dtype != dtype or v.dtype != dtype:
        raise CrispEmbedError("attention_masked: q, k, v in fp16 or bf16, all alike, expected")
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[2] != q.shape[2]:
        raise CrispEmbedError("attention_masked: q [rows, heads, head_dim], k and v [keys, key heads, head_dim] expected")
    (qr, qh, q1), (kr, kh, k1), (vr, vh, v1) = q.stride(), k.stride(), v.stride()
    if q1 != 1 or k1 != 1 or v1 != 1:
        raise CrispEmbedError("attention_masked: the values of a head must be contiguous")
    if cu_k is None:
        cu_k = cu_q
    if doc_k is None:
        doc_k = doc_q
    dev = _same_device("attention_masked", q, (k, v, cu_q, cu_k, prefix, doc_q, doc_k, slopes, rel_bias, out))
    rows, n_head, hd = q.shape
    keys, n = k.shape[0], cu_q.numel() - 1
    if n < 0:
        raise CrispEmbedError("attention_masked: row offsets expected")
    i32, f32 = torch.int32, torch.float32
    _vector(cu_q, i32, n + 1, "attention_masked: cu_q")
    _vector(cu_k, i32, n + 1, "attention_masked: cu_k")
    _vector(prefix, i32, n, "attention_masked: prefix")
    _vector(doc_q, i32, rows, "attention_masked: doc_q")
    _vector(doc_k, i32, keys, "attention_masked: doc_k")
    _vector(slopes, f32, n_head, "attention_masked: slopes")
    radius = 0
    if rel_bias is not None:
        if rel_bias.dim() != 2 or rel_bias.shape[1] % 2 != 1:
            raise CrispEmbedError("attention_masked: rel_bias [heads, 2 R + 1] expected")
        radius = rel_bias.shape[1] // 2
        _vector(rel_bias, f32, n_head * (2 * radius + 1), "attention_masked: rel_bias")
    if max_q is None:
        max_q = int((cu_q[1:] - cu_q[:-1]).max().item()) if n else 0
    if max_k is None:
        max_k = int((cu_k[1:] - cu_k[:-1]).max().item()) if n else 0
    if out is None:
        out = q.new_empty((rows, n_head, hd))
    elif out.shape != q.shape or out.dtype != dtype:
        raise CrispEmbedError("attention_masked: out must have q's shape and type")
    rr, rh, r1 = out.stride()
    if r1 != 1:
        raise CrispEmbedError("attention_masked: the values of a head must be contiguous")
    try:
        p = _ATTN_PARAMS.pack(types[dtype], n_head, k.shape[1], hd, n, rows, keys, max_q, max_k, qr, qh, kr, kh, vr, vh, rr, rh,
                              cu_q.data_ptr(), cu_k.data_ptr(), hd ** -0.5 if scale is None else scale, softcap, window[0],
                              window[1], 0 if prefix is None else prefix.data_ptr(), 0 if doc_q is None else doc_q.data_ptr(),
                              0 if doc_k is None else doc_k.data_ptr(), 0 if slopes is None else slopes.data_ptr(),
                              0 if rel_bias is None else rel_bias.data_ptr(), radius)
    except (struct.error, OverflowError) as e:
        raise CrispEmbedError(f"attention_masked: an argument does not fit its 32 bits ({e})") from None
    rc = _call_on(torch, dev, stream, lib.ceb_attention_masked, p, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  out.data_ptr())
    if rc:
        _check(rc, "ceb_attention_masked")
    return out


ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}


class Rope:
    """Rotary positions: a plan of frequencies (ceb_rope_create) and the rotation (ceb_rope_forward)."""

    def __init__(self, rot_dim: int, theta: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                 context: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0):
        """The plan lies on the current device.  scaling: "none", "linear", "ntk" or "yarn"."""
        if scaling not in ROPE_SCALINGS:
            raise CrispEmbedError(f"Rope: scaling {scaling!r}: one of {', '.join(ROPE_SCALINGS)}")
        self._h = None
        self._lib = load_library()
        self.rot_dim = rot_dim
        self._h = self._lib.ceb_rope_create(_c_int("Rope: rot_dim", rot_dim), theta, ROPE_SCALINGS[scaling], factor,
                                            _c_int("Rope: context", context), beta_fast, beta_slow)
        if not self._h:
            raise CrispEmbedError(f"ceb_rope_create failed: {last_error()}")

    def __call__(self, x, out=None, positions=None, cu_seqlens=None, pos_offset: int = 0, interleaved: bool = False,
                 stream=None):
        """x: [rows, heads, head_dim] in fp32, fp16 or bf16, rows and heads strided at will.  Positions:
        int32 [rows], or the rows' places in the sequences of cu_seqlens (int32) plus pos_offset.
        out (default: new) may be x.  Runs on x's device and its current stream."""
        torch, types, lib = _block_state()
        dtype = x.dtype
        if x.dim() != 3 or dtype not in types:
            raise CrispEmbedError("Rope: x must be [rows, heads, head_dim] in fp32, fp16 or bf16")
        _c_int("Rope: pos_offset", pos_offset)
        rows, heads, hd = x.shape
        _c_int("Rope: rows", rows)
        dev = _same_device("Rope", x, (out, positions, cu_seqlens))
        if positions is None and cu_seqlens is None:
            raise CrispEmbedError("Rope: positions or cu_seqlens must be given")
        n = 0
        _vector(positions, torch.int32, rows, "Rope: positions")
        if cu_seqlens is not None:
            n = cu_seqlens.numel() - 1
            _vector(cu_seqlens, torch.int32, n + 1, "Rope: cu_seqlens")
        if out is None:
            out = x.new_empty((rows, heads, hd))
        elif out.shape != x.shape or out.dtype != dtype:
            raise CrispEmbedError("Rope: out must have x's shape and type")
        (xr, xh, x1), (rr, rh, r1) = x.stride(), out.stride()
        if (x1 != 1 or r1 != 1) and hd > 1:
            raise CrispEmbedError("Rope: the values of a head must be contiguous")
        rc = _call_on(torch, dev, stream, lib.ceb_rope_forward, self._h, x.data_ptr(), out.data_ptr(), types[dtype], rows,
                      heads, hd, xr, xh, rr, rh, interleaved, None if positions is None else positions.data_ptr(),
                      None if cu_seqlens is None else cu_seqlens.data_ptr(), n, pos_offset)
        if rc:
            _check(rc, "ceb_rope_forward")
        return out

    def close(self):
        if getattr(self, "_h", None):
            self._lib.ceb_rope_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def gguf_dequantize(ggml_type: int, raw: np.ndarray, n_rows: int, k: int) -> np.ndarray:
    """ceb_gguf_dequantize: host decoding of n_rows GGUF rows of k values to fp32."""
    raw = np.ascontiguousarray(raw)
    out = np.empty((n_rows, k), dtype=np.float32)
    _check(load_library().ceb_gguf_dequantize(int(ggml_type), raw.ctypes.data, int(n_rows), int(k),
                                              out.ctypes.data), "ceb_gguf_dequantize")
    return out


class Tokenizer:
    """The text tokenizer of a GGUF (WordPiece or SentencePiece Unigram), without a device."""

    def __init__(self, gguf_path: str, max_tokens: int = 512):
        self._lib = load_library()
        self._h = self._lib.ceb_tokenizer_load(gguf_path.encode(), int(max_tokens))
        if not self._h:
            raise CrispEmbedError(f"ceb_tokenizer_load failed: {last_error()}")
        self.max_tokens = int(max_tokens)

    @property
    def kind(self) -> int:
        return self._lib.ceb_tokenizer_kind_of(self._h)

    def encode(self, text: str):
        cap = self.max_tokens
        buf = (ctypes.c_int32 * cap)()
        n = self._lib.ceb_tokenizer_encode(self._h, text.encode("utf-8"), buf, cap)
        if n < 0:
            raise CrispEmbedError(f"ceb_tokenizer_encode failed: {last_error()}")
        return [int(buf[i]) for i in range(min(n, cap))]

    def close(self):
        if self._h:
            self._lib.ceb_tokenizer_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def sync_check(stream=None):
    _check(load_library().ceb_sync_check(_stream_ptr(stream)), "device check")


PROFILE_CATEGORIES = ("gemm", "attention", "routing", "rowwise", "exchange", "exchange_wait", "moe_gemm")


def launch_count() -> int:
    return int(load_library().ceb_launch_count())


def profile_enable(on: bool = True):
    load_library().ceb_profile_enable(int(on))


def profile_read() -> dict:
    n = len(PROFILE_CATEGORIES)
    L = (ctypes.c_longlong * n)()
    ms, fl, by = (ctypes.c_double * n)(), (ctypes.c_double * n)(), (ctypes.c_double * n)()
    _check(load_library().ceb_profile_read(L, ms, fl, by, n), "ceb_profile_read")
    return {c: dict(launches=int(L[i]), ms=float(ms[i]), flops=float(fl[i]), bytes=float(by[i]))
            for i, c in enumerate(PROFILE_CATEGORIES)}
