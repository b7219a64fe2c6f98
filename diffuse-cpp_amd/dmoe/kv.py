"""The paged KV cache of include/dmoe.h (dmoe_kv_cache, dmoe_kv_batch) over
torch tensors on the context's GPU, which the caller keeps alive.

    cache = dmoe.KvCache.empty("e4m3", n_pages, n_head_kv=4, head_dim=128, page_tokens=64)
    batch = dmoe.KvBatch(q_start, kv_len, pages, n_tokens)       # int32 tensors
    ctx.kv_append_device(cache, batch, ap, qkv, q, q_norm, k_norm, stream=s)
    ctx.kv_attn_device(cache, batch, ap, q, out, stream=s)

The cache's and the batch's tensors are checked here, once; a call's own buffers
are contiguous float32 tensors of the size that the header states, as in the
other device calls.
"""
from __future__ import annotations

import ctypes as C

from ._abi import AttnHParams, KvBatchStruct, KvCacheStruct

KV_F16, KV_E4M3 = 0, 1
KV_TYPES = {"f16": KV_F16, "e4m3": KV_E4M3}
KV_BLOCK = 32


def attn_hparams(n_head: int, n_head_kv: int, head_dim: int, rotary_dim: int = 0, block_length: int = 0,
                 rope_base: float = 1e6, rms_eps: float = 1e-6, use_qk_norm: bool = False,
                 n_embd: int = 0) -> AttnHParams:
    """dmoe_attn_hparams of a call without a layer."""
    return AttnHParams(n_embd, n_head, n_head_kv, head_dim, rotary_dim, int(use_qk_norm), block_length, rope_base,
                       rms_eps)


def _whole(t, dtype, name):
    if str(t.dtype) != dtype or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous {dtype} tensor is needed, not {t.dtype} with strides {t.stride()}")
    return t


def _one_gpu(*tensors):
    devices = {str(t.device) for t in tensors if t is not None}
    if len(devices) != 1 or not tensors[0].is_cuda:
        raise ValueError(f"the tensors are on {sorted(devices)}, not on one GPU")


class KvCache:
    """k [n_pages, n_head_kv, page_tokens, head_dim]; v [n_pages, n_head_kv,
    page_tokens / 32, head_dim, 32] (float16) or [.., head_dim / 2, 4, 2, 8]
    (float8_e4m3fn, with int8 k_exp, v_exp [n_pages, n_head_kv, page_tokens / 32])."""

    def __init__(self, k, v, k_exp=None, v_exp=None):
        if k.dim() != 4:
            raise ValueError(f"k: 4 dimensions are needed, not {tuple(k.shape)}")
        f8 = "float8_e4m3fn" in str(k.dtype)
        P, H, T, D = k.shape
        dtype = "torch.float8_e4m3fn" if f8 else "torch.float16"
        blocks = (P, H, T // KV_BLOCK)
        if T % KV_BLOCK:
            raise ValueError(f"k: {T} tokens a page are not a multiple of {KV_BLOCK}")
        want = blocks + ((D // 2, 4, 2, 8) if f8 else (D, KV_BLOCK))
        if tuple(v.shape) != want:
            raise ValueError(f"v: {tuple(v.shape)}, {want} is needed")
        _whole(k, dtype, "k")
        _whole(v, dtype, "v")
        if f8:
            for name, e in (("k_exp", k_exp), ("v_exp", v_exp)):
                if e is None or tuple(e.shape) != blocks:
                    raise ValueError(f"{name}: shape {blocks} is needed")
                _whole(e, "torch.int8", name)
        _one_gpu(k, v, *([k_exp, v_exp] if f8 else []))
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.struct = KvCacheStruct(KV_E4M3 if f8 else KV_F16, H, D, T, P, k.data_ptr(), v.data_ptr(),
                                    k_exp.data_ptr() if f8 else None, v_exp.data_ptr() if f8 else None)
        self.ref = C.byref(self.struct)

    @classmethod
    def empty(cls, kvtype: str, n_pages: int, n_head_kv: int, head_dim: int, page_tokens: int = 64, device="cuda:0"):
        import torch
        f8 = KV_TYPES[kvtype] == KV_E4M3
        dt = torch.float8_e4m3fn if f8 else torch.float16
        nb = page_tokens // KV_BLOCK
        make = lambda shape, dtype: torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
        k = make((n_pages, n_head_kv, page_tokens, head_dim), dt)
        v = make((n_pages, n_head_kv, nb) + ((head_dim // 2, 4, 2, 8) if f8 else (head_dim, KV_BLOCK)), dt)
        exps = [make((n_pages, n_head_kv, nb), torch.int8) if f8 else None for _ in range(2)]
        return cls(k, v, *exps)


class KvBatch:
    """The sequences of one call: int32 tensors q_start [n_seqs + 1], kv_len
    [n_seqs], pages [n_seqs, max_pages]; n_tokens rows in the call's buffers."""

    def __init__(self, q_start, kv_len, pages, n_tokens: int):
        n = kv_len.numel()
        if tuple(q_start.shape) != (n + 1,) or kv_len.dim() != 1 or pages.dim() != 2 or pages.shape[0] != n:
            raise ValueError(f"q_start {tuple(q_start.shape)}, kv_len {tuple(kv_len.shape)}, pages {tuple(pages.shape)}")
        for name, t in (("q_start", q_start), ("kv_len", kv_len), ("pages", pages)):
            _whole(t, "torch.int32", name)
        _one_gpu(q_start, kv_len, pages)
        self.q_start, self.kv_len, self.pages, self.n_tokens = q_start, kv_len, pages, int(n_tokens)
        self.struct = KvBatchStruct(n, self.n_tokens, pages.shape[1], q_start.data_ptr(), kv_len.data_ptr(),
                                    pages.data_ptr())
        self.ref = C.byref(self.struct)
