"""Per-head norms of queries and keys, the position rotation and the cache write.

``qk_norm_rope`` does in one pass over a step's q, k and v what stands between
the projections and the attention in a model with normed heads: the norm of
every query and key head, the rotation of its first columns by the token's
position, and (given a cache) the write that ``kv_cache.reshape_and_cache`` would
do, into either 16-bit layout or the 4-bit cache.  The reference leaves the first
two to the model and does the third in ``do_kv_cache_update``
(hcp_vllm_plugin/ring_backend.py:501-539).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .kv_cache import _cache_desc, _check_slots, fp4_desc
from .varlen import PagedCache

__all__ = ["qk_norm_rope"]

_INDEX = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}


def _rows(name: str, t: torch.Tensor, like: torch.Tensor, heads: int | None = None) -> None:
    """``t`` [T, heads, D] with the kernel's rows, of like's tokens, width, type and device."""
    if t.dim() != 3 or t.shape[0] != like.shape[0] or t.shape[2] != like.shape[2] or \
            (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name}: shape {tuple(t.shape)} does not fit query and key")
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be of query's dtype and device")
    if t.stride(2) != 1 or t.data_ptr() % 16 or t.stride(0) % 8 or t.stride(1) % 8:
        raise ValueError(f"{name}: 16-byte aligned rows with contiguous head_dim")


def qk_norm_rope(
    query: torch.Tensor,
    key: torch.Tensor,
    positions: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    *,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    value: torch.Tensor | None = None,
    kv_cache: torch.Tensor | None = None,
    slot_mapping: torch.Tensor | None = None,
    query_out: torch.Tensor | None = None,
    key_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Normed and rotated query and key ``[T, heads, D]`` (fp16 / bf16).

    With a weight ``[D]``, each head's row is ``x / sqrt(mean(x^2) + eps) *
    weight``; without, it is not normed.  The first ``rot`` columns are rotated
    by row ``positions[t]`` of ``cos_sin_cache`` ``[max_positions, rot]`` (``rot /
    2`` cosines, then as many sines; float32 or query's dtype): columns i and i +
    rot / 2 as a pair, with ``interleaved`` 2 i and 2 i + 1.  A position outside
    the table takes its first or last row.  Everything is computed in 32 bits and
    then rounded (a key for the 4-bit cache in 64 up to that, and rounded to
    query's dtype before it is coded, so that the cache holds what
    ``reshape_and_cache`` of that key would).

    With ``value``, ``kv_cache`` and ``slot_mapping``, key and value of token t go
    into the cache at ``slot_mapping[t]`` (tokens past its length and negative
    slots are not written); the key then comes back only where ``key_out`` asks
    for it.  ``query_out`` / ``key_out`` may be query and key themselves."""
    if query.dtype not in (torch.float16, torch.bfloat16) or not query.is_cuda:
        raise ValueError("query must be float16/bfloat16 on the GPU")
    _rows("query", query, query)
    _rows("key", key, query)
    t, h, d = query.shape
    hkv, dev = key.shape[1], query.device
    if positions.dtype not in _INDEX or tuple(positions.shape) != (t,) or \
            not positions.is_contiguous() or positions.device != dev:
        raise ValueError("positions must be contiguous int32/int64 [T] on query's device")
    tab = cos_sin_cache
    if tab.dim() != 2 or tab.stride(1) != 1 or tab.device != dev or \
            tab.dtype not in (torch.float32, query.dtype):
        raise ValueError("cos_sin_cache must be [max_positions, rot], float32 or query's dtype, on "
                         "query's device")
    if tab.shape[1] % 16 or tab.shape[1] > d or (tab.shape[1] and tab.shape[0] == 0):
        raise ValueError("rot must be a multiple of 16 up to head_dim, and the table not empty")
    if tab.shape[1] and (tab.data_ptr() % 16 or tab.stride(0) % 8):
        raise ValueError("cos_sin_cache: 16-byte aligned rows")
    wide = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if tuple(w.shape) != (d,) or w.stride(0) != 1 or w.device != dev or w.data_ptr() % 16 or \
                w.dtype not in (torch.float32, query.dtype) or w.dtype != (wide or w.dtype):
            raise ValueError("weights must be [head_dim] and of one dtype, float32 or query's, on "
                             "query's device")
        wide = w.dtype
    a = _lib.QkRopeArgs()
    a.slot_dtype, hold = _lib.DTYPE_I64, None
    if kv_cache is None:
        if value is not None or slot_mapping is not None:
            raise ValueError("value and slot_mapping go with a kv_cache")
        if key_out is None:
            key_out = torch.empty_like(key, memory_format=torch.contiguous_format)
    else:
        if value is None or slot_mapping is None:
            raise ValueError("a cache write needs value and slot_mapping")
        _rows("value", value, query, hkv)
        _check_slots(slot_mapping, kv_cache)
        if kv_cache.device != dev:
            raise ValueError("kv_cache must be on query's device")
        if slot_mapping.shape[0] > t:
            raise ValueError(f"{slot_mapping.shape[0]} slots for {t} tokens")
        slots = slot_mapping.contiguous()
        a.slot_mapping, a.num_slots, a.slot_dtype = slots.data_ptr(), slots.shape[0], \
            _INDEX[slots.dtype]
        a.v, a.v_stride_tok, a.v_stride_head = value.data_ptr(), value.stride(0), value.stride(1)
        if kv_cache.dtype == torch.uint8:
            pc = PagedCache.from_tensor(kv_cache)
            c_hkv, c_d, desc = pc.num_kv_heads, pc.head_dim, fp4_desc(pc)
            a.cache_kind, a.fp4 = 2, ctypes.addressof(desc)
        else:
            if kv_cache.dtype != query.dtype:
                raise ValueError("kv_cache must be of query's dtype, or a 4-bit cache (uint8)")
            desc, addr, c_hkv, c_d = _cache_desc(kv_cache)
            a.cache_kind, a.cache = 1, addr
        if c_hkv != hkv or c_d != d:
            raise ValueError("key heads or head_dim do not match the cache")
        hold = (slots, desc)
    if query_out is None:
        query_out = torch.empty_like(query, memory_format=torch.contiguous_format)
    else:
        _rows("query_out", query_out, query, h)
    if key_out is not None:
        _rows("key_out", key_out, query, hkv)
        a.k_out, a.ko_stride_tok, a.ko_stride_head = key_out.data_ptr(), key_out.stride(0), \
            key_out.stride(1)
    a.q, a.q_stride_tok, a.q_stride_head = query.data_ptr(), query.stride(0), query.stride(1)
    a.k, a.k_stride_tok, a.k_stride_head = key.data_ptr(), key.stride(0), key.stride(1)
    a.q_out, a.qo_stride_tok, a.qo_stride_head = query_out.data_ptr(), query_out.stride(0), \
        query_out.stride(1)
    if q_weight is not None:
        a.q_weight = q_weight.data_ptr()
    if k_weight is not None:
        a.k_weight = k_weight.data_ptr()
    a.positions, a.pos_dtype = positions.data_ptr(), _INDEX[positions.dtype]
    if tab.shape[1]:
        a.cos_sin, a.table_stride, a.max_positions = tab.data_ptr(), tab.stride(0), tab.shape[0]
    a.num_tokens, a.eps = t, eps
    a.num_heads, a.num_kv_heads, a.head_dim, a.rot = h, hkv, d, tab.shape[1]
    a.dtype, a.table_dtype = _lib.dtype_code(query.dtype), _lib.dtype_code(tab.dtype)
    a.weight_dtype = _lib.dtype_code(wide or query.dtype)
    a.interleaved = bool(interleaved)
    with _lib.on_device(dev):
        rc = _lib.lib().hcp_qk_norm_rope(ctypes.addressof(a), _lib.stream_ptr(dev))
    _lib.check(rc, "hcp_qk_norm_rope")
    return query_out, key_out
