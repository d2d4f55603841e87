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
from .kv_cache import _cache_desc, check_slots
from .varlen import fp4_desc

__all__ = ["qk_norm_rope"]

_INDEX = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}


def _rows(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype,
          device: torch.device) -> tuple[int, int]:
    """Token and head stride of ``t``, which must have the kernel's rows."""
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, not {shape}")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be of query's dtype and device")
    tok, head, col = t.stride()
    if col != 1 or (t.data_ptr() | 2 * tok | 2 * head) & 15:
        raise ValueError(f"{name}: 16-byte aligned rows with contiguous head_dim")
    return tok, head


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
    dt, dev = query.dtype, query.device
    if dt not in (torch.float16, torch.bfloat16) or dev.type != "cuda" or query.dim() != 3 or \
            key.dim() != 3:
        raise ValueError("query and key must be float16/bfloat16 [T, heads, D] on the GPU")
    t, h, d = query.shape
    hkv = key.shape[1]
    a = _lib.QkRopeArgs()
    a.q_stride_tok, a.q_stride_head = _rows("query", query, (t, h, d), dt, dev)
    a.k_stride_tok, a.k_stride_head = _rows("key", key, (t, hkv, d), dt, dev)
    if positions.dtype not in _INDEX or positions.shape != (t,) or positions.device != dev or \
            not positions.is_contiguous():
        raise ValueError("positions must be contiguous int32/int64 [T] on query's device")
    tab = cos_sin_cache
    if tab.dim() != 2 or tab.device != dev or tab.dtype not in (torch.float32, dt):
        raise ValueError("cos_sin_cache must be [max_positions, rot], float32 or query's dtype, on "
                         "query's device")
    most, rot = tab.shape
    if rot:
        row, col = tab.stride()
        if rot % 16 or rot > d or most == 0:
            raise ValueError("rot must be a multiple of 16 up to head_dim, and the table not empty")
        if col != 1 or tab.data_ptr() % 16 or row % 8:
            raise ValueError("cos_sin_cache: 16-byte aligned rows")
        a.cos_sin, a.table_stride, a.max_positions = tab.data_ptr(), row, most
    wide = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if w.shape != (d,) or w.stride(0) != 1 or w.device != dev or w.data_ptr() % 16 or \
                w.dtype not in (torch.float32, dt) or w.dtype != (wide or w.dtype):
            raise ValueError("weights must be [head_dim] and of one dtype, float32 or query's, on "
                             "query's device")
        wide = w.dtype
    a.slot_dtype = _lib.DTYPE_I64
    if kv_cache is None:
        if value is not None or slot_mapping is not None:
            raise ValueError("value and slot_mapping go with a kv_cache")
        if key_out is None:
            key_out = torch.empty((t, hkv, d), dtype=dt, device=dev)
    else:
        if value is None or slot_mapping is None:
            raise ValueError("a cache write needs value and slot_mapping")
        a.v_stride_tok, a.v_stride_head = _rows("value", value, (t, hkv, d), dt, dev)
        a.v = value.data_ptr()
        slots = check_slots(slot_mapping, kv_cache)
        if kv_cache.device != dev:
            raise ValueError("kv_cache must be on query's device")
        if slots.shape[0] > t:
            raise ValueError(f"{slots.shape[0]} slots for {t} tokens")
        a.slot_mapping, a.num_slots, a.slot_dtype = slots.data_ptr(), slots.shape[0], \
            _INDEX[slots.dtype]
        if kv_cache.dtype == torch.uint8:
            desc, c_hkv, c_d = fp4_desc(kv_cache)
            a.cache_kind, a.fp4 = 2, ctypes.addressof(desc)
        else:
            if kv_cache.dtype != dt:
                raise ValueError("kv_cache must be of query's dtype, or a 4-bit cache (uint8)")
            desc, a.cache, c_hkv, c_d = _cache_desc(kv_cache)
            a.cache_kind = 1
        if c_hkv != hkv or c_d != d:
            raise ValueError("key heads or head_dim do not match the cache")
    if query_out is None:
        query_out = torch.empty((t, h, d), dtype=dt, device=dev)
        a.qo_stride_tok, a.qo_stride_head = h * d, d
    else:
        a.qo_stride_tok, a.qo_stride_head = _rows("query_out", query_out, (t, h, d), dt, dev)
    if key_out is not None:
        a.ko_stride_tok, a.ko_stride_head = _rows("key_out", key_out, (t, hkv, d), dt, dev)
        a.k_out = key_out.data_ptr()
    a.q, a.k, a.q_out = query.data_ptr(), key.data_ptr(), query_out.data_ptr()
    if q_weight is not None:
        a.q_weight = q_weight.data_ptr()
    if k_weight is not None:
        a.k_weight = k_weight.data_ptr()
    a.positions, a.pos_dtype = positions.data_ptr(), _INDEX[positions.dtype]
    a.num_tokens, a.eps, a.interleaved = t, eps, bool(interleaved)
    a.num_heads, a.num_kv_heads, a.head_dim, a.rot = h, hkv, d, rot
    a.dtype = a.weight_dtype = _lib.dtype_code(dt)
    if wide == torch.float32:
        a.weight_dtype = _lib.DTYPE_F32
    a.table_dtype = _lib.DTYPE_F32 if tab.dtype == torch.float32 else a.dtype
    with _lib.on_device(dev):
        rc = _lib.lib().hcp_qk_norm_rope(ctypes.addressof(a), _lib.stream_ptr(dev))
    _lib.check(rc, "hcp_qk_norm_rope")
    return query_out, key_out
