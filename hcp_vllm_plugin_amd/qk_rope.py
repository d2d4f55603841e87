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
from .varlen import fp4_desc, rows_apart

__all__ = ["qk_norm_rope"]

_INDEX = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}


_TYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


def _rows(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype,
          index: int) -> tuple[int, int, int]:
    """Address, token and head stride of ``t``, which must have the kernel's rows."""
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, not {shape}")
    if t.dtype != dtype or t.get_device() != index:
        raise ValueError(f"{name} must be of query's dtype and device")
    (tok, head, col), at = t.stride(), t.data_ptr()
    if col != 1 or (at | 2 * tok | 2 * head) & 15:
        raise ValueError(f"{name}: 16-byte aligned rows with contiguous head_dim")
    return at, tok, head


def _out_rows(name: str, t: torch.Tensor, shape: tuple, dtype: torch.dtype,
              index: int) -> tuple[int, int, int]:
    """``_rows`` of a tensor that is written: its rows are apart."""
    at, tok, head = _rows(name, t, shape, dtype, index)
    if not rows_apart(t):
        raise ValueError(f"{name}: rows on top of each other")
    return at, tok, head


def _weight(t: torch.Tensor, d: int, dtype: torch.dtype, index: int) -> tuple[int, torch.dtype]:
    at, wd = t.data_ptr(), t.dtype
    if t.shape != (d,) or not t.is_contiguous() or at & 15 or t.get_device() != index or \
            (wd != dtype and wd != torch.float32):
        raise ValueError("weights must be [head_dim], float32 or of query's dtype, on its device")
    return at, wd


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
    slots are not written, the others are distinct); the key then comes back only where ``key_out`` asks
    for it.  ``query_out`` / ``key_out`` may be query and key themselves."""
    dt, index = query.dtype, query.get_device()
    code = _TYPES.get(dt)
    if code is None or index < 0 or query.dim() != 3 or key.dim() != 3:
        raise ValueError("query and key must be float16/bfloat16 [T, heads, D] on the GPU")
    t, h, d = query.shape
    hkv = key.shape[1]
    kv_shape = (t, hkv, d)
    q, q_tok, q_head = _rows("query", query, (t, h, d), dt, index)
    k, k_tok, k_head = _rows("key", key, kv_shape, dt, index)
    pos_code = _INDEX.get(positions.dtype)
    if pos_code is None or positions.shape != (t,) or positions.get_device() != index or \
            not positions.is_contiguous():
        raise ValueError("positions must be contiguous int32/int64 [T] on query's device")
    tab = cos_sin_cache
    wide_table = tab.dtype == torch.float32
    if tab.dim() != 2 or tab.get_device() != index or not (wide_table or tab.dtype == dt):
        raise ValueError("cos_sin_cache must be [max_positions, rot], float32 or query's dtype, on "
                         "query's device")
    (most, rot), (tab_row, col), tab_at = tab.shape, tab.stride(), tab.data_ptr()
    if rot:
        if rot % 16 or rot > d or most == 0:
            raise ValueError("rot must be a multiple of 16 up to head_dim, and the table not empty")
        if col != 1 or tab_at & 15 or tab_row & 7:
            raise ValueError("cos_sin_cache: 16-byte aligned rows")
    else:
        tab_at = tab_row = 0
    wq = wk = 0
    w_type = dt
    if q_weight is not None:
        wq, w_type = _weight(q_weight, d, dt, index)
    if k_weight is not None:
        wk, wt = _weight(k_weight, d, dt, index)
        if wq and wt != w_type:
            raise ValueError("q_weight and k_weight must be of one dtype")
        w_type = wt
    v = v_tok = v_head = slots_at = num_slots = cache = fp4 = kind = 0
    slot_code = pos_code
    if kv_cache is None:
        if value is not None or slot_mapping is not None:
            raise ValueError("value and slot_mapping go with a kv_cache")
    else:
        if value is None or slot_mapping is None:
            raise ValueError("a cache write needs value and slot_mapping")
        v, v_tok, v_head = _rows("value", value, kv_shape, dt, index)
        slots = check_slots(slot_mapping, kv_cache)
        if kv_cache.get_device() != index:
            raise ValueError("kv_cache must be on query's device")
        slots_at, num_slots, slot_code = slots.data_ptr(), slots.shape[0], _INDEX[slots.dtype]
        if num_slots > t:
            raise ValueError(f"{num_slots} slots for {t} tokens")
        if kv_cache.dtype == torch.uint8:
            desc, c_hkv, c_d = fp4_desc(kv_cache)
            kind, fp4 = 2, ctypes.addressof(desc)
        else:
            if kv_cache.dtype != dt:
                raise ValueError("kv_cache must be of query's dtype, or a 4-bit cache (uint8)")
            desc, cache, c_hkv, c_d = _cache_desc(kv_cache)
            kind = 1
        if c_hkv != hkv or c_d != d:
            raise ValueError("key heads or head_dim do not match the cache")
    if query_out is None:
        query_out = torch.empty(t, h, d, dtype=dt, device=query.device)
        qo, qo_tok, qo_head = query_out.data_ptr(), h * d, d
    else:
        qo, qo_tok, qo_head = _out_rows("query_out", query_out, (t, h, d), dt, index)
    ko = ko_tok = ko_head = 0
    if key_out is None and not kind:
        key_out = torch.empty(t, hkv, d, dtype=dt, device=query.device)
        ko, ko_tok, ko_head = key_out.data_ptr(), hkv * d, d
    elif key_out is not None:
        ko, ko_tok, ko_head = _out_rows("key_out", key_out, kv_shape, dt, index)
    _lib.launch(_lib.lib().hcp_qk_norm_rope, index, "hcp_qk_norm_rope", _lib.pack_qk_rope(
        q, q_tok, q_head, k, k_tok, k_head, v, v_tok, v_head, qo, qo_tok, qo_head, ko, ko_tok,
        ko_head, wq, wk, positions.data_ptr(), tab_at, tab_row, most, slots_at, num_slots, cache,
        fp4, t, eps, h, hkv, d, rot, code, code if w_type == dt else _lib.DTYPE_F32,
        _lib.DTYPE_F32 if wide_table else code, pos_code, slot_code, bool(interleaved), kind, 0))
    return query_out, key_out
