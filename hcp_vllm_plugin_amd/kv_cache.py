"""Paged KV-cache write on the HIP kernel (the step before the attention path).

``reshape_and_cache(key, value, kv_cache, slot_mapping)`` writes this step's
K/V rows into the paged cache at ``slot_mapping`` (slot = block * block_size
+ offset): the operation of the reference's ``do_kv_cache_update``
(hcp_vllm_plugin/ring_backend.py:501-539), which does it with torch advanced
indexing into the vLLM 0.23 layout ``[nb, 2, bs, Hkv, D]``, and of vLLM's
``reshape_and_cache`` for the 0.31 layout ``[nb, Hkv, bs, 2*D]`` that the
paged local-segment reader consumes (file_connector.py:13-16).  Rows ``t <
len(slot_mapping)`` of key/value are written (key may be padded past that, as
in the reference's ``key[:n]``); a negative slot is a padding token and is
skipped.

The 4-bit cache (``fp4_cache_shape``) holds K and V as 4-bit codes (sign, two
bits of exponent, one of mantissa) with a power-of-two scale for 32 columns of a
head's row, 17 / 32 byte a value; the format is in include/hcp_mi355x.h
(``hcp_fp4_cache``).  ``reshape_and_cache`` writes it, ``gather_kv`` reads back
what it stands for, ``varlen.decode_fp4`` and the backend with
``kv_cache_dtype="fp4"`` attend over it.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .varlen import PagedCache, fp4_fields

__all__ = ["reshape_and_cache", "fp4_cache_shape", "gather_kv"]

# Cache descriptors by (address, shape, strides, dtype): the write runs once per
# layer and step, and building the descriptor each time was a third of its
# host cost.  The key fixes every field the descriptor holds, so a descriptor
# found here is the one the tensor would produce.
_DESCS: dict = {}
_MAX_DESCS = 1024


def _cache_desc(kv_cache: torch.Tensor):
    ck = (kv_cache.data_ptr(), tuple(kv_cache.shape), kv_cache.stride(), kv_cache.dtype)
    ent = _DESCS.get(ck)
    if ent is None:
        pc = PagedCache.from_tensor(kv_cache)
        desc = _lib.PagedCacheDesc()
        desc.k_addr = pc.k_addr
        desc.v_addr = pc.v_addr
        desc.stride_block = pc.stride_block
        desc.stride_head = pc.stride_head
        desc.stride_tok = pc.stride_tok
        desc.num_blocks = kv_cache.shape[0]
        desc.block_size = pc.block_size
        if len(_DESCS) >= _MAX_DESCS:
            _DESCS.clear()
        ent = _DESCS[ck] = (desc, ctypes.addressof(desc), pc.num_kv_heads, pc.head_dim)
    return ent


def fp4_cache_shape(num_blocks: int, num_kv_heads: int, block_size: int,
                    head_dim: int) -> tuple[int, int, int, int]:
    """Shape of the uint8 tensor that is a 4-bit cache of these sizes."""
    if head_dim % 32 or not 0 < head_dim <= 256:
        raise ValueError(f"4-bit cache: head_dim {head_dim} is not a multiple of 32 up to 256")
    if block_size & (block_size - 1) or not 16 <= block_size <= 65536:
        raise ValueError(f"4-bit cache: block_size {block_size} is not a power of two from 16 to 65536")
    return (num_blocks, num_kv_heads, block_size, head_dim + head_dim // 16)


_INDEX_CODES = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}
_TYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


def check_slots(slot_mapping: torch.Tensor, kv_cache: torch.Tensor) -> torch.Tensor:
    """``slot_mapping`` as the kernels read it."""
    if slot_mapping.dtype not in _INDEX_CODES or slot_mapping.dim() != 1:
        raise ValueError("slot_mapping must be int32 or int64, of one dimension")
    index = kv_cache.get_device()
    if index < 0 or slot_mapping.get_device() != index:
        raise ValueError("slot_mapping must be on the cache's GPU")
    return slot_mapping if slot_mapping.is_contiguous() else slot_mapping.contiguous()


def _write_fp4(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor,
               slot_mapping: torch.Tensor) -> None:
    cache, hkv, d = fp4_fields(kv_cache)
    n, shape, dt, index = slot_mapping.shape[0], key.shape, key.dtype, kv_cache.get_device()
    if shape != value.shape or len(shape) != 3:
        raise ValueError("key/value must be [N, Hkv, D] of one shape")
    if shape[0] < n:
        raise ValueError(f"{n} slots for {shape[0]} key rows")
    if shape[1] != hkv or shape[2] != d:
        raise ValueError("key/value heads or head_dim do not match the cache")
    code = _TYPES.get(dt)
    if code is None or value.dtype != dt:
        raise ValueError("key/value must both be float16 or bfloat16")
    (k_tok, k_head, k_col), (v_tok, v_head, v_col) = key.stride(), value.stride()
    if k_col != 1 or v_col != 1:
        raise ValueError("key/value head_dim must be contiguous")
    slots = check_slots(slot_mapping, kv_cache)
    if key.get_device() != index or value.get_device() != index:
        raise ValueError("key/value must be on the cache's GPU")
    if n == 0:
        return
    _lib.launch(_lib.lib().hcp_fp4_write, index, "hcp_fp4_write", key.data_ptr(), k_tok, k_head,
                value.data_ptr(), v_tok, v_head, slots.data_ptr(), _INDEX_CODES[slots.dtype], n,
                hkv, _lib.pack_fp4_cache(*cache), code)


def gather_kv(kv_cache: torch.Tensor, slot_mapping: torch.Tensor,
              dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V ``[n, Hkv, D]`` that a 4-bit cache stands for at ``slot_mapping``,
    in the 16-bit ``dtype`` they were written in (exactly: a code's value has two
    significant bits).  A slot that is negative or past the cache reads as zeros."""
    code = _TYPES.get(dtype)
    if code is None:
        raise ValueError("dtype must be float16 or bfloat16")
    cache, hkv, d = fp4_fields(kv_cache)
    slots = check_slots(slot_mapping, kv_cache)
    n, index = slots.shape[0], slots.get_device()
    kv = torch.empty(2, n, hkv, d, dtype=dtype, device=kv_cache.device)
    base = kv.data_ptr()
    _lib.launch(_lib.lib().hcp_fp4_read, index, "hcp_fp4_read", slots.data_ptr(),
                _INDEX_CODES[slots.dtype], n, hkv, _lib.pack_fp4_cache(*cache), code, base,
                base + 2 * n * hkv * d)
    return kv.unbind(0)


def reshape_and_cache(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor,
                      slot_mapping: torch.Tensor) -> None:
    """Write ``key``/``value`` ``[N, Hkv, D]`` rows ``[0, n)``, ``n =
    slot_mapping.numel()``, into ``kv_cache`` at ``slot_mapping``; into a 4-bit
    cache (uint8) as its codes.  Slots inside the cache are distinct."""
    if kv_cache.dtype == torch.uint8:
        return _write_fp4(key, value, kv_cache, slot_mapping)
    _, desc_addr, hkv, d = _cache_desc(kv_cache)
    n = slot_mapping.numel()
    if key.shape != value.shape or key.dim() != 3:
        raise ValueError("key/value must be [N, Hkv, D] of one shape")
    if key.shape[0] < n:
        raise ValueError(f"{n} slots for {key.shape[0]} key rows")
    if key.shape[1] != hkv or key.shape[2] != d:
        raise ValueError("key/value heads or head_dim do not match the cache")
    if key.dtype != kv_cache.dtype or value.dtype != kv_cache.dtype:
        raise ValueError("key/value dtype must match the cache dtype")
    if key.stride(-1) != 1 or value.stride(-1) != 1:
        raise ValueError("key/value head_dim must be contiguous")
    if slot_mapping.dtype not in (torch.int32, torch.int64):
        raise ValueError("slot_mapping must be int32 or int64")
    if n == 0:
        return
    slots = slot_mapping.contiguous()
    L = _lib.lib()
    args = (key.data_ptr(), key.stride(0), key.stride(1),
            value.data_ptr(), value.stride(0), value.stride(1),
            slots.data_ptr(), _lib.DTYPE_I64 if slots.dtype == torch.int64 else _lib.DTYPE_I32,
            n, hkv, d, desc_addr, _lib.dtype_code(key.dtype))
    dev = key.device
    if dev.index == torch.cuda.current_device():
        rc = L.hcp_reshape_and_cache(*args, torch.cuda.current_stream(dev).cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = L.hcp_reshape_and_cache(*args, _lib.stream_ptr(dev))
    _lib.check(rc, "hcp_reshape_and_cache")
