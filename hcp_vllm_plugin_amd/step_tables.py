"""A step's block table, slots and positions, built on the GPU.

The reference's engine makes these on the host and uploads them each step.
``build_step_tables`` makes them from the requests' lengths where those already
are: it takes the new blocks of every request off a list of free ones, and gives
the query starts, lengths, positions and slots that ``qk_rope.qk_norm_rope``,
``kv_cache.reshape_and_cache`` and ``HcpRingAttentionImpl.forward`` read, in one
launch and without waiting for the device.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

__all__ = ["StepTables", "build_step_tables"]

_INDEX = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}

# Storages that are written where no version counter tells: by every replay of a
# captured call, or as a table made under inference mode.
_UNSEEN: set[int] = set()


def written_unseen(*tensors: torch.Tensor) -> bool:
    """Whether ``build_step_tables`` writes one of these without a trace on the host."""
    return bool(_UNSEEN) and any(t.untyped_storage().data_ptr() in _UNSEEN for t in tensors)


class StepTables(NamedTuple):
    query_start_loc: torch.Tensor  # int32 [n + 1]
    seq_lens: torch.Tensor         # int32 [n]
    positions: torch.Tensor        # int64 [num_tokens]
    slot_mapping: torch.Tensor     # int64 [num_tokens]
    blocks_used: torch.Tensor      # int32 [1]


def _note_written(block_table: torch.Tensor, ints: torch.Tensor, index: int) -> None:
    """Who caches what a table says goes by its version counter (``ring_backend._step``)."""
    torch._C._increment_version((block_table,))  # (nothing under inference mode)
    if _lib.capturing(index):
        _UNSEEN.add(ints.untyped_storage().data_ptr())
        _UNSEEN.add(block_table.untyped_storage().data_ptr())
    elif block_table.is_inference():
        _UNSEEN.add(block_table.untyped_storage().data_ptr())


def build_step_tables(ctx_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                      free_blocks: torch.Tensor, block_size: int, num_tokens: int) -> StepTables:
    """Tables of a step in which request r, with ``ctx_lens[r]`` tokens in the
    cache, gets ``new_lens[r]`` more (int32 / int64 ``[n]``, at most 4096 requests).

    ``block_table`` (int32, n rows or more) names the blocks that hold the cached
    tokens; entries ``ceil(ctx / block_size)`` .. ``ceil((ctx + new) / block_size)
    - 1`` of row r are written, with the next ids of ``free_blocks`` (int32), the
    requests in order.  The step takes the first ``blocks_used`` of them; where
    that is more than there are, the entries without a block become -1 and the
    slots in them -1, which the cache writes skip, so a caller that may run out
    looks at ``blocks_used`` before it uses the step.  Tokens past the keys that a
    table row can name get slot -1 too, and take no block.

    ``positions`` and ``slot_mapping`` have ``num_tokens`` rows: the new tokens,
    then (padding) position 0 and slot -1.  Lengths below 0 count as 0.

    A captured call writes the same tensors at every replay, unseen by ``forward``
    outside the graph, as is a table made under inference mode that any call writes.
    ``forward`` reads these anew for a new metadata object, or when a layer comes
    again with a kept one; a caller whose next step begins with a layer that the last
    one left out calls ``ring_backend.invalidate_step_cache`` in between."""
    index, ints_of = block_table.get_device(), _INDEX.get
    ctx_code, new_code, (n, *more) = ints_of(ctx_lens.dtype), ints_of(new_lens.dtype), ctx_lens.shape
    if more or ctx_code is None or new_code is None or new_lens.shape != (n,):
        raise ValueError("ctx_lens and new_lens must be int32/int64 of one dimension and length")
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be int32 of two dimensions")
    (rows, width), (row, col) = block_table.shape, block_table.stride()
    if rows < n or (width > 1 and col != 1) or (n > 1 and row < width):
        raise ValueError("block_table must have contiguous rows, one for each request")
    if free_blocks.dtype != torch.int32 or free_blocks.dim() != 1 or not free_blocks.is_contiguous():
        raise ValueError("free_blocks must be contiguous int32 of one dimension")
    if index < 0 or ctx_lens.get_device() != index or new_lens.get_device() != index or \
            free_blocks.get_device() != index:
        raise ValueError("all tensors must be on one GPU")
    if block_size <= 0 or block_size & (block_size - 1):
        raise ValueError("block_size must be a power of two")
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    ints = torch.empty(2 * n + 2, dtype=torch.int32, device=block_table.device)
    wide = torch.empty(2, num_tokens, dtype=torch.int64, device=block_table.device)
    at, wide_at = ints.data_ptr(), wide.data_ptr()
    _lib.launch(_lib.lib().hcp_step_tables, index, "hcp_step_tables", _lib.pack_step_tables(
        ctx_lens.data_ptr(), new_lens.data_ptr(), ctx_lens.stride(0), new_lens.stride(0),
        block_table.data_ptr(), row, width, free_blocks.data_ptr(), free_blocks.shape[0],
        num_tokens, at, at + 4 * (n + 1), at + 4 * (2 * n + 1), wide_at, wide_at + 8 * num_tokens,
        ctx_code, new_code, n, block_size))
    _note_written(block_table, ints, index)
    starts, lens, used = ints.split_with_sizes((n + 1, n, 1))
    positions, slots = wide.unbind(0)
    return StepTables(starts, lens, positions, slots, used)
