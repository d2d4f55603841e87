"""A decode step with drafted tokens: their attention, and which of them stay.

``decode_drafts`` is the attention of every sequence's last few tokens (the newest
one and those drafted behind it) over the paged cache, in 16 bits or 4, one launch
for a ragged batch.  ``verify_drafts`` takes the target model's logits (or
probabilities) for these rows and says which drafts are accepted and what comes after
them.  The reference has neither: vLLM hands such rows to its prefill path
(hcp_vllm_plugin/ring_backend.py:820-830 runs them request by request).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .varlen import PagedCache, fp4_fields, rows_apart

__all__ = ["decode_drafts", "verify_drafts", "VerifiedDrafts"]

_INDEX = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}
_TYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_REAL = {**_TYPES, torch.float32: _lib.DTYPE_F32}
# partials of one launch, at most (a larger batch takes several)
_WORKSPACE = 1 << 28


def decode_drafts(
    q: torch.Tensor,
    kv_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    max_tokens: int,
    scale: float,
    window: int | None = None,
    out: torch.Tensor | None = None,
    with_lse: bool = False,
):
    """Attention of q ``[T, H, D]`` (fp16 / bf16), whose rows ``query_start_loc[r]`` ..
    ``query_start_loc[r + 1] - 1`` are the last n tokens of sequence r, over a paged cache
    that holds their keys: token i of them sees keys ``[0, seq_lens[r] - n + 1 + i)`` of
    row r of ``block_table``, the last ``window`` of them.  The first ``max_tokens`` (1 to
    64) of a sequence's n are run; the others, and those in rows past q's, are not.

    ``kv_cache`` is of q's dtype, in either 16-bit layout, or a 4-bit cache (uint8).
    Lengths (int32 / int64 ``[S]``), row starts (``[S + 1]``, of their dtype) and block ids
    are read on the device when the call executes; a length past its table row counts as
    the row's keys, a block id past the cache as its last block.  A token that sees no
    key (or none with a score above -inf) gets out 0 and LSE -inf, one with a NaN score NaN;
    a key that it does not see cannot reach it, whatever it holds.  Rows of ``out`` that belong to no sequence are
    left as they were.  Returns out (and lse float32 ``[H, T]``), to be merged with other
    keys' by ``merge_attn_states``."""
    dt, index = q.dtype, q.get_device()
    code = _TYPES.get(dt)
    if code is None or q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("q must be float16/bfloat16 [T, H, D] with contiguous head_dim")
    t, h, d = q.shape
    fp4 = kv_cache.dtype == torch.uint8
    if fp4:
        (k_at, c_block, c_head, blocks, bs, dim), hkv, _ = fp4_fields(kv_cache)
        v_at = c_tok = 0
    else:
        if kv_cache.dtype != dt:
            raise ValueError("kv_cache must be of q's dtype, or a 4-bit cache (uint8)")
        pc = PagedCache.from_tensor(kv_cache)
        k_at, v_at, c_tok, c_head, c_block = \
            pc.k_addr, pc.v_addr, pc.stride_tok, pc.stride_head, pc.stride_block
        blocks, bs, hkv, dim = kv_cache.shape[0], pc.block_size, pc.num_kv_heads, pc.head_dim
    if d != dim or not hkv or h % hkv or not h:
        raise ValueError("the cache must have q's head_dim, its heads dividing q's")
    if not 1 <= max_tokens <= _lib.DRAFTS_MAX_TOKENS:
        raise ValueError(f"max_tokens must be 1 to {_lib.DRAFTS_MAX_TOKENS}")
    if window is not None and window <= 0:
        raise ValueError("window must be a positive number of keys")
    lens_code, s = _INDEX.get(seq_lens.dtype), seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    if lens_code is None or s < 0 or not seq_lens.is_contiguous() or seq_lens.get_device() != index:
        raise ValueError("seq_lens must be contiguous int32/int64 [S] on q's GPU")
    if query_start_loc.dtype != seq_lens.dtype or query_start_loc.shape != (s + 1,) or \
            not query_start_loc.is_contiguous() or query_start_loc.get_device() != index:
        raise ValueError("query_start_loc must be [S + 1], of seq_lens' dtype and device")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or \
            block_table.get_device() != index:
        raise ValueError("block_table must be int32 of two dimensions on q's GPU")
    (rows, width), (bt_row, bt_col) = block_table.shape, block_table.stride()
    if rows < s or (width > 1 and bt_col != 1):
        raise ValueError("block_table must have contiguous rows, one for each sequence")
    if index < 0 or kv_cache.get_device() != index:
        raise ValueError("all tensors must be on one GPU")
    q_at, (q_tok, q_head, _) = q.data_ptr(), q.stride()
    if (q_at | 2 * q_tok | 2 * q_head) & 15:
        q = q.contiguous()
        q_at, (q_tok, q_head, _) = q.data_ptr(), q.stride()
    if out is None:
        out = torch.empty(t, h, d, dtype=dt, device=q.device)
    elif out.shape != q.shape or out.dtype != dt or out.stride(2) != 1 or \
            out.get_device() != index or not rows_apart(out):
        raise ValueError("out must be as q, with contiguous head_dim and its rows apart")
    lse = torch.empty(h, t, dtype=torch.float32, device=q.device) if with_lse else None
    out_at, (o_tok, o_head, _), lse_at = out.data_ptr(), out.stride(), \
        lse.data_ptr() if with_lse else 0
    bt_at, lens_at, starts_at = block_table.data_ptr(), seq_lens.data_ptr(), \
        query_start_loc.data_ptr()
    wide = 8 if lens_code == _lib.DTYPE_I64 else 4
    # (a launch's keys are counted in 32-key chunks, in 32 bits)
    most = max(1, min(_lib.DECODE_PAGED_MAX_SEQS, (1 << 34) // max(1, width * bs)))
    if s > 1:
        one, two = (_lib.decode_drafts_workspace(n, max_tokens, h, hkv, d, fp4) for n in (1, 2))
        most = min(most, max(1, (_WORKSPACE - one) // max(1, two - one)))
    for r in range(0, s if t else 0, most):
        n = min(s - r, most)
        # fp32 partials: stream-ordered scratch from torch's caching allocator
        size = _lib.decode_drafts_workspace(n, max_tokens, h, hkv, d, fp4)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        _lib.launch(_lib.lib().hcp_decode_drafts, index, "hcp_decode_drafts", _lib.pack_decode_drafts(
            q_at, q_tok, q_head, k_at, v_at, bt_at + 4 * r * bt_row, c_tok, c_head, c_block, 0, 0,
            bs, blocks, bt_row, width, lens_at + wide * r, ws.data_ptr(), size, out_at, o_tok,
            o_head, lse_at, t, lens_code, n, min(window or 0, 0x3fffffff), h, hkv, d, code, 0,
            scale, 0, starts_at + wide * r, t, max_tokens, fp4))
    return (out, lse) if with_lse else out


class VerifiedDrafts(NamedTuple):
    tokens: torch.Tensor      # [S, max_tokens], as the drafts: the accepted ones, one more, -1
    num_tokens: torch.Tensor  # int32 [S]


def verify_drafts(
    target: torch.Tensor,
    tokens: torch.Tensor,
    query_start_loc: torch.Tensor,
    uniform: torch.Tensor,
    *,
    draft_probs: torch.Tensor | None = None,
    temperature: torch.Tensor | None = None,
    probs: bool = False,
) -> VerifiedDrafts:
    """Which drafted tokens the target model accepts, and the token after them.

    ``target`` ``[T, V]`` (fp16 / bf16 / float32) are its logits, -inf for tokens that were
    cut off, or with ``probs`` its probabilities (of any sum); ``tokens`` ``[T]`` (int32 /
    int64) what the step ran on.  Rows ``query_start_loc[r]`` .. ``query_start_loc[r + 1] -
    1`` are sequence r's newest token and its drafts: row i judges the token of row i + 1,
    the last row is the one after all of them.  A draft d with probability p(d) by the
    target is accepted while ``uniform[r, i] < p(d) / q(d)``, q being ``draft_probs[r, i]``
    ``[S, max_tokens - 1, V]`` (float32), or 1: a draft looked up, not drawn.  The token
    after the accepted ones is drawn from ``max(p - q, 0)`` of the row that refused (from p
    without the draft where there is no q), or from the last row's p, at
    ``uniform[r, -1]`` of the sum in the order of the tokens.  So a sequence without drafts
    has its next token drawn.  ``uniform`` is float32 ``[S, max_tokens]`` in [0, 1): its
    second size says how many rows of a sequence are looked at, 1 to 64.

    ``temperature`` float32 ``[S]`` divides the logits (None: 1); where it is not above 0
    the largest entry above -inf, the lowest index of equal ones, takes the place of the
    draw.  Tokens are as sums in 64 bits give them, at any temperature.  A NaN has no weight and
    is no entry; a row without any accepts no draft and gives no token, and a draft that is
    no token of the vocabulary is refused."""
    code, index = _REAL.get(target.dtype), target.get_device()
    if code is None or target.dim() != 2 or (target.shape[1] > 1 and target.stride(1) != 1):
        raise ValueError("target must be float16/bfloat16/float32 [T, V] with contiguous rows")
    (t, v), row = target.shape, target.stride(0)
    tok_code = _INDEX.get(tokens.dtype)
    if tok_code is None or tokens.shape != (t,) or not tokens.is_contiguous() or \
            tokens.get_device() != index:
        raise ValueError("tokens must be contiguous int32/int64 [T] on target's GPU")
    start_code = _INDEX.get(query_start_loc.dtype)
    if start_code is None or query_start_loc.dim() != 1 or query_start_loc.shape[0] < 1 or \
            not query_start_loc.is_contiguous() or query_start_loc.get_device() != index:
        raise ValueError("query_start_loc must be contiguous int32/int64 [S + 1] on target's GPU")
    s = query_start_loc.shape[0] - 1
    if uniform.dtype != torch.float32 or uniform.dim() != 2 or uniform.shape[0] != s or \
            not 1 <= uniform.shape[1] <= _lib.VERIFY_MAX_TOKENS or uniform.get_device() != index or \
            (uniform.shape[1] > 1 and uniform.stride(1) != 1):
        raise ValueError("uniform must be float32 [S, max_tokens] with contiguous rows on target's "
                         f"GPU, max_tokens 1 to {_lib.VERIFY_MAX_TOKENS}")
    most = uniform.shape[1]
    q_at = q_seq = q_row = 0
    if draft_probs is not None:
        if draft_probs.dtype != torch.float32 or draft_probs.dim() != 3 or \
                draft_probs.shape[0] != s or draft_probs.shape[1] < most - 1 or \
                draft_probs.shape[2] != v or (v > 1 and draft_probs.stride(2) != 1) or \
                draft_probs.get_device() != index:
            raise ValueError("draft_probs must be float32 [S, max_tokens - 1, V] with contiguous "
                             "rows on target's GPU")
        q_at, (q_seq, q_row, _) = draft_probs.data_ptr(), draft_probs.stride()
    t_at = 0
    if temperature is not None:
        if temperature.dtype != torch.float32 or temperature.shape != (s,) or \
                not temperature.is_contiguous() or temperature.get_device() != index:
            raise ValueError("temperature must be contiguous float32 [S] on target's GPU")
        t_at = temperature.data_ptr()
    if index < 0:
        raise ValueError("all tensors must be on one GPU")
    if not v:
        raise ValueError("target must have tokens")
    out = torch.empty(s, most, dtype=tokens.dtype, device=target.device)
    num = torch.empty(s, dtype=torch.int32, device=target.device)
    if s:
        size = _lib.verify_workspace(s, most, v)
        ws = torch.empty(size, dtype=torch.uint8, device=target.device)
        _lib.launch(_lib.lib().hcp_verify_drafts, index, "hcp_verify_drafts", _lib.pack_verify(
            target.data_ptr(), row, t, tokens.data_ptr(), query_start_loc.data_ptr(),
            uniform.data_ptr(), uniform.stride(0), q_at, q_seq, q_row, t_at, out.data_ptr(),
            num.data_ptr(), ws.data_ptr(), size, v, s, most, code, tok_code, start_code, probs, 0))
    return VerifiedDrafts(out, num)
