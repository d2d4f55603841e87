"""HCP ring-attention backend on the MI355X HIP kernels.

Drop-in for hcp_vllm_plugin/ring_backend.py's hot path:

* ``HcpRingAttentionBackend`` -- ``get_name() == "CUSTOM"``, ``get_impl_cls``,
  ``get_builder_cls``, ``forward_includes_kv_cache_update = False``
  (ring_backend.py:427-449).  When vLLM is importable it subclasses vLLM's
  ``FlashAttentionBackend`` exactly as the reference does (ring_backend.py:71-74);
  without vLLM it is a plain class with the same static methods.
* ``HcpRingAttentionImpl`` -- ``__init__`` (ring_backend.py:464-498) and
  ``forward(layer, query, key, value, kv_cache, attn_metadata, output,
  output_scale=None, output_block_scale=None)`` (ring_backend.py:576-834) with
  the reference's segmentation: vanilla causal attention when a request has no
  peer, plain causal attention for the ``n_a`` queries inside the peer region,
  and for the rest local causal attention over ``[peer_end, tk)`` at offset
  ``qpos0 + n_a - peer_end`` merged with non-causal attention over the peer.
  Instead of a Python loop with a gather copy and 5-6 launches per request,
  a whole batch runs as one launch over the staged peer KV and one varlen
  launch over the paged cache (read in place) that also merges the peer
  result into the output; a pure decode batch runs the split-KV decode
  kernel.
* ``_attn`` / ``_merge`` (ring_backend.py:309-360) with ``HCP_RING_IMPL`` /
  ``HCP_RING_MERGE`` read on every call.  ``hip`` is the default; ``triton``
  is accepted as an alias so existing launch scripts keep working.  There is
  no torch fallback in this package: ``torch`` raises, and a kernel error
  raises instead of silently switching paths.
* The peer-KV staging input contract (ring_backend.py:78-136):
  ``PEER_KV_STAGING[(chunk_key, layer_name)] = (k, v)`` with k/v
  ``[n, Hkv, D]`` post-RoPE, ``PEER_REQ_MAP[first_block_id] = [chunk keys]``.
* Memory-split decode (accumulator ring, ring_backend.py:140-227, :632-722):
  ``register_decode_ring`` / ``clear_decode_ring`` / ``DECODE_RING_MAP``.  A
  registered request's single-token decode step skips the pool write, and its
  attention is the owner's local partial (own chunk in the pool + owned growth
  + current token) sent around the ring by ``ring_decode.ring_decode_step``;
  decode growth is sharded by ``ring_decode.growth_assignee``.  In a pure
  decode batch the owner partials run in the same split-KV launch as the
  other rows.
* ``kv_cache_dtype="fp4"``: the paged cache holds 4-bit codes (``kv_cache``).
  Decode rows read them as they lie; prefill chunks run on their keys expanded
  to 16 bits, per layer, in scratch.  Staged peers stay 16-bit and merge with
  either as ever; the decode ring and ``HCP_RING_SPLIT_TOKENS`` need a 16-bit
  cache.
* ``IMPL_STATS`` evidence counters (ring_backend.py:295-306).  ``attn_hip`` /
  ``merge_hip`` count kernel launches and merges (a merge done inside the
  local pass counts as one); the legacy keys ``attn_triton`` /
  ``merge_triton`` mirror them so validators that read those names still see
  which path ran, and ``attn_torch`` / ``merge_torch`` stay 0.
* The validators' other evidence (ring_backend.py:228-275, :790-810), same
  names and meaning: ``STAGING_STATS`` / ``reset_staging_stats`` (staging
  high-water marks), ``WRITE_TRACK`` / ``reset_write_tracking`` (pool slots
  written, the chunk-A ``overlap`` probe in ``forward``, decode-ring
  ``skipped`` writes) and ``BATCH_STATS`` / ``reset_batch_stats``.
"""

from __future__ import annotations

import enum
import logging
import os
import threading

import numpy as np
import torch

from . import _lib
from .kv_cache import reshape_and_cache
from .merge import merge_attn_states
from .ring_attn import COPY_STATS, ring_attn_with_lse
from .ring_decode import GrowthBuffer, growth_assignee, local_partial, ring_decode_step
from .step_tables import written_unseen
from .varlen import (
    _MIN_PAGED_BLOCK,
    ENTRY_DTYPE,
    head_major,
    DecodeBatch,
    PagedCache,
    PagedDecode,
    VarlenLaunch,
    _upload,
    make_entry,
    paged_entry_array,
    segment_contiguous,
    segment_paged,
    trim_segment,
    window_tail,
)

logger = logging.getLogger(__name__)

try:  # optional: the real vLLM base classes, as the reference uses them
    from vllm.v1.attention.backend import AttentionImpl as _ImplBase  # type: ignore
    from vllm.v1.attention.backend import AttentionType  # type: ignore
    from vllm.v1.attention.backends.flash_attn import (  # type: ignore
        FlashAttentionBackend as _BackendBase,
        FlashAttentionMetadataBuilder as _BuilderCls,
    )

    HAVE_VLLM = True
except ImportError:  # vLLM absent: same surface, no base classes
    HAVE_VLLM = False
    _ImplBase = object
    _BackendBase = object
    _BuilderCls = None

    class AttentionType(str, enum.Enum):  # type: ignore[no-redef]
        DECODER = "decoder"
        ENCODER = "encoder"
        ENCODER_ONLY = "encoder_only"
        ENCODER_DECODER = "encoder_decoder"


# ---------------------------------------------------------------------------
# Peer KV staging (input contract; the connector writes, forward reads)
# ---------------------------------------------------------------------------
PEER_KV_STAGING: dict[tuple[str, str], tuple[torch.Tensor, torch.Tensor]] = {}
PEER_REQ_MAP: dict[int, list[str]] = {}
# (chunk_key, layer_name) -> (event recorded after the staged copy was queued,
# streams already ordered after it); a forward on any stream waits on the
# event once before reading the chunk
_STAGE_READY: dict[tuple[str, str], tuple[torch.cuda.Event, set]] = {}
# Bumped whenever a chunk key appears in or leaves the staging dict, or the
# request map changes: which requests take which chunks (the decode-step
# template) is decided from these, and stays valid while the count holds.
# (A further layer of an already staged chunk does not bump it; each layer's
# lookup checks its own entry.)
_STAGE_GEN = [0]
_CHUNK_LAYERS: dict[str, int] = {}  # chunk key -> layers staged


def stage_peer_kv(chunk_key: str, layer_name: str, k: torch.Tensor, v: torch.Tensor,
                  ready: torch.cuda.Event | None = None) -> None:
    """Stage a peer chunk's K/V ``[n, Hkv, D]`` (post-RoPE) for one layer.

    Stored head-major (one copy per chunk and layer): a chunk is staged once
    and read by every decode step, and the split-KV decode streams a KV head's
    keys 5% faster as one contiguous run than as rows interleaved with the
    other heads'; the prefill passes read either layout at the same rate.

    Ordering: the copy is queued on the caller's current stream.  ``ready``
    (e.g. ``IngestedKV.event`` of a ``PeerIngest.load`` on a side stream) is
    waited on by that stream first, so the copy reads landed bytes.  An event
    recorded after the copy is kept with the entry and every forward that
    reads the chunk makes its own stream wait on it, so staging from a
    connector thread's stream and reading from the model's stream is ordered
    on the device without a host synchronisation.
    """
    on_gpu = k.is_cuda
    if on_gpu and ready is not None:
        torch.cuda.current_stream(k.device).wait_event(ready)
    key = (chunk_key, layer_name)
    if key not in PEER_KV_STAGING:
        _CHUNK_LAYERS[chunk_key] = _CHUNK_LAYERS.get(chunk_key, 0) + 1
        if _CHUNK_LAYERS[chunk_key] == 1:
            _STAGE_GEN[0] += 1
    PEER_KV_STAGING[key] = (head_major(k), head_major(v))
    if on_gpu:
        st = torch.cuda.current_stream(k.device)
        ev = torch.cuda.Event()
        ev.record(st)
        _STAGE_READY[key] = (ev, {st})
    else:
        _STAGE_READY.pop(key, None)
    _note_staging(k)


# High-water marks of the staging dict (ring_backend.py:228-251): staging is
# freed when a request finishes, so post-run checks read these instead.
STAGING_STATS: dict = {"max_concurrent_chunks": 0, "max_staged_layers": 0, "last_chunk_len": 0}


def reset_staging_stats() -> None:
    STAGING_STATS["max_concurrent_chunks"] = 0
    STAGING_STATS["max_staged_layers"] = 0
    STAGING_STATS["last_chunk_len"] = 0


def _note_staging(k: torch.Tensor) -> None:
    """Raise the high-water marks after a stage: (chunk, layer) entries held,
    distinct chunks held, and the token count of the chunk just staged."""
    STAGING_STATS["max_staged_layers"] = max(STAGING_STATS["max_staged_layers"],
                                             len(PEER_KV_STAGING))
    chunks = {key[0] for key in PEER_KV_STAGING}
    STAGING_STATS["max_concurrent_chunks"] = max(STAGING_STATS["max_concurrent_chunks"],
                                                 len(chunks))
    STAGING_STATS["last_chunk_len"] = int(k.shape[0])


def _wait_staged(key: tuple[str, str], kv: tuple[torch.Tensor, torch.Tensor],
                 cur: torch.cuda.Stream | None = None) -> None:
    """Order the current stream after the staging copy of ``key`` (once per
    stream).  A chunk staged on another stream is also marked as used on this
    one, so the caching allocator keeps its memory until this stream's reads
    are done even if the chunk is dropped meanwhile."""
    ent = _STAGE_READY.get(key)
    if ent is None:
        return
    ev, seen = ent
    if cur is None:  # (a caller with many chunks looks it up once)
        cur = torch.cuda.current_stream(kv[0].device)
    if cur in seen:
        return
    cur.wait_event(ev)
    for t in kv:
        t.record_stream(cur)
    seen.add(cur)


def drop_chunk_kv(chunk_key: str) -> int:
    keys = [key for key in PEER_KV_STAGING if key[0] == chunk_key]
    for key in keys:
        del PEER_KV_STAGING[key]
        _STAGE_READY.pop(key, None)
    if _CHUNK_LAYERS.pop(chunk_key, None) is not None:
        _STAGE_GEN[0] += 1
    return len(keys)


def map_request_peer(first_block_id: int, chunk_keys) -> None:
    """Bind a request (by its first block id) to its ordered prefix chunks."""
    if isinstance(chunk_keys, str):
        chunk_keys = [chunk_keys]
    chunk_keys = list(chunk_keys)
    if PEER_REQ_MAP.get(first_block_id) != chunk_keys:
        PEER_REQ_MAP[first_block_id] = chunk_keys
        _STAGE_GEN[0] += 1


def unmap_request_peer(first_block_id: int) -> None:
    if PEER_REQ_MAP.pop(first_block_id, None) is not None:
        _STAGE_GEN[0] += 1


def request_peer_chunk(first_block_id: int) -> list[str] | None:
    return PEER_REQ_MAP.get(first_block_id)


def clear_peer_kv() -> None:
    PEER_KV_STAGING.clear()
    PEER_REQ_MAP.clear()
    _STAGE_READY.clear()
    _CHUNK_LAYERS.clear()
    _STAGE_GEN[0] += 1


# ---------------------------------------------------------------------------
# Memory-split decode registry (ring_backend.py:140-227)
# ---------------------------------------------------------------------------
DECODE_RING_MAP: dict[int, dict] = {}
_STAGING_RELEASE_FN = None


def _decode_ring_enabled() -> bool:
    return os.environ.get("HCP_RING_DECODE_RING", "1") == "1"


def _growth_policy() -> str:
    return os.environ.get("HCP_RING_DECODE_GROWTH", "rr")


def set_staging_release_fn(fn) -> None:
    """Connector callback that frees a request's staged prefix KV."""
    global _STAGING_RELEASE_FN
    _STAGING_RELEASE_FN = fn


def register_decode_ring(first_block_id: int, peer_chunks: list[tuple[str, str]],
                         prefix_len: int, transport=None) -> None:
    """Switch a request to memory-split decode (ring_backend.py:175-208).

    ``peer_chunks``: ordered ``(chunk_key, peer_url)`` of the prefix (entries
    with an empty url are dropped); ``prefix_len``: tokens of the prefix;
    ``transport``: the ring transport (``send_packet`` / ``recv_packet``).
    Ring indices: 0..N-2 the prefix peers, N-1 the owner.
    """
    import uuid

    peers = [(ck, u) for ck, u in peer_chunks if u]
    DECODE_RING_MAP[first_block_id] = {
        "peer_chunks": peers,
        "prefix_len": prefix_len,
        "req_tag": f"{first_block_id}:{uuid.uuid4().hex[:8]}",
        "ring_size": len(peers) + 1,
        "own_index": len(peers),
        "own_chunk_len": None,     # set at the first decode step
        "growth": {},              # layer -> GrowthBuffer (owner's share)
        "pending_growth": {},      # layer -> (assignee, k, v), shipped next step
        "growth_policy": _growth_policy(),
        "transport": transport,
    }


def clear_decode_ring(first_block_id: int) -> None:
    DECODE_RING_MAP.pop(first_block_id, None)


def _release_staged_for_request(first_block_id: int) -> None:
    """Free a request's staged prefix KV at its decode-ring transition
    (ring_backend.py:214-225)."""
    if first_block_id not in PEER_REQ_MAP:
        return
    if _STAGING_RELEASE_FN is not None:
        _STAGING_RELEASE_FN(first_block_id)
    else:
        for ck in PEER_REQ_MAP.pop(first_block_id, None) or []:
            drop_chunk_kv(ck)


def _chunk_words(kvs: list) -> np.ndarray:
    """K address, V address, token and head stride of each staged chunk
    (contiguous k/v ``[n, Hkv, D]``), checked as ``segment_contiguous`` checks
    one."""
    rows, low = [], 0
    for k, v in kvs:
        st, kp, vp = k.stride(), k.data_ptr(), v.data_ptr()
        es = k.element_size()
        low |= kp | vp | st[0] * es | st[1] * es
        if st != v.stride() or not 0 < st[0] < 1 << 24:
            raise ValueError("staged chunk: k/v layout not loadable")
        rows.append((kp, vp, st[0], st[1]))
    if low % 16:
        raise ValueError("staged chunk: k/v layout not loadable")
    return np.array(rows, dtype=np.uint64)


# (what torch.cuda.is_current_stream_capturing calls, looked up once)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing",
                     torch.cuda.is_current_stream_capturing)


class _Step:
    """What a step's layers share: the host copy of its metadata, its block
    table as contiguous int32, its lengths on the device as the host saw them
    (``lens``, None where the copy took the general path) and the plans made
    from them (``fast``).  A layer keeps the record it got, so another thread's
    step can neither take the plans away under it nor be given them.  ``names``:
    the layers that have run, where that is what tells one step from the next."""

    __slots__ = ("meta", "stamp", "host", "bt", "lens", "owner", "fast", "names")

    def __init__(self, meta, stamp, host, bt, lens, owner):
        self.meta, self.stamp, self.host, self.bt = meta, stamp, host, bt
        self.lens, self.owner, self.fast, self.names = lens, owner, {}, set()

    def serves(self, layer_name: str) -> bool:
        """Whether this may still be the step of ``layer_name``'s call, the metadata
        object and its stamp being the same: metadata that ``build_step_tables`` writes
        with no trace on the host is another step's when a layer comes again."""
        meta = self.meta
        if not written_unseen(meta.query_start_loc, meta.seq_lens, meta.block_table) or \
                _capturing():
            return True
        if not layer_name or layer_name in self.names:
            return False
        self.names.add(layer_name)
        return True

    def lens_on(self, stream: int, device: torch.device, given: torch.Tensor):
        """The lengths for launches on ``stream`` that read them on the device,
        or None.  Not the caller's tensor: that may be refilled for the next
        step while they are queued.  ``lens`` itself is written again by the
        next step of its thread on its stream, in order there; any other
        thread or stream gets a copy of the host's.  Under capture it is the
        caller's, whose contents at each replay are what a graph runs on."""
        if _capturing():
            return given
        if self.lens is None or self.owner == (threading.get_ident(), stream):
            return self.lens
        own = self.fast.get(("lens", stream))
        if own is None:
            words = np.asarray(self.host[1], dtype=np.int64)
            dev, _ = _upload([words], device)
            own = self.fast[("lens", stream)] = dev[:words.nbytes].view(torch.int64)
        return own


# The newest step.  vLLM hands every layer the same metadata object, so one
# device->host copy serves all layers of a step (the reference syncs three
# times per layer, ring_backend.py:604-605).  Holding the object keeps its
# identity from being reused by a later step's metadata.
_STEP: dict = {"step": None, "fast": {}}


def _version_of(t: torch.Tensor) -> int:
    try:
        return t._version
    except RuntimeError:  # inference-mode tensors keep no version counter
        return -1


def _meta_stamp(attn_metadata) -> tuple:
    """What identifies one step's metadata contents without reading them:
    the object, and the storage, shape and in-place version counter of each
    tensor the forward reads.  A caller that keeps one metadata object and
    refills its tensors in place between steps through torch's in-place ops
    bumps the version counters, so the next step does not reuse the previous
    step's host copy or plans; ``build_step_tables`` bumps its table's, and what it
    writes unseen is told by the layers (``_Step.serves``).  (vLLM builds a new
    metadata object every step; tensors made under inference mode keep no version
    counter, and a caller that refills such tensors in one reused object calls
    ``invalidate_step_cache`` between steps.)"""
    st = [id(attn_metadata)]
    for t in (attn_metadata.query_start_loc, attn_metadata.seq_lens, attn_metadata.block_table):
        st.extend((t.data_ptr(), tuple(t.shape), _version_of(t)))
    return tuple(st)


def invalidate_step_cache() -> None:
    """Drop the cached host copy of the step's metadata and the plans built
    from it: for a caller that rewrites the metadata tensors behind torch's
    back (a kernel writing into them directly) before reusing the object."""
    _STEP.update(step=None, fast={})


def _host_metadata(attn_metadata):
    """(query_start_loc, seq_lens, first block ids) as lists, and the block
    table as contiguous int32, for this step's metadata."""
    st = _step(attn_metadata)
    return st.host, st.bt


def _step(attn_metadata, queue=None, layer_name: str = "") -> _Step:
    """This step's record.  ``queue``: called, when the metadata is not on the
    host yet, between queueing its copy and waiting for it."""
    stamp = _meta_stamp(attn_metadata)
    st = _STEP["step"]
    if st is not None and st.meta is attn_metadata and st.stamp == stamp and \
            st.serves(layer_name):
        return st
    block_table = attn_metadata.block_table
    if block_table.dtype != torch.int32:
        block_table = block_table.to(torch.int32)
    block_table = block_table.contiguous()
    qsl_t = attn_metadata.query_start_loc
    sl_t = attn_metadata.seq_lens
    n = sl_t.shape[0]
    lens = owner = None
    if _fetchable(qsl_t, n + 1) and _fetchable(sl_t, n) and block_table.is_cuda \
            and block_table.shape[0] >= n:  # (the copy reads a first block per request)
        # (the lengths of this thread's step before are written over: its record
        # goes first, in case this one fails)
        _STEP.update(step=None, fast={})
        host, lens, owner = _fetch_metadata(qsl_t, sl_t, block_table, n, queue)
    else:
        fb = block_table[:, 0] if block_table.shape[1] > 0 else sl_t.new_zeros(n)
        packed = torch.cat([qsl_t.reshape(-1).to(torch.int64), sl_t.reshape(-1).to(torch.int64),
                            fb.reshape(-1).to(torch.int64)]).tolist()
        host = (packed[:n + 1], packed[n + 1:2 * n + 1], packed[2 * n + 1:])
    st = _Step(attn_metadata, stamp, host, block_table, lens, owner)
    st.names.add(layer_name)
    _STEP.update(step=st, fast=st.fast)
    return st


_INDEX_CODES = {torch.int32: _lib.DTYPE_I32, torch.int64: _lib.DTYPE_I64}
# per thread: the page-locked block (read before the call returns) and the
# words on the device
_fetch_buf = threading.local()


def _fetchable(t: torch.Tensor, n: int) -> bool:
    return t.is_cuda and t.dim() == 1 and t.shape[0] == n and t.dtype in _INDEX_CODES


def _fetch_metadata(qsl_t, sl_t, block_table, n: int, queue=None):
    """The step's metadata as host lists, its lengths on the device and whose
    they are (thread and stream), by one kernel that writes both (the former to
    page-locked memory) and one wait for that memory; what ``queue`` puts on
    the stream runs while the host waits and goes on."""
    dev, L = qsl_t.device, _lib.lib()
    with _lib.on_device(dev):
        stream = _lib.stream_ptr(dev)
        f = _fetch_buf
        if getattr(f, "key", None) != (dev, stream, n):
            # the lengths, for a launch queued ahead and for all others:
            # written by each step of this thread and stream, in order
            f.words = torch.empty(2 * n, dtype=torch.int64, device=dev)
            f.ahead, f.lens = f.words[:n], f.words[n:]
            f.key = (dev, stream, n)
            if getattr(f, "buf", None) is None or f.buf.shape[0] < 3 * n + 2:
                f.buf = torch.zeros(max(1024, 4 * n), dtype=torch.int64, pin_memory=True)
                f.np, f.token = f.buf.numpy(), 0
        f.token += 1
        rc = L.hcp_fetch_metadata(
            qsl_t.data_ptr(), _INDEX_CODES[qsl_t.dtype], qsl_t.stride(0),
            sl_t.data_ptr(), _INDEX_CODES[sl_t.dtype], sl_t.stride(0),
            block_table.data_ptr() if block_table.shape[1] > 0 else 0, _lib.DTYPE_I32,
            block_table.stride(0), n, 0 if queue is None else queue.max_len, f.words.data_ptr(),
            f.token, f.buf.data_ptr(), stream)
        _lib.check(rc, "hcp_fetch_metadata")
        try:
            if queue is not None:
                queue(f.ahead)
        finally:  # the buffer is not left to be written later
            _lib.check(L.hcp_wait_metadata(f.buf.data_ptr(), f.token, stream), "hcp_wait_metadata")
    packed = f.np[1:3 * n + 2].tolist()
    return ((packed[:n + 1], packed[n + 1:2 * n + 1], packed[2 * n + 1:]), f.lens,
            (threading.get_ident(), stream))


def _forward_attn_metadata(layer):
    """This step's attention metadata for ``layer`` from vLLM's forward
    context, or None (no vLLM, or no context)."""
    try:
        from vllm.forward_context import get_forward_context  # type: ignore

        raw = get_forward_context().attn_metadata
    except Exception:  # noqa: BLE001 -- no context: attribute nothing
        return None
    if isinstance(raw, dict):
        return raw.get(layer.layer_name)
    if isinstance(raw, list):
        return raw[0].get(layer.layer_name)
    return raw


# Pool-write evidence (ring_backend.py:254-267), validation only.  While
# enabled, do_kv_cache_update records the pool slots this worker wrote, and
# forward counts in "overlap" every slot of a request's peer (chunk-A) region
# among them: a memory-splitting worker never writes one.  "skipped" counts
# decode-ring tokens whose pool write was skipped (always counted).
WRITE_TRACK: dict = {"enabled": False, "slots": set(), "overlap": 0, "skipped": 0}


def reset_write_tracking() -> None:
    """Enable write tracking and clear its evidence (ring_backend.py:260-265)."""
    WRITE_TRACK["enabled"] = True
    WRITE_TRACK["slots"] = set()
    WRITE_TRACK["overlap"] = 0
    WRITE_TRACK["skipped"] = 0


enable_write_tracking = reset_write_tracking  # earlier name of the same call


def _probe_chunk_a_writes(block_row: torch.Tensor, peer_end: int, block_size: int) -> int:
    """Slots of the first ``peer_end`` positions of a request (its peer region,
    through its block-table row) that this worker wrote; added to
    ``WRITE_TRACK["overlap"]`` with a warning (ring_backend.py:790-810)."""
    nb_a = (peer_end + block_size - 1) // block_size
    blocks = block_row[:nb_a].tolist()
    slots = [b * block_size + o for b in blocks for o in range(block_size)][:peer_end]
    overlap = WRITE_TRACK["slots"].intersection(slots)
    if overlap:
        WRITE_TRACK["overlap"] += len(overlap)
        logger.warning("HCP ring: %d chunk-A pool slots were written locally "
                       "(expected 0 in a memory-splitting worker)", len(overlap))
    return len(overlap)


# ---------------------------------------------------------------------------
# Switches and evidence counters
# ---------------------------------------------------------------------------
BATCH_STATS: dict = {"max_reqs": 0}

IMPL_STATS: dict = {
    "attn_hip": 0,
    "merge_hip": 0,
    "decode_hip": 0,
    "ring_decode_steps": 0,
    "attn_triton": 0,
    "merge_triton": 0,
    "attn_torch": 0,
    "merge_torch": 0,
}

_FAST_IMPLS = ("hip", "triton")


def reset_impl_stats() -> None:
    for key in IMPL_STATS:
        IMPL_STATS[key] = 0
    for key in COPY_STATS:
        COPY_STATS[key] = 0


def reset_batch_stats() -> None:
    BATCH_STATS["max_reqs"] = 0


def _ring_enabled() -> bool:
    return os.environ.get("HCP_RING_ENABLED", "1") == "1"


def _split_tokens() -> int:
    return int(os.environ.get("HCP_RING_SPLIT_TOKENS", "0"))


def _ring_impl() -> str:
    return os.environ.get("HCP_RING_IMPL", "hip")


def _merge_impl() -> str:
    return os.environ.get("HCP_RING_MERGE", "hip")


def _require_fast(kind: str, value: str) -> None:
    if value not in _FAST_IMPLS:
        raise NotImplementedError(
            f"{kind}={value!r}: this build runs the HIP kernels only "
            f"(accepted: {', '.join(_FAST_IMPLS)}); there is no torch path"
        )


def _count(kind: str, n: int = 1) -> None:
    IMPL_STATS[f"{kind}_hip"] += n
    legacy = f"{kind}_triton"
    if legacy in IMPL_STATS:
        IMPL_STATS[legacy] += n


def _attn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    scale: float,
    q_pos0_in_kv: int | None,
    window: int | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention + LSE on the HIP kernel (ring_backend.py:309-336 contract),
    sliding window included (the reference sends windowed calls to its torch
    path, :323,336; here the kernel applies it).

    Returns (out ``[Tq, H, D]`` in q.dtype, lse ``[H, Tq]`` float32).
    """
    _require_fast("HCP_RING_IMPL", _ring_impl())
    o, lse = ring_attn_with_lse(q, k, v, scale, q_pos0_in_kv, window)
    _count("attn")
    return o, lse


def _merge(
    o_loc: torch.Tensor, lse_loc: torch.Tensor, o_peer: torch.Tensor, lse_peer: torch.Tensor
) -> torch.Tensor:
    """Local + peer LSE merge on the HIP kernel (ring_backend.py:339-360).

    Same argument order as the reference: ``merge_attn_states(out, o_peer,
    lse_peer, o_loc, lse_loc)`` with out in ``o_loc.dtype``.
    """
    _require_fast("HCP_RING_MERGE", _merge_impl())
    out = torch.empty_like(o_loc, memory_format=torch.contiguous_format)
    merge_attn_states(out, o_peer, lse_peer, o_loc, lse_loc)
    _count("merge")
    return out


# Most bytes of scratch that a prefill launch over a 4-bit cache expands keys into
# (more for a single request with more keys than fit).
_FP4_SCRATCH = 1 << 30


# ---------------------------------------------------------------------------
# Backend class (registered as CUSTOM)
# ---------------------------------------------------------------------------
class HcpRingAttentionBackend(_BackendBase):  # type: ignore[misc,valid-type]
    """Ring-attention backend: FlashAttention cache layout + metadata builder
    (inherited when vLLM is present), HIP attention impl with LSE peer merge.

    ``get_name()`` stays "CUSTOM": vLLM's Attention layer looks the backend up
    by that enum member (ring_backend.py:439-441).
    """

    forward_includes_kv_cache_update: bool = False

    @staticmethod
    def get_name() -> str:
        return "CUSTOM"

    @staticmethod
    def get_impl_cls() -> type["HcpRingAttentionImpl"]:
        return HcpRingAttentionImpl

    @staticmethod
    def get_builder_cls():
        return _BuilderCls


def _check_base(pc: PagedCache) -> None:
    """A layer's cache address, the one thing of its layout that a step's plan
    is not keyed on."""
    if pc.k_addr % 16 or pc.v_addr % 16:
        raise ValueError("k/v base addresses must be 16-byte aligned")


class _Ahead:
    """A decode layer queued before the host has seen the step's metadata:
    called by ``_step`` between queueing the metadata's copy and
    waiting for it (not at all when the host has it already).  The copy's
    kernel looks whether the batch is what the layer was queued for, with
    lengths within ``max_len``; if not, the layer writes nothing."""

    def __init__(self, impl, query, out, meta, pc):
        self.args = (impl, query, out, meta, pc)
        self.max_len = meta.block_table.shape[1] * pc.block_size
        self.dec = None

    def __call__(self, lens):
        impl, query, out, meta, pc = self.args
        if PagedDecode.takes(meta.block_table, lens, pc.block_size):
            self.dec = PagedDecode(pc, meta.block_table, lens, impl.num_heads,
                                   impl.sliding_window)
            self.dec.run(query, out, pc, impl.scale)


class _Plan:
    """Launch descriptors for one forward call."""

    def __init__(self):
        # causal entries over the paged cache: (q row, rows, request, first key,
        # keys, causal offset)
        self.local: list = []
        self.peer_rounds: list = []     # per round: {"contig": [...], "paged": [...]}
        self.any_peer = False
        self.decode: list = []  # single-token rows for the decode kernel: (q row, segments)
        self.decode_peer = False  # one of them has a peer segment
        self.ring: list = []  # decode-ring rows: (r, q row, tk, ring state, bt row, block 0)


class HcpRingAttentionImpl(_ImplBase):  # type: ignore[misc,valid-type]
    """HIP attention + LSE merge with peer chunk KV (ring_backend.py:452-834).

    Reads the paged cache in either vLLM 0.31 ``[nb, Hkv, bs, 2*D]`` or vLLM
    0.23 ``[nb, 2, bs, Hkv, D]`` layout, in place.  Peer KV is consumed from
    the staging dict (or from a split of the local cache) and never written.
    """

    def __init__(
        self,
        num_heads: int,
        head_size: int,
        scale: float,
        num_kv_heads: int | None = None,
        alibi_slopes: list[float] | None = None,
        sliding_window: int | None = None,
        kv_cache_dtype: str = "auto",
        logits_soft_cap: float | None = None,
        attn_type=AttentionType.DECODER,
        kv_sharing_target_layer_name: str | None = None,
        **kwargs,
    ) -> None:
        self.num_heads = num_heads
        self.head_size = head_size
        self.scale = float(scale)
        self.num_kv_heads = num_kv_heads if num_kv_heads is not None else num_heads
        self.kv_cache_dtype = kv_cache_dtype
        self.attn_type = attn_type
        self.kv_sharing_target_layer_name = kv_sharing_target_layer_name
        self.supports_quant_query_input = False
        if alibi_slopes is not None:
            raise NotImplementedError("HCP ring backend: ALiBi not supported")
        if logits_soft_cap:
            raise NotImplementedError("HCP ring backend: soft cap not supported")
        if sliding_window is not None and int(sliding_window) <= 0:
            raise ValueError("sliding_window must be a positive number of keys")
        if kv_cache_dtype not in ("auto", "float16", "bfloat16", "fp4"):
            raise NotImplementedError(f"kv_cache_dtype {kv_cache_dtype} not supported")
        if kv_cache_dtype == "fp4" and head_size % 32:
            raise NotImplementedError(
                f"HCP ring backend: head_size {head_size} not supported by the 4-bit cache "
                "(a multiple of 32 up to 256)")
        # the paged cache is read in place in 16-byte pieces (vLLM's flash
        # backends take the same head sizes)
        if head_size % 8 or not 0 < head_size <= 256:
            raise NotImplementedError(
                f"HCP ring backend: head_size {head_size} not supported (a multiple of 8 up to 256)")
        # applied to every causal pass (local segments), never to the
        # non-causal peer pass -- ring_backend.py:490-492,786,815,826-830
        self.sliding_window = int(sliding_window) if sliding_window is not None else None
        self.num_queries_per_kv = self.num_heads // self.num_kv_heads
        self._heads = (self.num_heads, self.num_kv_heads, self.head_size)

    # -- paged KV write (the step before the path) ----------------------------
    def do_kv_cache_update(
        self,
        layer,
        key: torch.Tensor,
        value: torch.Tensor,
        kv_cache: torch.Tensor,
        slot_mapping: torch.Tensor,
    ) -> None:
        """Write this step's K/V into the paged cache at ``slot_mapping``.

        ring_backend.py:501-539 on the HIP cache-write kernel: slot = block *
        bs + offset, either cache layout.  The single-token decode steps of
        decode-ring requests are not written (their KV is decode growth,
        routed by the ring): those rows get slot -1, which the kernel skips,
        instead of three gather copies.
        """
        if self.attn_type in (AttentionType.ENCODER_ONLY, AttentionType.ENCODER):
            return
        skip = self._decode_ring_skip_positions(layer, slot_mapping)
        if skip:
            WRITE_TRACK["skipped"] += len(skip)
            slot_mapping = slot_mapping.clone()
            idx = torch.tensor(sorted(skip), dtype=torch.long, device=slot_mapping.device)
            slot_mapping.index_fill_(0, idx, -1)
        reshape_and_cache(key, value, kv_cache, slot_mapping)
        if WRITE_TRACK["enabled"]:
            WRITE_TRACK["slots"].update(s for s in slot_mapping.tolist() if s >= 0)

    def _decode_ring_skip_positions(self, layer, slot_mapping: torch.Tensor) -> set[int]:
        """Rows of this step's slot_mapping that are decode-ring requests'
        single-token decode steps (ring_backend.py:541-574); empty when the
        step's metadata is unavailable (never skip what cannot be attributed)."""
        if not (_decode_ring_enabled() and DECODE_RING_MAP):
            return set()
        meta = _forward_attn_metadata(layer)
        if meta is None:
            return set()
        qsl = meta.query_start_loc.tolist()
        first = meta.block_table[:, 0].tolist() if meta.block_table.shape[1] else []
        return {qsl[r] for r in range(len(qsl) - 1)
                if qsl[r + 1] - qsl[r] == 1 and int(first[r]) in DECODE_RING_MAP
                and qsl[r] < slot_mapping.shape[0]}

    # -- planning -------------------------------------------------------------
    def _peer_for_request(self, first_block: int, layer_name: str, n_reqs: int,
                          probe: bool = False):
        """Ordered staged (k, v) chunks of a request, or None (ring_backend.py:738-772).
        ``probe``: only look (no warning, no stream ordering)."""
        ck_list = PEER_REQ_MAP.get(first_block)
        if ck_list is None and n_reqs == 1:
            chunks = {key[0] for key in PEER_KV_STAGING}
            if len(chunks) == 1:
                ck_list = [next(iter(chunks))]
        if not ck_list:
            return None
        parts = []
        for ck in ck_list:
            kv = PEER_KV_STAGING.get((ck, layer_name))
            if kv is None:
                if not probe:
                    logger.warning(
                        "HCP ring: request mapped to chunks %s but staging incomplete at "
                        "layer %s; falling back to local path", ck_list, layer_name)
                return None
            parts.append(kv)
        if not probe:
            for ck, kv in zip(ck_list, parts):
                _wait_staged((ck, layer_name), kv)
        return parts

    def _write_probe(self, layer_name, qsl, seq_lens, block_table, first_blocks, pc,
                     ring_on: bool, split: int) -> None:
        """With write tracking on: every request that takes the ring path
        (a peer region of ``peer_end > 0`` positions, from staged chunks or the
        split env; decode-ring rows excepted) has its peer region's pool slots
        checked against the slots this worker wrote (ring_backend.py:790-810)."""
        ring_rows = _decode_ring_enabled() and bool(DECODE_RING_MAP)
        n = len(seq_lens)
        for r in range(n):
            tq, tk = qsl[r + 1] - qsl[r], int(seq_lens[r])
            if tq == 0 or (ring_rows and tq == 1 and first_blocks[r] in DECODE_RING_MAP):
                continue
            staged = (self._peer_for_request(first_blocks[r], layer_name, n, probe=True)
                      if ring_on else None)
            if staged is not None:
                peer_end = min(sum(int(kv[0].shape[0]) for kv in staged), tk)
            else:
                peer_end = min(split, tk) if split > 0 else 0
            if peer_end > 0:
                _probe_chunk_a_writes(block_table[r], peer_end, pc.block_size)

    def _decode_rows_apart(self, qsl, seq_lens, each_layer: bool = False) -> bool:
        """Whether a mixed batch's single-token rows leave the prefill launch
        for a decode launch of their own.  In the prefill launch such a row is
        a 128-row block per query head, one of whose four waves has a row, each
        reading its KV head's keys (the window's) again: 0.27, 0.49 or 0.88 us of
        a CU per 64 keys and head at 64, 128 or 256 columns.  The decode launch
        reads the keys once, but is two more kernels; where a plan is made once
        per step it pays past 20 us of the machine, where each layer makes its
        own (``each_layer``: staged or split peers) past 60 us and 6 us a row.

        256 new tokens next to the rows, us per layer in one launch / apart:
        28 / 4 x 128, 16 x 1536 keys (20 us by this count) 73 / 79, 8 x 4096 (27)
        87 / 79, 32 x 4096 (109) 224 / 96; 14 / 2 x 64, 32 x 4096 (30) 99 / 79;
        16 / 8 x 256, 2 x 8192 (14) 98 / 90.  With 1024 staged keys each, 28 / 4 x
        128, 2 x 24576 (42) 145 / 164, 2 x 49152 (83) 201 / 171; 8 x 12000 (86) 221 /
        240, 8 x 16384 (115) 268 / 249; 32 x 8192 (244) 497 / 503, 32 x 16384 (462)
        849 / 519.

        Over a 4-bit cache the rows' keys are expanded too where they stay, and the
        same 20 us are about where both take as long at 64 and 128 columns, but late at
        256: 28 / 4 x 128, 16 x 512 (7) 83 / 96, 16 x 1536 (21) 94 / 93, 8 x 4096 (27) 110 /
        93, 32 x 4096 (110) 315 / 96; 14 / 2 x 64, 8 x 1024 (2) 74 / 93, 32 x 4096 (30) 120
        / 93; 16 / 8 x 256, 2 x 2048 (4) 91 / 93, 2 x 8192 (14) 131 / 95."""
        w = self.sliding_window
        keys = [tk if w is None else min(tk, w)
                for r, tk in enumerate(seq_lens) if qsl[r + 1] - qsl[r] == 1]
        tile_us = {64: 0.27, 128: 0.49, 256: 0.88}[
            next(c for c in (64, 128, 256) if self.head_size <= c)]
        est = sum(-(-tk // 64) for tk in keys) * self.num_heads * tile_us / 256
        return est > (60 + 6 * len(keys) if each_layer else 20)

    def _plan(self, layer_name, qsl, seq_lens, block_table, first_blocks, pc, split):
        plan = _Plan()
        n = len(seq_lens)
        # (Over a 4-bit cache they stay: the decode launch of these rows takes segments,
        # which that has not.  The prefill launch expands their keys as it does the
        # others': 256 new tokens behind 1024 staged ones next to 16 rows of 1536 keys at
        # 28 / 4 x 128 159 us a layer, next to 32 of 4096 382, of 16384 1228; over a 16-bit
        # cache 144, 282 and 377.)
        apart = qsl != list(range(n + 1)) and pc.layout != "fp4" and \
            self._decode_rows_apart(qsl, seq_lens, True)
        ring_on = _decode_ring_enabled() and bool(DECODE_RING_MAP)
        for r in range(len(seq_lens)):
            qs, qe = qsl[r], qsl[r + 1]
            tq, tk = qe - qs, seq_lens[r]
            if tq == 0:
                continue
            if ring_on and tq == 1:
                dr = DECODE_RING_MAP.get(first_blocks[r])
                if dr is not None:
                    plan.ring.append((r, qs, tk, dr, block_table[r], first_blocks[r]))
                    continue
            qpos0 = tk - tq
            staged = None
            if _ring_enabled():
                staged = self._peer_for_request(first_blocks[r], layer_name, len(seq_lens))
            peer_segs = []
            if staged is not None:
                total = sum(int(kv[0].shape[0]) for kv in staged)
                peer_end = min(total, tk)
                for kk, vv in staged:
                    if kk.shape[0] > 0:
                        peer_segs.append(segment_contiguous(kk, vv))
            elif split > 0:
                peer_end = min(split, tk)
                peer_segs.append(segment_paged(pc, block_table[r], 0, peer_end))
            else:
                peer_end = 0
            if apart and tq == 1:
                # one query at position tk - 1: inside the prefix it sees the
                # whole local range, past it the local keys (the last `w` of
                # them) and every staged chunk
                lo = peer_end if peer_end < tk else 0
                segs = [segment_paged(pc, block_table[r], lo, tk - lo)]
                segs = window_tail(segs, self.sliding_window)
                if 0 < peer_end < tk and peer_segs:
                    segs += peer_segs
                    plan.decode_peer = True
                plan.decode.append((qs, segs))
                continue
            if peer_end == 0:
                plan.local.append((qs, tq, r, 0, tk, qpos0))
                continue
            n_a = max(0, min(tq, peer_end - qpos0))
            if n_a > 0:
                plan.local.append((qs, n_a, r, 0, tk, qpos0))
            if n_a < tq:
                qb0, nb = qs + n_a, tq - n_a
                plan.local.append((qb0, nb, r, peer_end, tk - peer_end, qpos0 + n_a - peer_end))
                for i, seg in enumerate(peer_segs):
                    while len(plan.peer_rounds) <= i:
                        plan.peer_rounds.append({"contig": [], "paged": []})
                    kind = "paged" if seg.block_table else "contig"
                    plan.peer_rounds[i][kind].append(make_entry(qb0, nb, seg, 0))
                    plan.any_peer = True
        return plan

    # -- forward ----------------------------------------------------------------
    def forward(
        self,
        layer,
        query: torch.Tensor,
        key: torch.Tensor,
        value: torch.Tensor,
        kv_cache: torch.Tensor,
        attn_metadata,
        output: torch.Tensor,
        output_scale: torch.Tensor | None = None,
        output_block_scale: torch.Tensor | None = None,
    ) -> torch.Tensor:
        if output_scale is not None or output_block_scale is not None:
            raise NotImplementedError("fused output quant not supported")
        if attn_metadata is None:  # profiling run
            if output.is_cuda and not _capturing():
                # the partials of a cut launch and a 4-bit cache's expanded keys, so
                # that the engine's peak has them
                _lib.scratch(_lib.split_limits(self.head_size).max_workspace +
                             (_FP4_SCRATCH if self.kv_cache_dtype == "fp4" else 0), output.device)
            return output.fill_(0)
        if self.attn_type != AttentionType.DECODER:
            raise NotImplementedError("HCP ring backend supports decoder attention only")
        _require_fast("HCP_RING_IMPL", _ring_impl())
        _require_fast("HCP_RING_MERGE", _merge_impl())

        num_actual = attn_metadata.num_actual_tokens
        query = query[:num_actual]
        out = output[:num_actual]
        pc = PagedCache.from_tensor(kv_cache)
        if pc.num_kv_heads != self.num_kv_heads or pc.head_dim != self.head_size:
            raise ValueError("kv_cache shape does not match the layer's heads/head_size")
        if (pc.layout == "fp4") != (self.kv_cache_dtype == "fp4"):
            raise ValueError(f"a {kv_cache.dtype} cache for kv_cache_dtype {self.kv_cache_dtype!r}")
        ring_on = _ring_enabled()
        split = _split_tokens() if ring_on else 0
        # One token per request and nothing that gives a request peers: a
        # decode batch whose lengths and blocks the kernels read themselves.
        # Its first layer is queued before the host has seen the metadata; a
        # batch that turns out otherwise runs again as what it is.
        ahead = None
        if num_actual == attn_metadata.seq_lens.shape[0] and split == 0 and \
                not (ring_on and PEER_KV_STAGING) and \
                not (DECODE_RING_MAP and _decode_ring_enabled()):
            ahead = _Ahead(self, query, out, attn_metadata, pc)
        # small metadata tensors: one host sync per step (see _step)
        layer_name = getattr(layer, "layer_name", "")
        step = _step(attn_metadata, ahead, layer_name)
        (qsl, seq_lens, first_blocks), block_table = step.host, step.bt
        BATCH_STATS["max_reqs"] = max(BATCH_STATS["max_reqs"], len(seq_lens))
        n = len(seq_lens)
        if len(first_blocks) < n and qsl[n] > qsl[len(first_blocks)]:
            raise ValueError("the block table has no row for a request")
        if self._peer_free(ring_on, split, first_blocks, n):
            self._forward_local_only(query, out, step, pc, attn_metadata.seq_lens, ahead)
            return output
        if WRITE_TRACK["enabled"]:
            self._write_probe(layer_name, qsl, seq_lens, block_table, first_blocks, pc,
                              ring_on, split)

        is_decode = n > 0 and qsl == list(range(n + 1))
        if pc.layout == "fp4":
            if split > 0:
                raise NotImplementedError("HCP_RING_SPLIT_TOKENS needs a 16-bit cache")
            if _decode_ring_enabled() and any(fb in DECODE_RING_MAP for fb in first_blocks):
                raise NotImplementedError("the decode ring needs a 16-bit cache")
            if is_decode:
                self._forward_decode_fp4(query, out, step, pc, layer_name)
                return output
        if is_decode and self._forward_decode_staged(query, out, step, pc, layer_name, ring_on,
                                                     split):
            return output
        plan = self._plan(layer_name, qsl, seq_lens, block_table, first_blocks, pc, split)
        ring_local = self._ring_local_segments(plan, pc, key, value, layer_name)
        if is_decode:
            lse = self._forward_decode(query, out, plan, block_table, pc, n, ring_local)
            parts = {r: (out[qs:qs + 1], lse[:, qs:qs + 1]) for (r, qs, *_r) in plan.ring}
        else:
            if plan.local or plan.any_peer:
                self._forward_prefill(query, out, plan, step, pc)
            if plan.decode:
                # NaN scores as the prefill launches leave them: in the row, or,
                # where these merge with peers, a side without weight
                keep_nan = not (plan.any_peer or plan.decode_peer)
                DecodeBatch([segs for _, segs in plan.decode], self.num_heads, self.num_kv_heads,
                            self.head_size, query.device,
                            rows=[qs for qs, _ in plan.decode]).run(
                    query, out, None, self.scale, keep_nan=keep_nan)
                _count("decode")
            parts = {}
            for (r, qs, *_r) in plan.ring:
                parts[r] = self._local_partial(query[qs:qs + 1], ring_local[r])
        for (r, qs, tk, dr, *_r) in plan.ring:
            o_acc, lse_acc = parts[r]
            out[qs:qs + 1] = self._ring_step(dr, layer_name, query[qs:qs + 1],
                                             o_acc, lse_acc)
        return output

    # -- memory-split decode (owner side) ----------------------------------------
    def _ring_local_segments(self, plan: _Plan, pc: PagedCache, key, value, layer_name):
        """Owner-side local segments of each decode-ring row: own chunk in the
        pool, the owner's growth share, the current token (ring_backend.py:
        643-671), with the growth bookkeeping of :652-689 done here (the
        current token joins the owner's growth or waits to be shipped)."""
        segs = {}
        for (r, qs, tk, dr, row, fb) in plan.ring:
            _release_staged_for_request(fb)
            plen = dr["prefix_len"]
            if dr["own_chunk_len"] is None:
                dr["own_chunk_len"] = tk - 1 - plen
            own_len = dr["own_chunk_len"]
            pos = tk - 1
            assignee = growth_assignee(pos, dr["ring_size"], dr["growth_policy"])
            dr["ship"] = dr["pending_growth"].pop(layer_name, None)
            k_cur = key[qs:qs + 1].contiguous()
            v_cur = value[qs:qs + 1].contiguous()
            g = dr["growth"].get(layer_name)
            if g is None:
                g = dr["growth"][layer_name] = GrowthBuffer(
                    self.num_kv_heads, self.head_size, k_cur.dtype, k_cur.device)
            own = segment_paged(pc, row, plen, own_len) if own_len > 0 else None
            if assignee == dr["own_index"]:
                g.append(k_cur, v_cur)
                local = [own, g.segment()]
            else:
                local = [own, g.segment(), segment_contiguous(k_cur, v_cur)]
                dr["pending_growth"][layer_name] = (assignee, k_cur, v_cur)
            # causal at len - 1 over the concatenation (:672-679): every key,
            # or the last `sliding_window` of them
            segs[r] = window_tail(local, self.sliding_window)
        return segs

    def _local_partial(self, q_r, segs):
        o, lse = local_partial(q_r, segs, self.num_kv_heads, self.scale)
        _count("decode")
        return o, lse

    def _ring_step(self, dr, layer_name, q_r, o_acc, lse_acc):
        """Send the owner's accumulator around the ring (ring_backend.py:
        690-722); the returned (O, LSE) is the exact attention of the step."""
        transport = dr.get("transport")
        if transport is None:
            raise RuntimeError("HCP decode ring requires a ring transport "
                               "(register_decode_ring(..., transport=...))")
        ship = dr.pop("ship", None)
        gk = gv = None
        target = -1
        if ship is not None:
            gk, gv = ship[1], ship[2]
            target = ship[0] + 1   # growth index 0..N-2 -> transport index 1..N-1
        first_chunk = dr["peer_chunks"][0][0] if dr["peer_chunks"] else ""
        o, _lse = ring_decode_step(transport, q_r, o_acc, lse_acc, self.scale, layer_name,
                                   first_chunk, req=dr["req_tag"], growth_k=gk,
                                   growth_v=gv, growth_target=target)
        IMPL_STATS["ring_decode_steps"] += 1
        return o

    # -- batches with no peer KV and no decode-ring rows -------------------------
    @staticmethod
    def _peer_free(ring_on: bool, split: int, first_blocks, n: int) -> bool:
        """No request of the batch takes a peer segment or the decode ring:
        the plain causal pass over the paged cache (ring_backend.py:783-789)."""
        if DECODE_RING_MAP and _decode_ring_enabled() and \
                any(fb in DECODE_RING_MAP for fb in first_blocks):
            return False
        if not ring_on:
            return True
        if split > 0:
            return False
        if not PEER_KV_STAGING:
            return True
        return n > 1 and not any(fb in PEER_REQ_MAP for fb in first_blocks)

    # -- pure decode batches with staged peers ------------------------------------
    def _decode_staged_template(self, seq_lens, block_table, first_blocks, pc, layer_name):
        """The step's decode entries with every field that does not change
        from layer to layer (lengths, block-table rows, strides of the cache;
        paged addresses relative to the layer's cache), and which staged chunk
        each contiguous one reads; False if some request's staging is
        incomplete (the general path then decides, per layer, as the reference
        does)."""
        n = len(seq_lens)
        w = self.sliding_window
        ring_on = _ring_enabled()
        lone = None  # the single-request fallback of _peer_for_request
        if n == 1 and ring_on:
            chunks = {key[0] for key in PEER_KV_STAGING}
            lone = list(chunks) if len(chunks) == 1 else None
        seq, kinds, starts, lens, peers = [], [], [], [], []
        for r, (tk, fb) in enumerate(zip(seq_lens, first_blocks)):
            peer_end, ck_list, chunk_lens = 0, None, ()
            if ring_on:
                ck_list = PEER_REQ_MAP.get(fb)
                if ck_list is None:
                    ck_list = lone
                if ck_list:
                    kvs = [PEER_KV_STAGING.get((ck, layer_name)) for ck in ck_list]
                    if any(kv is None for kv in kvs):
                        return False  # staging still arriving: decided per layer
                    chunk_lens = [kv[0].shape[0] for kv in kvs]
                    peer_end = min(sum(chunk_lens), tk)
            # one query at position tk - 1 (ring_backend.py:626-627): inside the
            # prefix it sees the whole local range (:811-817), else the local
            # keys past the prefix plus every staged chunk (:820-830)
            lo = 0 if peer_end == 0 or peer_end >= tk else peer_end
            if w is not None:  # the causal pass sees the last `w` local keys
                lo = max(lo, tk - w)
            seq.append(r)
            kinds.append(0)
            starts.append(lo)
            lens.append(tk - lo)
            if 0 < peer_end < tk:
                for ck, cl in zip(ck_list, chunk_lens):
                    if cl > 0:
                        peers.append((ck, cl))
                        seq.append(r)
                        kinds.append(1)
                        starts.append(0)
                        lens.append(cl)
        kinds = np.asarray(kinds)
        seq = np.asarray(seq, dtype=np.int32)
        loc = np.nonzero(kinds == 0)[0]
        tmpl = np.zeros(len(seq), dtype=ENTRY_DTYPE)
        tmpl["q_start"] = seq
        tmpl["q_len"] = 1
        tmpl["len"] = lens
        tmpl[loc] = paged_entry_array(pc, block_table, seq[loc], seq[loc], 1, 0,
                                      np.asarray(starts)[loc], tmpl["len"][loc], relative=True)
        return {"tmpl": tmpl, "seq": seq, "at": np.nonzero(kinds == 1)[0], "peers": peers,
                "batch": None}

    def _forward_decode_staged(self, query, out, step, pc, layer_name, ring_on, split) -> bool:
        """A pure decode batch without decode-ring rows: one split-KV launch
        over every request's local paged segment and staged peer chunks, its
        split plan built once per step and reused by every layer, each layer
        writing only its staged chunks' addresses into the records and
        uploading them in one small copy (the cache's address is a launch
        argument).  False when the general path must run (split env,
        decode-ring rows, staging that differs from the step's template)."""
        (_qsl, seq_lens, first_blocks), block_table = step.host, step.bt
        if split > 0 or (_decode_ring_enabled() and DECODE_RING_MAP
                         and any(fb in DECODE_RING_MAP for fb in first_blocks)):
            return False
        # (the staging generation: a chunk staged, dropped or mapped after the
        # template was built -- even for a request the template saw without
        # peers -- makes the next layer build a new one; the stream: the plan's
        # upload is ordered on the one it was made on)
        key = (*self._layout_key("dec_staged", pc), ring_on, _STAGE_GEN[0],
               _lib.stream_ptr(query.device))
        st = step.fast.get(key)
        if st is None:
            st = self._decode_staged_template(seq_lens, block_table, first_blocks, pc, layer_name)
            step.fast[key] = st
        if st is False:
            return False
        _check_base(pc)
        kvs = []
        cur = torch.cuda.current_stream(query.device)
        for ck, nt in st["peers"]:
            kv = PEER_KV_STAGING.get((ck, layer_name))
            if kv is None or kv[0].shape[0] != nt:
                return False
            _wait_staged((ck, layer_name), kv, cur)
            kvs.append(kv)
        words = _chunk_words(kvs) if kvs else None
        batch = st["batch"]
        if batch is None:
            ent, at = st["tmpl"].copy(), st["at"]
            if kvs:
                for i, f in enumerate(("k_addr", "v_addr", "stride_tok", "stride_head")):
                    ent[f][at] = words[:, i]
            batch = st["batch"] = DecodeBatch.from_entries(
                ent, self.num_heads, self.num_kv_heads, self.head_size, query.device,
                keep=block_table, entry_seq=st["seq"], num_seqs=len(seq_lens))
        elif kvs:
            batch = batch.rebind_chunks(words, (block_table, kvs))
        batch.run(query, out, None, self.scale, kv_base=pc.k_addr)
        _count("decode")
        return True

    def _layout_key(self, kind: str, pc) -> tuple:
        """What a step's plan of this kind depends on besides the metadata."""
        return (kind, self.sliding_window, pc.layout, pc.stride_tok, pc.stride_head,
                pc.stride_block, pc.block_size, pc.num_blocks, pc.v_addr - pc.k_addr, self._heads)

    def _forward_local_only(self, query, out, step, pc, lens_t, ahead):
        """Causal attention of every request over its paged KV: for a pure
        decode batch ``PagedDecode``, which needs no plan (``ahead``: already
        queued for this layer), or, past its limits, a planned split-KV decode;
        else one varlen launch (and a decode launch for the single-token rows).
        Planned and uploaded once per step, cache layout and stream; a layer's
        launch adds its cache's address."""
        (qsl, seq_lens, _first), block_table, fast = step.host, step.bt, step.fast
        n = len(seq_lens)
        if n == 0:
            return
        stream = _lib.stream_ptr(query.device)
        lens = step.lens_on(stream, query.device, lens_t)
        on = (stream, 0 if lens is None else lens.data_ptr())
        if qsl == list(range(n + 1)):
            key = (*self._layout_key("paged", pc), on)
            dec = fast.get(key)
            if dec is None:
                dec = fast[key] = self._plan_paged(seq_lens, block_table, pc, lens, ahead)
            if dec:
                if ahead is None or ahead.dec is None:
                    _check_base(pc)
                    dec.run(query, out, pc, self.scale)
                _count("decode")
                return
        # The single-token rows first: they seldom need a plan, and the
        # prefill's is made while they run.  In the prefill launch a NaN score
        # makes its row NaN (a decode batch leaves the split out): here too.
        key = (*self._layout_key("rows", pc), on)
        dec = fast.get(key, fast)  # (fast itself: not planned yet)
        if dec is fast:
            dec = fast[key] = self._plan_rows(query, qsl, seq_lens, block_table, pc, lens)
        _check_base(pc)
        if dec is not None:
            if isinstance(dec, list):  # a 4-bit cache's
                self._run_fp4_rows(dec, query, out, pc, keep_nan=qsl != list(range(n + 1)))
            elif isinstance(dec, tuple):  # a run of rows, unplanned
                a, b, rows = dec
                rows.run(query[a:b], out[a:b], pc, self.scale, keep_nan=True)
            else:
                dec.run(query, out, None, self.scale, kv_base=pc.k_addr,
                        keep_nan=qsl != list(range(n + 1)))
            _count("decode")
        key = (*self._layout_key("chunks", pc), stream)
        pre = fast.get(key, fast)
        if pre is fast:
            pre = fast[key] = self._plan_chunks(query, qsl, seq_lens, block_table, pc)
        if pre is not None:
            self._run_chunks(pre, query, out, block_table, pc)
            _count("attn")

    def _plan_paged(self, seq_lens, block_table, pc, lens, ahead):
        """A pure decode batch without a plan, or False past its limits.
        Lengths that the block table cannot name are refused."""
        if lens is None or not PagedDecode.takes(block_table, lens, pc.block_size):
            return False
        if min(seq_lens) < 0:
            raise ValueError("negative segment start/length")
        if max(seq_lens) > block_table.shape[1] * pc.block_size:
            raise ValueError("segment extends past the block-table row")
        if ahead is not None and ahead.dec is not None and ahead.args[3].block_table is block_table:
            return ahead.dec
        return PagedDecode(pc, block_table, lens, self.num_heads, self.sliding_window)

    def _rows_apart(self, qsl, seq_lens):
        """(query starts, new tokens, keys of each request, which of them are
        single-token rows for the decode launch) of a batch without peers."""
        tq = np.diff(np.asarray(qsl, dtype=np.int64))
        dec = tq == 1
        if qsl != list(range(len(qsl))) and not self._decode_rows_apart(qsl, seq_lens):
            dec[:] = False
        return (np.asarray(qsl[:-1], dtype=np.int64), tq,
                np.asarray(seq_lens, dtype=np.int64), dec)

    def _plan_chunks(self, query, qsl, seq_lens, block_table, pc):
        """The prefill launch (or None) of a batch without peers, with
        addresses relative to the layer's cache; over blocks under 16 tokens
        its entries instead."""
        qs, tq, tk, dec = self._rows_apart(qsl, seq_lens)
        pre = np.nonzero((tq > 0) & ~dec)[0]
        if len(pre) == 0:
            return None
        return self._chunk_launch(
            paged_entry_array(pc, block_table, pre, qs[pre], tq[pre], (tk - tq)[pre], 0, tk[pre],
                              relative=True), query, block_table, pc)

    def _chunk_launch(self, ent, query, block_table, pc):
        """The causal launch of entries with addresses relative to a layer's
        cache; over blocks under 16 tokens, which are gathered from absolute
        addresses, the entries; over a 4-bit cache a list of launches, each with
        keys that fit the scratch they are expanded into."""
        if pc.layout == "fp4":
            w = self.sliding_window
            if w is not None:  # keys before every query's window are not expanded
                skip = np.clip(ent["causal_offset"] - w + 1, 0, ent["len"])
                ent["start"] += skip
                ent["len"] -= skip
                ent["causal_offset"] -= skip
            most = _FP4_SCRATCH // (4 * self.num_kv_heads * self.head_size)
            launches, first, keys = [], 0, 0
            for i, n in enumerate([*ent["len"].tolist(), most + 1]):
                if keys + n > most and i > first:
                    launches.append(VarlenLaunch(ent[first:i], True, True, query.device,
                                                 keep=block_table, heads=self._heads,
                                                 window=self.sliding_window, fp4=pc))
                    first, keys = i, 0
                keys += n
            return launches
        if pc.block_size < _MIN_PAGED_BLOCK:
            return ent
        return VarlenLaunch(ent, True, True, query.device, keep=block_table, heads=self._heads,
                            window=self.sliding_window)

    def _run_chunks(self, pre, query, out, block_table, pc, acc=None):
        """A layer's run of what ``_chunk_launch`` made, merged with ``acc`` as
        its prefix."""
        if isinstance(pre, list):
            for launch in pre:
                launch.run(query, out, None, self.num_kv_heads, self.scale, self.sliding_window,
                           acc=acc, kv_base=pc.k_addr)
            return
        if isinstance(pre, np.ndarray):
            ent = pre.copy()
            ent["k_addr"] = pc.k_addr
            ent["v_addr"] = pc.v_addr
            pre, base = VarlenLaunch(ent, True, True, query.device, keep=(pc.cache, block_table),
                                     heads=self._heads, window=self.sliding_window), 0
        else:
            base = pc.k_addr
        pre.run(query, out, None, self.num_kv_heads, self.scale, self.sliding_window, acc=acc,
                kv_base=base)

    def _plan_rows(self, query, qsl, seq_lens, block_table, pc, lens):
        """The launch of a batch's single-token rows: (first, end, launch) of a
        run of query rows without a plan where they are neighbouring requests,
        as a scheduler lists them, else a planned one; None without such rows.
        A length past the block table is refused, in a prefill chunk too, before
        anything of the layer is queued."""
        qs, tq, tk, dec = self._rows_apart(qsl, seq_lens)
        limit = block_table.shape[1] * pc.block_size
        used = tk[tq > 0]
        if len(used) and used.min() < 0:
            raise ValueError("negative segment start/length")
        if len(used) and used.max() > limit:
            raise ValueError("segment extends past the block-table row")
        rows = np.nonzero(dec)[0]
        if len(rows) == 0:
            return None
        w = self.sliding_window
        a, b = int(rows[0]), int(rows[-1]) + 1
        if b - a == len(rows) and lens is not None and \
                PagedDecode.takes(block_table[a:b], lens[a:b], pc.block_size):
            return (int(qs[a]), int(qs[a]) + b - a,
                    PagedDecode(pc, block_table[a:b], lens[a:b], self.num_heads, w))
        if pc.layout == "fp4":
            return self._plan_fp4_rows(query, rows, qs[rows], tk[rows], block_table, pc)
        # one query at the end of its keys: all of them visible, or the last `w`
        # of them (ring_backend.py:397-398)
        start = np.zeros(len(rows), np.int64) if w is None else np.maximum(tk[rows] - w, 0)
        return DecodeBatch.from_entries(
            paged_entry_array(pc, block_table, rows, qs[rows], 1, 0, start, tk[rows] - start,
                              relative=True),
            self.num_heads, self.num_kv_heads, self.head_size, query.device, keep=block_table,
            rows=None if qsl == list(range(len(qsl))) else qs[rows])

    # -- a 4-bit cache's single-token rows ---------------------------------------
    def _plan_fp4_rows(self, query, rows, qs, keys, block_table, pc, starts=None):
        """Launches of the batch's requests ``rows`` (query rows ``qs``, ``keys``
        keys each, the first seen ``starts``): [(first, end of a run of query rows,
        or their indices and None, launch)], each of as many as one takes."""
        # (a launch's keys are counted in 32-key chunks, in 32 bits)
        named = max(1, block_table.shape[1] * pc.block_size)
        most = max(1, min(_lib.DECODE_PAGED_MAX_SEQS, (1 << 34) // named))
        words = [np.ascontiguousarray(x, dtype=np.int64) for x in (rows, qs, keys, starts)
                 if x is not None]
        dev, _ = _upload(words, query.device)
        at, cols = 0, []
        for x in words:
            cols.append(dev[at:at + x.nbytes].view(torch.int64))
            at += (x.nbytes + 255) & ~255
        plans = []
        for a in range(0, len(rows), most):
            b = min(len(rows), a + most)
            run = qs[b - 1] - qs[a] == b - 1 - a and rows[b - 1] - rows[a] == b - 1 - a
            table = block_table[rows[a]:rows[a] + b - a] if run else block_table[cols[0][a:b]]
            dec = PagedDecode(pc, table, cols[2][a:b], self.num_heads, self.sliding_window,
                              None if starts is None else cols[3][a:b])
            plans.append((int(qs[a]), int(qs[a]) + b - a, dec) if run else (cols[1][a:b], None, dec))
        return plans

    def _run_fp4_rows(self, plans, query, out, pc, keep_nan: bool, lse=None) -> None:
        """``lse``: of query rows, all of them in one run."""
        for a, b, dec in plans:
            if b is None:
                part = torch.empty((a.shape[0], *out.shape[1:]), dtype=out.dtype, device=out.device)
                dec.run(query[a], part, pc, self.scale, keep_nan)
                out[a] = part
            else:
                dec.run(query[a:b], out[a:b], pc, self.scale, keep_nan,
                        None if lse is None else lse[:, a:b])

    def _forward_decode_fp4(self, query, out, step, pc, layer_name) -> None:
        """A pure decode batch with staged peers over a 4-bit cache: the local
        keys past each prefix (or, inside it, all of them: ring_backend.py:811-830)
        in the 4-bit decode, then the peers, which take that result as their
        running accumulator.  It is of the model's type there, as the decode ring's
        accumulator and the prefill's peer results are: half a step of the local
        result, weighed by its share, next to the half step that the output takes.

        us a layer (over a 16-bit cache, in one launch): 16 rows of 8192 keys, 4096 of
        them staged, at 28 / 4 x 128 172 (98); 64 of 34000, 32768 staged, 780 (744)."""
        (_qsl, seq_lens, first_blocks), block_table = step.host, step.bt
        _check_base(pc)
        n = len(seq_lens)
        staged = [self._peer_for_request(fb, layer_name, n) if _ring_enabled() else None
                  for fb in first_blocks]
        ends = [min(sum(int(kv[0].shape[0]) for kv in s), tk) if s else 0
                for s, tk in zip(staged, seq_lens)]
        starts = [0 if end >= tk else end for end, tk in zip(ends, seq_lens)]
        kvs, of = [], []  # chunks that some query sees, and whose
        for r, (chunks, start) in enumerate(zip(staged, starts)):
            if start:
                kvs += [kv for kv in chunks if kv[0].shape[0] > 0]
                of += [r] * (len(kvs) - len(of))
        lens = [int(k.shape[0]) for k, _ in kvs]
        # planned for a step's first layer, the others bring their chunks' addresses
        key = (*self._layout_key("fp4_rows", pc), _lib.stream_ptr(query.device), tuple(starts),
               tuple(of), tuple(lens))
        plan = step.fast.get(key)
        if plan is None:
            if max(seq_lens) > block_table.shape[1] * pc.block_size:
                raise ValueError("segment extends past the block-table row")
            if min(seq_lens) < 0:
                raise ValueError("negative segment start/length")
            rows = np.arange(n)
            plan = step.fast[key] = {"batch": None, "rows": self._plan_fp4_rows(
                query, rows, rows, seq_lens, block_table, pc, starts)}
        lse = torch.empty((self.num_heads, n), dtype=torch.float32, device=query.device)
        self._run_fp4_rows(plan["rows"], query, out, pc, False, lse)
        _count("decode")
        if not kvs:
            return
        words, batch = _chunk_words(kvs), plan["batch"]
        if batch is None:
            ent = np.zeros(len(kvs), dtype=ENTRY_DTYPE)
            ent["q_start"], ent["q_len"], ent["len"] = of, 1, lens
            for i, f in enumerate(("k_addr", "v_addr", "stride_tok", "stride_head")):
                ent[f] = words[:, i]
            batch = plan["batch"] = DecodeBatch.from_entries(
                ent, self.num_heads, self.num_kv_heads, self.head_size, query.device, keep=kvs,
                entry_seq=np.asarray(of, dtype=np.int32), num_seqs=n)
        else:
            batch = batch.rebind_chunks(words, kvs)
        batch.run(query, out, None, self.scale, acc=(out, lse))
        _count("decode")

    def _local_launch(self, query, plan: _Plan, step, pc):
        """The launch of a plan's local entries, shared by the layers that plan
        the same ones (a layer whose staging differs makes its own)."""
        _check_base(pc)
        key = (*self._layout_key("local", pc), _lib.stream_ptr(query.device), tuple(plan.local))
        pre = step.fast.get(key)
        if pre is None:
            a = np.array(plan.local, dtype=np.int64).reshape(-1, 6)
            pre = step.fast[key] = self._chunk_launch(
                paged_entry_array(pc, step.bt, a[:, 2], a[:, 0], a[:, 1], a[:, 5], a[:, 3],
                                  a[:, 4], relative=True), query, step.bt, pc)
        return pre

    def _forward_prefill(self, query, out, plan: _Plan, step, pc) -> None:
        dev = query.device
        h = self.num_heads
        if not plan.any_peer:
            self._run_chunks(self._local_launch(query, plan, step, pc), query, out, step.bt, pc)
            _count("attn")
            return
        o_peer = lse_peer = None
        for rnd in plan.peer_rounds:
            o_r = torch.empty_like(query, memory_format=torch.contiguous_format)
            lse_r = torch.full((h, query.shape[0]), float("-inf"), dtype=torch.float32,
                               device=dev)
            for kind in ("contig", "paged"):
                if rnd[kind]:
                    VarlenLaunch(rnd[kind], False, kind == "paged", dev, heads=self._heads).run(
                        query, o_r, lse_r, self.num_kv_heads, self.scale)
                    _count("attn")
            if o_peer is None:
                o_peer, lse_peer = o_r, lse_r
            else:  # running merge of further prefix chunks (ring_decode.py:46-61)
                o_m = torch.empty_like(o_peer)
                lse_m = torch.empty_like(lse_peer)
                merge_attn_states(o_m, o_peer, lse_peer, o_r, lse_r, lse_m)
                _count("merge")
                o_peer, lse_peer = o_m, lse_m
        # Local causal pass merged with the peer result in the same launch:
        # merge_attn_states(out, o_peer, lse_peer, o_loc, lse_loc) with prefix
        # = peer, suffix = local (ring_backend.py:354,820-831), bit for bit.
        # The local entries cover every query row of the plan; rows without a
        # peer have lse_peer = -inf and get the local result.
        # (planned, in a step's first layer, while the peer launches run)
        self._run_chunks(self._local_launch(query, plan, step, pc), query, out, step.bt, pc,
                         acc=(o_peer, lse_peer))
        _count("attn")
        _count("merge")

    def _forward_decode(self, query, out, plan: _Plan, block_table, pc, n: int, ring_local=None):
        """One split-KV launch for the whole decode batch; decode-ring rows
        get their owner-local partial (with LSE) from the same launch."""
        segs: list[list] = [[] for _ in range(n)]
        w = self.sliding_window
        for (qs, _tq, r, start, length, off) in plan.local:
            kv = segment_paged(pc, block_table[r], start, length)
            if w is not None:  # the causal local pass sees keys (off - w, off]
                kv = trim_segment(kv, min(kv.len, max(0, off - w + 1)))
            segs[qs].append(kv)
        for rnd in plan.peer_rounds:
            for kind in ("contig", "paged"):
                for e in rnd[kind]:
                    segs[e.q_start].append(e.kv)
        lse = None
        for (r, qs, *_r) in plan.ring:
            segs[qs] = [s for s in ring_local[r] if s is not None and s.len > 0]
        if plan.ring:
            lse = torch.empty((self.num_heads, n), dtype=torch.float32, device=query.device)
        DecodeBatch(segs, self.num_heads, self.num_kv_heads, self.head_size,
                    query.device).run(query, out, lse, self.scale)
        _count("decode")
        return lse
