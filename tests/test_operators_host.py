"""CPU: what the 4-bit cache, ``qk_norm_rope`` and ``build_step_tables`` refuse before
anything reaches the GPU, and the layout of their argument blocks."""

import ctypes
import os
import re

import pytest
import torch

from hcp_vllm_plugin_amd import _lib, build_step_tables, decode_fp4, qk_norm_rope
from hcp_vllm_plugin_amd.kv_cache import fp4_cache_shape, gather_kv, reshape_and_cache
from hcp_vllm_plugin_amd.ring_backend import HcpRingAttentionImpl
from hcp_vllm_plugin_amd.varlen import PagedCache, rows_apart, segment_paged
from tests import _fp4_util as f4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def _header_fields(struct):
    src = open(os.path.join(ROOT, "include", "hcp_mi355x.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), src, re.S).group(1)
    out = []
    for decl in body.split(";"):
        names = re.findall(r"(\w+)(?=\s*(?:,|$))", decl.strip())
        kind = "p" if "*" in decl else decl.strip().split(" ")[0] if decl.strip() else ""
        out += [(n, kind) for n in names]
    return out


@pytest.mark.parametrize("struct,cls", [("hcp_fp4_cache", _lib.Fp4CacheDesc),
                                        ("hcp_qk_rope_args", _lib.QkRopeArgs),
                                        ("hcp_step_tables_args", _lib.StepTablesArgs)])
def test_argument_blocks_match_the_header(struct, cls):
    kinds = {"p": ctypes.c_uint64, "uint64_t": ctypes.c_uint64, "int64_t": ctypes.c_int64,
             "int32_t": ctypes.c_int32, "double": ctypes.c_double}
    want = [(n, kinds[k]) for n, k in _header_fields(struct)]
    assert [(n, t) for n, t in cls._fields_] == want


def test_limits_match_the_header():
    src = open(os.path.join(ROOT, "include", "hcp_mi355x.h")).read()
    assert int(re.search(r"HCP_STEP_MAX_SEQS (\d+)", src).group(1)) == _lib.STEP_MAX_SEQS


def test_shapes():
    assert fp4_cache_shape(7, 4, 16, 128) == (7, 4, 16, 136)
    pc = PagedCache.from_tensor(torch.zeros(7, 4, 32, 68, dtype=torch.uint8))
    assert (pc.layout, pc.num_kv_heads, pc.head_dim, pc.block_size) == ("fp4", 4, 64, 32)
    assert (pc.stride_block, pc.stride_head) == (4 * 32 * 68, 32 * 68)
    for d, bs in ((80, 16), (0, 16), (288, 16), (128, 8), (128, 24), (128, 1 << 17)):
        with pytest.raises(ValueError, match="4-bit cache"):
            fp4_cache_shape(1, 1, bs, d)
    for shape in ((7, 4, 16, 128), (7, 2, 4, 16, 136), (7, 16, 136)):
        with pytest.raises(ValueError):
            PagedCache.from_tensor(torch.zeros(shape, dtype=torch.uint8))
    apart = torch.zeros(7, 4, 16, 272, dtype=torch.uint8)[..., :136]
    with pytest.raises(ValueError, match="contiguous"):
        PagedCache.from_tensor(apart)
    with pytest.raises(ValueError, match="no segments"):
        segment_paged(pc, torch.zeros(2, dtype=torch.int32), 0, 5)


def test_format():
    """The plain format itself: every code reads back as itself; the values of one scale."""
    x = torch.tensor([7.0, 6.0, 5.0, -5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.26, 0.0] + [0] * 20,
                     dtype=torch.bfloat16)
    assert f4.scale_bytes(x).tolist() == [127]
    want = [6, 6, 4, -4, 4, 2, 2, 1, 1, 0, -0.5, 0]
    assert f4.stand_for(x)[:12].tolist() == want
    y = f4.stand_for(x).to(torch.bfloat16)
    assert torch.equal(f4.stand_for(y), y.double())
    assert f4.scale_bytes(torch.tensor([7.0625] + [0] * 31, dtype=torch.bfloat16)).item() == 128
    big = torch.tensor([65504.0] + [0] * 31, dtype=torch.float16)
    assert f4.stand_for(big)[0] == 6 * 2.0 ** 13  # the largest finite value of a code
    assert f4.stand_for(torch.tensor([2.0 ** -24] + [0] * 31, dtype=torch.float16))[0] == 2.0 ** -24
    bad = torch.tensor([1.0, float("inf")] + [0] * 30, dtype=torch.bfloat16)
    assert torch.isnan(f4.stand_for(bad)).all()


def _cache_desc(**kw):
    d = _lib.Fp4CacheDesc(0x1000, 4 * 2176, 2176, 10, 16, 128)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,status", [
    ({"head_dim": 80}, _lib.HCP_EUNSUPPORTED), ({"head_dim": 288}, _lib.HCP_EUNSUPPORTED),
    ({"block_size": 8}, _lib.HCP_EUNSUPPORTED), ({"block_size": 48}, _lib.HCP_EUNSUPPORTED),
    ({"addr": 0x1008}, _lib.HCP_EINVAL), ({"addr": 0}, _lib.HCP_EINVAL),
    ({"stride_head": 2184}, _lib.HCP_EINVAL), ({"num_blocks": -1}, _lib.HCP_EINVAL),
    ({"num_blocks": 1 << 31}, _lib.HCP_EINVAL)])
def test_c_entries_refuse_a_cache(L, kw, status):
    d = _cache_desc(**kw)
    at = ctypes.addressof(d)
    assert L.hcp_fp4_write(4096, 512, 128, 4096, 512, 128, 4096, _lib.DTYPE_I64, 5, 4, at,
                           _lib.DTYPE_BF16, None) == status
    assert L.hcp_fp4_read(4096, _lib.DTYPE_I64, 5, 4, at, _lib.DTYPE_BF16, 4096, 4096, None) == status
    assert L.hcp_fp4_gather(4096, 1, 4096, 5, 4, at, _lib.DTYPE_BF16, 4096, 4096, None, None) == status
    a = _decode_args()
    a.kv.k_addr, a.kv.stride_block, a.kv.stride_head = d.addr, d.stride_block, d.stride_head
    a.kv.block_size, a.head_dim = d.block_size, d.head_dim
    if "num_blocks" not in kw:
        got = L.hcp_decode_fp4(ctypes.addressof(a), None)
        assert got == status or (kw.get("head_dim") == 288 and got == _lib.HCP_EUNSUPPORTED)


def test_c_writes_and_reads_refuse(L):
    d = _cache_desc()
    at = ctypes.addressof(d)
    ok = [4096, 512, 128, 4096, 512, 128, 4096, _lib.DTYPE_I64, 5, 4, at, _lib.DTYPE_BF16, None]
    for i, x, status in ((0, None, _lib.HCP_EINVAL), (0, 4104, _lib.HCP_EINVAL),
                         (2, 100, _lib.HCP_EINVAL), (6, None, _lib.HCP_EINVAL),
                         (7, _lib.DTYPE_F32, _lib.HCP_EUNSUPPORTED), (8, -1, _lib.HCP_EINVAL),
                         (8, 1 << 40, _lib.HCP_EINVAL), (9, 0, _lib.HCP_EINVAL),
                         (10, None, _lib.HCP_EINVAL), (11, _lib.DTYPE_F32, _lib.HCP_EUNSUPPORTED)):
        args = list(ok)
        args[i] = x
        assert L.hcp_fp4_write(*args) == status, (i, x)
        assert b"hcp_fp4_write" in L.hcp_last_error()
    ok[8] = 0
    assert L.hcp_fp4_write(*ok) == _lib.HCP_OK  # nothing to write
    ok[8], d.num_blocks, d.addr = 5, 0, 0
    assert L.hcp_fp4_write(*ok) == _lib.HCP_OK  # nowhere to write
    d.num_blocks, d.addr = 10, 0x1000
    ok[8] = (1 << 32) // (4 * 16)  # threads past 32 bits
    assert L.hcp_fp4_write(*ok) == _lib.HCP_EINVAL
    ok = [4096, _lib.DTYPE_I64, 5, 4, at, _lib.DTYPE_BF16, 4096, 4096, None]
    for i, x in ((0, None), (2, -1), (3, 0), (4, None), (6, None), (7, 4104)):
        args = list(ok)
        args[i] = x
        assert L.hcp_fp4_read(*args) == _lib.HCP_EINVAL, (i, x)
    ok = [4096, 1, 4096, 5, 4, at, _lib.DTYPE_BF16, 4096, 4096, None, None]
    for i, x in ((0, None), (1, -1), (1, 65536), (2, None), (2, 4100), (3, -1), (5, None), (7, 4104),
                 (9, 4100)):
        args = list(ok)
        args[i] = x
        assert L.hcp_fp4_gather(*args) == _lib.HCP_EINVAL, (i, x)


def _decode_args():
    a = _lib.DecodePagedArgs()
    a.q = a.out = a.seq_lens = a.workspace = 0x10000
    a.q_stride_tok, a.q_stride_head = 28 * 128, 128
    a.o_stride_tok, a.o_stride_head = 28 * 128, 128
    a.kv.k_addr, a.kv.block_table = 0x1000, 0x2000
    a.kv.stride_head, a.kv.stride_block, a.kv.block_size, a.kv.num_blocks = 2176, 4 * 2176, 16, 10
    a.block_table_stride = a.block_table_width = 8
    a.lens_dtype, a.num_seqs = _lib.DTYPE_I32, 3
    a.num_heads, a.num_kv_heads, a.head_dim, a.dtype = 28, 4, 128, _lib.DTYPE_BF16
    a.scale, a.workspace_bytes = 0.1, 1 << 30
    return a


def test_c_decode_refuses(L):
    need = L.hcp_decode_fp4_workspace(3, 28, 4, 128)
    assert need >= (3 + 64) * 28 * 129 * 4 and need % 4 == 0
    assert L.hcp_decode_fp4_workspace(0, 28, 4, 128) == 0
    assert L.hcp_decode_fp4_workspace(3, 27, 4, 128) == 0
    assert L.hcp_decode_fp4(None, None) == _lib.HCP_EINVAL
    for field, x, status in (
            ("num_heads", 27, _lib.HCP_EINVAL), ("dtype", _lib.DTYPE_F32, _lib.HCP_EUNSUPPORTED),
            ("num_seqs", -1, _lib.HCP_EINVAL), ("num_seqs", 1025, _lib.HCP_EUNSUPPORTED),
            ("window", -1, _lib.HCP_EINVAL), ("block_table_width", 0, _lib.HCP_EINVAL),
            ("block_table_width", 1 << 28, _lib.HCP_EUNSUPPORTED),
            ("block_table_width", (1 << 27) - 20, _lib.HCP_EUNSUPPORTED), ("q", 0, _lib.HCP_EINVAL),
            ("q", 0x10008, _lib.HCP_EINVAL), ("q_stride_tok", 100, _lib.HCP_EINVAL),
            ("scale", 0.0, _lib.HCP_EINVAL), ("lens_dtype", 7, _lib.HCP_EUNSUPPORTED),
            ("workspace_bytes", need - 1, _lib.HCP_EWORKSPACE), ("workspace", 8, _lib.HCP_EINVAL)):
        a = _decode_args()
        setattr(a, field, x)
        assert L.hcp_decode_fp4(ctypes.addressof(a), None) == status, field
    a = _decode_args()
    a.kv.num_blocks = 0
    assert L.hcp_decode_fp4(ctypes.addressof(a), None) == _lib.HCP_EINVAL
    a = _decode_args()
    a.num_seqs = 0
    assert L.hcp_decode_fp4(ctypes.addressof(a), None) == _lib.HCP_OK
    a = _decode_args()  # the 16-bit cache's launch has no first keys
    a.kv.v_addr, a.kv.stride_tok, a.seq_starts = 0x1000, 512, 0x3000
    assert L.hcp_decode_paged(ctypes.addressof(a), None) == _lib.HCP_EUNSUPPORTED


def _rope_args():
    a = _lib.QkRopeArgs()
    for f in ("q", "k", "v", "q_out", "k_out", "positions", "cos_sin", "slot_mapping"):
        setattr(a, f, 0x10000)
    for f in ("q", "k", "v", "qo", "ko"):
        setattr(a, f + "_stride_tok", 512)
        setattr(a, f + "_stride_head", 128)
    a.table_stride, a.max_positions, a.num_slots, a.num_tokens = 128, 100, 5, 5
    a.eps, a.num_heads, a.num_kv_heads, a.head_dim, a.rot = 1e-6, 4, 4, 128, 128
    a.dtype = a.weight_dtype = a.table_dtype = _lib.DTYPE_BF16
    a.pos_dtype = a.slot_dtype = _lib.DTYPE_I64
    return a


def test_c_rope_refuses(L):
    assert L.hcp_qk_norm_rope(None, None) == _lib.HCP_EINVAL
    for kw, status in (
            ({"num_heads": 0}, _lib.HCP_EINVAL), ({"head_dim": 12}, _lib.HCP_EUNSUPPORTED),
            ({"head_dim": 264}, _lib.HCP_EUNSUPPORTED), ({"rot": 8}, _lib.HCP_EUNSUPPORTED),
            ({"rot": 144}, _lib.HCP_EUNSUPPORTED), ({"rot": -16}, _lib.HCP_EUNSUPPORTED),
            ({"dtype": _lib.DTYPE_F32}, _lib.HCP_EUNSUPPORTED),
            ({"table_dtype": _lib.DTYPE_F16}, _lib.HCP_EUNSUPPORTED),
            ({"weight_dtype": _lib.DTYPE_F16}, _lib.HCP_EUNSUPPORTED),
            ({"pos_dtype": 2}, _lib.HCP_EUNSUPPORTED), ({"cache_kind": 3}, _lib.HCP_EINVAL),
            ({"num_tokens": -1}, _lib.HCP_EINVAL), ({"num_slots": 6}, _lib.HCP_EINVAL),
            ({"num_tokens": 1 << 26}, _lib.HCP_EINVAL),
            ({"eps": -1.0}, _lib.HCP_EINVAL), ({"eps": float("nan")}, _lib.HCP_EINVAL),
            ({"q": 0}, _lib.HCP_EINVAL), ({"q_out": 0x10004}, _lib.HCP_EINVAL),
            ({"positions": 0}, _lib.HCP_EINVAL), ({"max_positions": 0}, _lib.HCP_EINVAL),
            ({"k_out": 0}, _lib.HCP_EINVAL), ({"k_stride_tok": 4}, _lib.HCP_EINVAL),
            ({"cache_kind": 1}, _lib.HCP_EINVAL), ({"cache_kind": 2}, _lib.HCP_EINVAL),
            ({"cache_kind": 2, "v": 0}, _lib.HCP_EINVAL)):
        a = _rope_args()
        for k, v in kw.items():
            setattr(a, k, v)
        assert L.hcp_qk_norm_rope(ctypes.addressof(a), None) == status, kw
    a = _rope_args()
    d = _cache_desc(head_dim=64)
    a.cache_kind, a.fp4 = 2, ctypes.addressof(d)
    assert L.hcp_qk_norm_rope(ctypes.addressof(a), None) == _lib.HCP_EINVAL
    c = _lib.PagedCacheDesc(0x1000, 0x1100, 16384, 4096, 256, 10, 12, 0)
    a.cache_kind, a.cache = 1, ctypes.addressof(c)
    assert L.hcp_qk_norm_rope(ctypes.addressof(a), None) == _lib.HCP_EINVAL  # block_size 12
    c.block_size, c.k_addr = 16, 0x1008
    assert L.hcp_qk_norm_rope(ctypes.addressof(a), None) == _lib.HCP_EINVAL
    a = _rope_args()
    a.num_tokens = a.num_slots = 0
    assert L.hcp_qk_norm_rope(ctypes.addressof(a), None) == _lib.HCP_OK


def test_c_tables_refuse(L):
    assert L.hcp_step_tables(None, None) == _lib.HCP_EINVAL

    def args():
        a = _lib.StepTablesArgs()
        for f in ("ctx_lens", "new_lens", "block_table", "free_blocks", "query_start_loc", "seq_lens",
                  "blocks_used", "positions", "slot_mapping"):
            setattr(a, f, 0x10000)
        a.ctx_stride = a.new_stride = 1
        a.table_stride = a.table_width = 8
        a.num_free, a.num_tokens, a.num_seqs, a.block_size = 4, 10, 3, 16
        a.ctx_dtype = a.new_dtype = _lib.DTYPE_I32
        return a

    for kw, status in (
            ({"num_seqs": -1}, _lib.HCP_EINVAL), ({"num_seqs": 4097}, _lib.HCP_EUNSUPPORTED),
            ({"num_tokens": -1}, _lib.HCP_EINVAL), ({"num_tokens": 1 << 31}, _lib.HCP_EUNSUPPORTED),
            ({"table_width": 1 << 20}, _lib.HCP_EUNSUPPORTED), ({"block_size": 24}, _lib.HCP_EINVAL),
            ({"block_size": 0}, _lib.HCP_EINVAL), ({"ctx_dtype": 0}, _lib.HCP_EUNSUPPORTED),
            ({"ctx_lens": 0}, _lib.HCP_EINVAL), ({"block_table": 0}, _lib.HCP_EINVAL),
            ({"free_blocks": 0}, _lib.HCP_EINVAL), ({"blocks_used": 0}, _lib.HCP_EINVAL),
            ({"slot_mapping": 0}, _lib.HCP_EINVAL), ({"num_free": -1}, _lib.HCP_EINVAL)):
        a = args()
        for k, v in kw.items():
            setattr(a, k, v)
        assert L.hcp_step_tables(ctypes.addressof(a), None) == status, kw


def test_python_refuses():
    """Shapes, types and places, on CPU tensors: nothing is launched."""
    cache = torch.zeros(fp4_cache_shape(4, 2, 16, 64), dtype=torch.uint8)
    k, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.arange(3)
    for key, value, s in ((k[:, :1], k[:, :1], slots), (k, k[:2], slots), (k[:2], k[:2], slots),
                          (k.float(), k.float(), slots), (k, k.half(), slots),
                          (k, k, slots.float()), (k, k, slots)):
        with pytest.raises(ValueError):
            reshape_and_cache(key, value, cache, s)
    for c, s, t in ((cache, slots, torch.float32), (cache.to(torch.int8), slots, torch.bfloat16),
                    (cache, slots, torch.bfloat16), (cache, slots[None], torch.bfloat16)):
        with pytest.raises(ValueError):
            gather_kv(c, s, t)
    q, bt = torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32)
    lens = torch.tensor([3, 4])
    for args in ((q.float(), cache, bt, lens), (q[0], cache, bt, lens), (q[:, :3], cache, bt, lens),
                 (q[..., :32], cache, bt, lens), (q, torch.zeros(4, 2, 16, 128), bt, lens),
                 (q, cache, bt, lens[:1]), (q, cache, bt, lens.float()), (q, cache, bt, lens)):
        with pytest.raises(ValueError):
            decode_fp4(*args, 0.1)
    with pytest.raises(ValueError, match="window"):
        decode_fp4(q, cache, bt, lens, 0.1, window=0)
    with pytest.raises(ValueError):
        qk_norm_rope(q, q[:, :2], torch.zeros(2, dtype=torch.int64), torch.zeros(4, 64))
    for bad in ({"block_size": 24}, {"num_tokens": -1}, {}):
        kw = {"block_size": 16, "num_tokens": 4, **bad}
        with pytest.raises(ValueError):
            build_step_tables(lens, lens, bt, torch.zeros(2, dtype=torch.int32), **kw)
    with pytest.raises(NotImplementedError):
        HcpRingAttentionImpl(4, 80, 0.1, 2, kv_cache_dtype="fp4")
    with pytest.raises(NotImplementedError):
        HcpRingAttentionImpl(4, 64, 0.1, 2, kv_cache_dtype="fp8")


def test_overlapping_table_rows_are_refused(L):
    lens, free = torch.tensor([3, 4]), torch.zeros(2, dtype=torch.int32)
    for bt in (torch.zeros(1, 3, dtype=torch.int32).expand(2, 3),
               torch.zeros(8, dtype=torch.int32).as_strided((2, 3), (2, 1))):
        with pytest.raises(ValueError, match="rows"):
            build_step_tables(lens, lens, bt, free, 16, 4)
    a = _lib.StepTablesArgs()
    for f in ("ctx_lens", "new_lens", "block_table", "query_start_loc", "seq_lens", "blocks_used"):
        setattr(a, f, 0x10000)
    a.table_stride, a.table_width, a.num_seqs, a.block_size = 7, 8, 2, 16
    a.ctx_dtype = a.new_dtype = _lib.DTYPE_I32
    assert L.hcp_step_tables(ctypes.addressof(a), None) == _lib.HCP_EINVAL


def test_outputs_on_top_of_each_other_are_refused(L):
    """Strides that let rows share bytes in part, not only strides of 0."""
    for field in ("qo_stride_tok", "qo_stride_head", "ko_stride_tok", "ko_stride_head"):
        for stride in (0, 64, 120, 504 if field.endswith("tok") else 632):
            a = _rope_args()
            setattr(a, field, stride)
            assert L.hcp_qk_norm_rope(ctypes.addressof(a), None) == _lib.HCP_EINVAL, (field, stride)
            assert b"on top" in L.hcp_last_error()
    for field, stride in (("o_stride_tok", 0), ("o_stride_tok", 28 * 128 - 1), ("o_stride_head", 127),
                          ("o_stride_head", 28 * 128 + 1)):
        a = _decode_args()
        setattr(a, field, stride)
        assert L.hcp_decode_fp4(ctypes.addressof(a), None) == _lib.HCP_EINVAL, (field, stride)
        assert b"on top" in L.hcp_last_error()


@pytest.mark.parametrize("shape,strides,apart", [
    ((3, 4, 64), (256, 64, 1), True), ((3, 4, 64), (64, 192, 1), True),  # tokens or heads outside
    ((3, 4, 64), (1000, 64, 1), True), ((3, 4, 64), (255, 64, 1), False),
    ((3, 4, 64), (256, 63, 1), False), ((3, 4, 64), (64, 191, 1), False),
    ((3, 4, 64), (0, 64, 1), False), ((3, 4, 64), (256, 0, 1), False),
    ((1, 4, 64), (0, 64, 1), True), ((1, 4, 64), (0, 63, 1), False),
    ((3, 1, 64), (64, 0, 1), True), ((3, 1, 64), (63, 0, 1), False),
    ((1, 1, 64), (0, 0, 1), True), ((0, 4, 64), (256, 64, 1), True)])
def test_rows_apart(shape, strides, apart):
    t = torch.zeros(4000).as_strided(shape, strides)
    assert rows_apart(t) == apart
    flat = torch.arange(4000).as_strided(shape, strides).flatten()
    assert (flat.unique().numel() == flat.numel()) == apart


def test_caches_on_top_of_themselves_are_not_written(L):
    """Blocks or heads of a cache that share bytes, whichever of the two is the outer one;
    reading them is no race."""
    region = 16 * 136
    for block, head, status in ((0, region, _lib.HCP_EINVAL), (4 * region, 0, _lib.HCP_EINVAL),
                                (4 * region - 16, region, _lib.HCP_EINVAL),
                                (4 * region, region - 16, _lib.HCP_EINVAL),
                                (region, 10 * region - 16, _lib.HCP_EINVAL),
                                (region - 16, 10 * region, _lib.HCP_EINVAL),
                                (4 * region, region, None), (region, 10 * region, None)):
        d = _cache_desc(stride_block=block, stride_head=head)
        at = ctypes.addressof(d)
        n = 5 if status is not None else 0  # (what is taken is not launched here)
        want = _lib.HCP_OK if status is None else status
        assert L.hcp_fp4_write(4096, 512, 128, 4096, 512, 128, 4096, _lib.DTYPE_I64, n, 4, at,
                               _lib.DTYPE_BF16, None) == want, (block, head)
        a = _rope_args()
        a.cache_kind, a.fp4 = 2, at
        if status is not None:
            assert L.hcp_qk_norm_rope(ctypes.addressof(a), None) == want, (block, head)
            assert b"on top" in L.hcp_last_error()
        assert L.hcp_fp4_read(4096, _lib.DTYPE_I64, 0, 4, at, _lib.DTYPE_BF16, 4096, 4096,
                              None) == _lib.HCP_OK
    # 16-bit layouts, in elements: K and V of a row side by side, or blocks of either
    for v, block, head, tok in ((256, 0, 4096, 256), (256, 16384, 0, 256), (256, 16384, 4096, 0),
                                (256, 16384, 4096, 248), (256, 16384, 4088, 256), (0, 16384, 4096, 256),
                                (128, 16384, 4096, 256), (16384, 16384 - 8, 128, 512)):
        a = _rope_args()
        c = _lib.PagedCacheDesc(0x1000, 0x1000 + v, block, head, tok, 10, 16, 0)
        a.cache_kind, a.cache = 1, ctypes.addressof(c)
        assert L.hcp_qk_norm_rope(ctypes.addressof(a), None) == _lib.HCP_EINVAL, (v, block, head, tok)
        assert b"on top" in L.hcp_last_error(), (v, block, head, tok)
