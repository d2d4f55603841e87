"""CPU: what ``decode_drafts``, ``verify_drafts`` and ``rope_table`` refuse before anything
reaches the GPU, and the layout of their argument blocks."""

import ctypes
import math
import os
import re

import pytest
import torch

from hcp_vllm_plugin_amd import _lib, decode_drafts, rope_table, verify_drafts
from hcp_vllm_plugin_amd.kv_cache import fp4_cache_shape
from tests._drafts_util import draw, verify

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def _header():
    src = open(os.path.join(ROOT, "include", "hcp_mi355x.h")).read()
    return re.sub(r"/\*.*?\*/", "", src, flags=re.S)


@pytest.mark.parametrize("struct,cls", [("hcp_decode_drafts_args", _lib.DecodeDraftsArgs),
                                        ("hcp_verify_args", _lib.VerifyArgs),
                                        ("hcp_rope_table_args", _lib.RopeTableArgs)])
def test_argument_blocks_match_the_header(struct, cls):
    kinds = {"p": ctypes.c_uint64, "uint64_t": ctypes.c_uint64, "int64_t": ctypes.c_int64,
             "int32_t": ctypes.c_int32, "double": ctypes.c_double,
             "hcp_decode_paged_args": _lib.DecodePagedArgs}
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), _header(), re.S).group(1)
    want = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        kind = "p" if "*" in decl else decl.split(" ")[0]
        want += [(n, kinds[kind]) for n in re.findall(r"(\w+)(?=\s*(?:,|$))", decl)]
    assert [(n, t) for n, t in cls._fields_] == want


def test_limits_match_the_header():
    src = _header()
    assert int(re.search(r"HCP_DRAFTS_MAX_TOKENS (\d+)", src).group(1)) == _lib.DRAFTS_MAX_TOKENS
    assert int(re.search(r"HCP_VERIFY_MAX_TOKENS (\d+)", src).group(1)) == _lib.VERIFY_MAX_TOKENS


def _drafts_args(fp4):
    a = _lib.DecodeDraftsArgs()
    d = a.decode
    d.q = d.out = d.seq_lens = d.workspace = 0x10000
    d.q_stride_tok, d.q_stride_head = 28 * 128, 128
    d.o_stride_tok, d.o_stride_head = 28 * 128, 128
    d.kv.k_addr, d.kv.v_addr, d.kv.block_table = 0x1000, 0x1100, 0x2000
    d.kv.stride_head, d.kv.stride_block = (2176, 4 * 2176) if fp4 else (16 * 256, 4 * 16 * 256)
    d.kv.stride_tok = 0 if fp4 else 256
    d.kv.block_size, d.kv.num_blocks = 16, 10
    d.block_table_stride = d.block_table_width = 8
    d.lens_dtype, d.num_seqs = _lib.DTYPE_I32, 3
    d.num_heads, d.num_kv_heads, d.head_dim, d.dtype = 28, 4, 128, _lib.DTYPE_BF16
    d.scale, d.workspace_bytes = 0.1, 1 << 30
    a.row_starts, a.q_rows, a.max_tokens, a.fp4 = 0x3000, 12, 4, fp4
    return a


@pytest.mark.parametrize("fp4", [0, 1])
def test_c_decode_drafts_refuses(L, fp4):
    need = L.hcp_decode_drafts_workspace(3, 4, 28, 4, 128, fp4)
    assert need >= (3 + 64) * 4 * 28 * 129 * 4 and need % 8 == 0
    for bad in ((0, 4, 28, 4, 128), (1025, 4, 28, 4, 128), (3, 0, 28, 4, 128), (3, 65, 28, 4, 128),
                (3, 4, 27, 4, 128), (3, 4, 28, 4, 0), (3, 4, 28, 4, 264)):
        assert L.hcp_decode_drafts_workspace(*bad, fp4) == 0, bad
    assert L.hcp_decode_drafts(None, None) == _lib.HCP_EINVAL
    E, U = _lib.HCP_EINVAL, _lib.HCP_EUNSUPPORTED
    for field, x, status in (
            ("num_heads", 27, E), ("dtype", _lib.DTYPE_F32, U), ("num_seqs", -1, E),
            ("num_seqs", 1025, U), ("window", -1, E), ("block_table_width", 0, E),
            ("block_table_width", 1 << 28, U), ("block_table_width", (1 << 27) - 60, U), ("q", 0, E),
            ("q", 0x10008, E), ("q_stride_tok", 100, E), ("scale", 0.0, E),
            ("scale", float("inf"), E), ("lens_dtype", 7, U), ("seq_lens", 0, E), ("out", 0, E),
            ("workspace_bytes", need - 1, _lib.HCP_EWORKSPACE), ("workspace", 0x10008, E),
            ("workspace", 0, _lib.HCP_EWORKSPACE), ("seq_starts", 0x5000, U), ("head_dim", 20, U),
            ("o_stride_tok", 0, E), ("o_stride_tok", 28 * 128 - 1, E), ("o_stride_head", 127, E),
            ("head_dim", 264, U)):
        a = _drafts_args(fp4)
        setattr(a.decode, field, x)
        assert L.hcp_decode_drafts(ctypes.addressof(a), None) == status, (field, x)
    a = _drafts_args(fp4)
    a.decode.num_seqs, a.decode.num_heads, a.decode.num_kv_heads, a.max_tokens = 1024, 65536, 65536, 64
    assert L.hcp_decode_drafts(ctypes.addressof(a), None) == U  # more merging waves than a launch has
    for field, x, status in (("row_starts", 0, E), ("q_rows", -1, E), ("q_rows", 1 << 31, U),
                             ("max_tokens", 0, E), ("max_tokens", 65, U)):
        a = _drafts_args(fp4)
        setattr(a, field, x)
        assert L.hcp_decode_drafts(ctypes.addressof(a), None) == status, (field, x)
    kv = [("num_blocks", 0, E), ("block_size", 24, U if fp4 else E), ("k_addr", 0x1008, E)]
    kv += [("stride_head", 2180, E), ("block_size", 8, U)] if fp4 else \
        [("v_addr", 0, E), ("stride_tok", 4, E), ("stride_tok", 1 << 25, U), ("block_size", 0, E)]
    for field, x, status in kv:
        a = _drafts_args(fp4)
        setattr(a.decode.kv, field, x)
        assert L.hcp_decode_drafts(ctypes.addressof(a), None) == status, (field, x)
    a = _drafts_args(fp4)
    a.decode.lse, a.decode.lse_stride_head = 0x9000, 11  # 12 rows to a head
    assert L.hcp_decode_drafts(ctypes.addressof(a), None) == E
    for field in ("num_seqs", "q_rows"):
        a = _drafts_args(fp4)
        setattr(a.decode if field == "num_seqs" else a, field, 0)
        assert L.hcp_decode_drafts(ctypes.addressof(a), None) == _lib.HCP_OK  # nothing to run


def _verify_args():
    a = _lib.VerifyArgs()
    for f in ("target", "tokens", "row_starts", "uniform", "draft_probs", "temperature", "out",
              "num_out", "workspace"):
        setattr(a, f, 0x10000)
    a.row_stride, a.num_rows, a.uniform_stride = 1000, 12, 4
    a.q_stride_seq, a.q_stride_row = 3000, 1000
    a.vocab, a.num_seqs, a.max_tokens, a.workspace_bytes = 1000, 3, 4, 1 << 20
    a.dtype, a.tokens_dtype, a.starts_dtype = _lib.DTYPE_F32, _lib.DTYPE_I64, _lib.DTYPE_I32
    return a


def test_c_verify_refuses(L):
    need = L.hcp_verify_workspace(3, 4, 1000)
    assert 0 < need <= 1 << 20
    for bad in ((0, 4, 1000), (65537, 4, 1000), (3, 0, 1000), (3, 65, 1000), (3, 4, 0),
                (3, 4, (1 << 22) + 1)):
        assert L.hcp_verify_workspace(*bad) == 0, bad
    assert L.hcp_verify_drafts(None, None) == _lib.HCP_EINVAL
    E, U = _lib.HCP_EINVAL, _lib.HCP_EUNSUPPORTED
    for field, x, status in (
            ("num_seqs", -1, E), ("num_seqs", 65537, U), ("num_rows", -1, E), ("vocab", 0, E),
            ("vocab", (1 << 22) + 1, U), ("max_tokens", 0, E), ("max_tokens", 65, U),
            ("dtype", _lib.DTYPE_I32, U), ("tokens_dtype", _lib.DTYPE_F32, U), ("starts_dtype", 0, U),
            ("target", 0, E), ("tokens", 0, E), ("row_starts", 0, E), ("uniform", 0, E), ("out", 0, E),
            ("num_out", 0, E), ("workspace", 0, _lib.HCP_EWORKSPACE), ("workspace", 0x10008, E),
            ("workspace_bytes", need - 1, _lib.HCP_EWORKSPACE)):
        a = _verify_args()
        setattr(a, field, x)
        assert L.hcp_verify_drafts(ctypes.addressof(a), None) == status, (field, x)
    a = _verify_args()
    a.num_seqs, a.max_tokens, a.vocab = 65536, 64, 1 << 22
    assert L.hcp_verify_drafts(ctypes.addressof(a), None) == U  # more workgroups than a launch has
    a = _verify_args()
    a.num_seqs = 0
    assert L.hcp_verify_drafts(ctypes.addressof(a), None) == _lib.HCP_OK


def test_c_rope_table_refuses(L):
    def args(**kw):
        a = _lib.RopeTableArgs()
        a.out, a.stride, a.num_positions, a.base, a.attention_factor = 0x10000, 64, 100, 1e4, 1.0
        a.rot, a.dtype = 64, _lib.DTYPE_F32
        a.factor, a.original, a.low_freq, a.high_freq = 4.0, 8192.0, 1.0, 4.0
        a.beta_fast, a.beta_slow = 32.0, 1.0
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    E, U, nan, inf = _lib.HCP_EINVAL, _lib.HCP_EUNSUPPORTED, float("nan"), float("inf")
    assert L.hcp_rope_table(None, None) == E
    divisors = (ctypes.c_double * 32)(*([1.0] * 31 + [0.0]))
    for kw, status in (
            ({"rot": 8}, U), ({"rot": 0}, U), ({"rot": 272}, U), ({"dtype": _lib.DTYPE_I32}, U),
            ({"num_positions": -1}, E), ({"num_positions": (1 << 28) + 1}, E), ({"base": 1.0}, E),
            ({"base": nan}, E), ({"base": inf}, E), ({"attention_factor": nan}, E), ({"scaling": 5}, U),
            ({"scaling": -1}, U), ({"scaling": 1, "factor": 0.0}, E), ({"scaling": 1, "factor": inf}, E),
            ({"scaling": 2, "original": 0.0}, E), ({"scaling": 2, "high_freq": 1.0}, E),
            ({"scaling": 2, "low_freq": 0.0}, E), ({"scaling": 3, "beta_slow": 0.0}, E),
            ({"scaling": 3, "beta_fast": 0.5}, E), ({"scaling": 3, "original": nan}, E),
            ({"scaling": 4}, E), ({"scaling": 4, "divisors": ctypes.addressof(divisors)}, E),
            ({"out": 0}, E), ({"out": 0x10008}, E), ({"stride": 66}, E), ({"stride": 60}, E),
            ({"stride": 0}, E)):
        assert L.hcp_rope_table(ctypes.addressof(args(**kw)), None) == status, kw
    assert L.hcp_rope_table(ctypes.addressof(args(num_positions=0)), None) == _lib.HCP_OK


def test_python_refuses():
    """Shapes, types and places, on CPU tensors: nothing is launched."""
    bf = torch.bfloat16
    q, bt = torch.zeros(5, 4, 64, dtype=bf), torch.zeros(2, 3, dtype=torch.int32)
    lens, starts = torch.tensor([30, 40]), torch.tensor([0, 2, 5])
    for cache in (torch.zeros(4, 2, 16, 128, dtype=bf), torch.zeros(4, 2, 16, 2, 64, dtype=bf),
                  torch.zeros(fp4_cache_shape(4, 2, 16, 64), dtype=torch.uint8)):
        good = dict(q=q, kv_cache=cache, block_table=bt, seq_lens=lens, query_start_loc=starts,
                    max_tokens=3, scale=0.1)
        for bad in ({"q": q.float()}, {"q": q[0]}, {"q": q[:, :3]}, {"q": q[..., :32]},
                    {"kv_cache": cache[..., :-2]}, {"kv_cache": cache.float()}, {"max_tokens": 0},
                    {"max_tokens": 65}, {"window": 0}, {"window": -1}, {"seq_lens": lens[:1]},
                    {"seq_lens": lens.float()}, {"seq_lens": lens[:, None]},
                    {"query_start_loc": starts[:2]}, {"query_start_loc": starts.int()},
                    {"block_table": bt.long()}, {"block_table": bt[:1]}, {"block_table": bt.t()},
                    {"out": q.float()}, {"out": q[:4]}, {}):
            with pytest.raises(ValueError):
                decode_drafts(**{**good, **bad})
    x, tokens, u = torch.zeros(5, 100), torch.zeros(5, dtype=torch.int64), torch.zeros(2, 3)
    good = dict(target=x, tokens=tokens, query_start_loc=starts, uniform=u)
    for bad in ({"target": x.double()}, {"target": x[0]}, {"target": x.t()}, {"tokens": tokens[:4]},
                {"tokens": tokens.float()}, {"query_start_loc": starts.float()},
                {"query_start_loc": starts[:2]}, {"query_start_loc": starts[:0]}, {"uniform": u.double()},
                {"uniform": u[:1]}, {"uniform": torch.zeros(2, 65)}, {"uniform": torch.zeros(2, 0)},
                {"draft_probs": torch.zeros(2, 1, 100)}, {"draft_probs": torch.zeros(2, 2, 99)},
                {"draft_probs": torch.zeros(2, 2, 100).double()}, {"temperature": torch.ones(3)},
                {"temperature": torch.ones(2).double()}, {}):
        with pytest.raises(ValueError):
            verify_drafts(**{**good, **bad})
    for bad in ({"rot": 24}, {"rot": 0}, {"rot": 272}, {"max_positions": -1}, {"base": 1.0},
                {"base": math.nan}, {"dtype": torch.float64, "device": "cpu"}, {"device": "cpu"},
                {"out": torch.zeros(10, 32)}, {"scaling": {"rope_type": "other"}}, {"scaling": {}},
                {"scaling": {"rope_type": "linear"}},
                {"scaling": {"rope_type": "linear", "factor": 2.0, "rope_theta": 5e5}},
                {"scaling": {"rope_type": "default", "factor": 2.0}},
                {"scaling": {"rope_type": "yarn", "factor": 4.0, "truncate": False,
                             "original_max_position_embeddings": 8}},
                {"scaling": {"rope_type": "yarn", "factor": 4.0}},
                {"scaling": {"rope_type": "llama3", "factor": 4.0, "low_freq_factor": 1.0,
                             "original_max_position_embeddings": 8}},
                {"scaling": {"rope_type": "dynamic", "factor": 0.5,
                             "original_max_position_embeddings": 8}},
                {"scaling": {"rope_type": "longrope", "original_max_position_embeddings": 8,
                             "long_factor": [1.0] * 31}}):
        with pytest.raises(ValueError):
            rope_table(**{"max_positions": 10, "rot": 64, "device": "cpu", **bad})


def test_the_definition_itself():
    """The tests' own statement of verification, where it can be told by hand."""
    w = torch.tensor([0.5, 0.25, 0.25])
    assert draw(w.double(), 0.0) == 0 and draw(w.double(), 0.5) == 1 and draw(w.double(), 0.75) == 2
    assert draw(torch.zeros(3), 0.5) is None
    both, q = torch.stack([w, w]), torch.tensor([[[0.25, 0.5, 0.25]]])
    starts, tokens = torch.tensor([0, 2]), torch.tensor([0, 1])
    # p / q = 1/2 for token 1: accepted below it; max(p - q, 0) holds token 0 alone
    assert verify(both, tokens, starts, torch.tensor([[0.49, 0.9]]), q, probs=True) == [[1, 2]]
    assert verify(both, tokens, starts, torch.tensor([[0.5, 0.9]]), q, probs=True) == [[0]]
    # without q: p(1) = 1/4, then p without it
    assert verify(both, tokens, starts, torch.tensor([[0.25, 0.7]]), probs=True) == [[2]]
    cold = torch.zeros(1)
    assert verify(both, tokens, starts, torch.zeros(1, 2), temperature=cold, probs=True) == [[0]]
