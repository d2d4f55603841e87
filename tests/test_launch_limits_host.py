"""CPU: calls whose launches would have 2^32 threads or more are refused by name."""

import ctypes

import pytest

from hcp_vllm_plugin_amd import _lib
from tests.test_drafts_host import _drafts_args, _verify_args


@pytest.mark.parametrize("seqs,most,vocab", [
    (65536, 64, 32768), (65536, 64, 152064), (65536, 32, 65536), (65536, 14, 152064),
    (16384, 1, (1 << 22) - 3000)])
def test_verify_drafts(seqs, most, vocab):
    a = _verify_args()
    a.num_seqs, a.max_tokens, a.vocab, a.workspace_bytes = seqs, most, vocab, 1 << 40
    assert _lib.lib().hcp_verify_drafts(ctypes.addressof(a), None) == _lib.HCP_EUNSUPPORTED


@pytest.mark.parametrize("fp4", [0, 1])
@pytest.mark.parametrize("heads", [4096, 4094, 16384])
def test_decode_drafts(fp4, heads):
    a = _drafts_args(fp4)
    a.max_tokens, a.q_rows, a.decode.num_seqs, a.decode.workspace_bytes = 64, 65536, 1024, 1 << 50
    a.decode.num_heads = a.decode.num_kv_heads = heads
    a.decode.o_stride_tok = heads * 128
    assert _lib.lib().hcp_decode_drafts(ctypes.addressof(a), None) == _lib.HCP_EUNSUPPORTED
