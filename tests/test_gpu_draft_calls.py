"""GPU: calls of ``decode_drafts``, ``verify_drafts`` and ``rope_table`` at the ends of what
they allow: nothing to look at, shared rows, places past 2^32 bytes."""

import pytest
import torch

from hcp_vllm_plugin_amd import decode_drafts, rope_table, verify_drafts
from tests._drafts_util import batch, check, check_verified, verify
from tests._util import scale_for
from tests.test_gpu_rope_table import YARN
from tests.test_gpu_rope_table_float32 import wanted

pytestmark = pytest.mark.gpu


def test_no_rows_at_all(dev):
    got = verify_drafts(torch.zeros(0, 100, device=dev), torch.zeros(0, dtype=torch.int32, device=dev),
                        torch.zeros(4, dtype=torch.int32, device=dev), torch.rand(3, 2, device=dev))
    assert got.tokens.tolist() == [[-1, -1]] * 3 and got.num_tokens.tolist() == [0, 0, 0]
    got = verify_drafts(torch.zeros(2, 100, device=dev), torch.zeros(2, dtype=torch.int64, device=dev),
                        torch.zeros(1, dtype=torch.int64, device=dev), torch.rand(0, 2, device=dev))
    assert got.tokens.shape == (0, 2) and got.num_tokens.shape == (0,)


@pytest.mark.parametrize("v,n", [(300, 3), (30000, 3), (70001, 40)])
@pytest.mark.parametrize("probs", [True, False])
def test_shared_rows(dev, v, n, probs):
    """One row of the target, of the draft model and of the random numbers for all sequences."""
    gen = torch.Generator().manual_seed(v)
    x, q = torch.randn(v, generator=gen), torch.softmax(torch.randn(v, generator=gen), 0)
    x = torch.softmax(x, 0) if probs else x
    tokens = torch.randint(0, v, (3 * n,), generator=gen)
    tokens[1::3] = x.argmax()
    u, starts = torch.tensor([0.01, 0.02, 0.6]), torch.arange(0, 3 * n + 1, 3)
    want = verify(x.expand(3 * n, v), tokens, starts, u.expand(n, 3), q.expand(n, 2, v), None, probs)
    got = verify_drafts(x.to(dev).expand(3 * n, v), tokens.to(dev), starts.to(dev),
                        u.to(dev).expand(n, 3), draft_probs=q.to(dev).expand(n, 2, v), probs=probs)
    check_verified(got, want, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [1000, 20000])
def test_far_rows(dev, dtype, v):
    """Rows of the target 2.5 GiB apart, of the draft probabilities 9."""
    gen = torch.Generator().manual_seed(v)
    x = torch.randn(4, v, generator=gen).to(dtype)
    dp = torch.softmax(torch.randn(2, 1, v, generator=gen), -1)
    tokens, starts = torch.randint(0, v, (4,), generator=gen), torch.tensor([0, 2, 4])
    u = torch.tensor([[0.3, 0.7], [0.0, 0.2]])
    row, seq = (5 << 30) // dtype.itemsize // 2, (9 << 30) // 4
    far = torch.empty(3 * row + v, dtype=dtype, device=dev).as_strided((4, v), (row, 1))
    far.copy_(x)
    far_q = torch.empty(seq + v, device=dev).as_strided((2, 1, v), (seq, v, 1))
    far_q.copy_(dp)
    for q, fq in ((None, None), (dp, far_q)):
        want = verify(x, tokens, starts, u, q)
        check_verified(verify_drafts(far, tokens.to(dev), starts.to(dev), u.to(dev), draft_probs=fq),
                       want, 2)


@pytest.mark.parametrize("kind", ["v031", "fp4"])
def test_far_queries_and_outputs(dev, kind):
    gen = torch.Generator().manual_seed(1)
    lens, counts, step = [50, 200], [2, 1], (3 << 30) // 2
    q, cache, bt, starts, kvs = batch(gen, dev, lens, counts, 4, 2, 64, 16, torch.bfloat16, kind)
    rows = [torch.empty(2 * step + 256, dtype=torch.bfloat16, device=dev).as_strided(
        (3, 4, 64), (step, 64, 1)) for _ in range(2)]
    rows[0].copy_(q)
    got = decode_drafts(rows[0], cache, bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                        starts.to(dev), 2, scale_for(64), out=rows[1], with_lse=True)
    check(got, q, counts, kvs, scale_for(64), torch.bfloat16)


def test_one_table_row_for_all_sequences(dev):
    """A prompt that several requests share, each with its own length."""
    gen = torch.Generator().manual_seed(2)
    q, cache, bt, starts, kvs = batch(gen, dev, [300], [1], 8, 2, 128, 16, torch.float16, "v023")
    lens, counts = [300, 17, 120, 1], [2, 3, 1, 1]
    q = torch.randn(7, 8, 128, generator=gen).to(torch.float16)
    starts = torch.tensor([0, 2, 5, 6, 7], dtype=torch.int32)
    got = decode_drafts(q.to(dev), cache, bt.to(dev).expand(4, -1),
                        torch.tensor(lens, dtype=torch.int32, device=dev), starts.to(dev), 3,
                        scale_for(128), with_lse=True)
    check(got, q, counts, [tuple(x[:n] for x in kvs[0]) for n in lens], scale_for(128), torch.float16)


def test_a_table_past_4_gib(dev):
    n, rot = (1 << 23) - 3, 256
    table = rope_table(n, rot, base=1e6, scaling=YARN, device=dev)
    rows = [0, 1, 4194303, 4194304, n - 2, n - 1]
    want, angle, a = wanted(rows, rot, 1e6, YARN, n)
    got = table[torch.tensor(rows, device=dev)].cpu().double()
    assert ((got - want).abs() <= a * (7e-8 + 2.0 ** -50 * angle) + 2.0 ** -24 * want.abs()).all()
