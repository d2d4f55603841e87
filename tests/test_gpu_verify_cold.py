"""GPU: ``verify_drafts`` at temperatures next to 0 (and at none, and without end), where
equal and almost equal largest entries share all the weight; tokens equal to those of
the definition in 64 bits."""

import pytest
import torch

from hcp_vllm_plugin_amd import verify_drafts
from tests._drafts_util import check_verified, verify

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")
# (a vocabulary, sequences): one workgroup to a sequence; step 2 in those of the sums; step 2
# by itself
SIZES = [(600, 24), (20000, 24), (70001, 48)]
COLD = [1e-5, 1e-6, 1e-7, 1e-8, 1e-9, 3e-10, 1e-12, 1e-20, 1e-30, 1e-37, 1e-39, 2e-45]


def compare(dev, c):
    want = verify(c["target"], c["tokens"], c["query_start_loc"], c["uniform"], c["draft_probs"],
                  c["temperature"], c.get("probs", False))
    got = verify_drafts(**{k: x.to(dev) if isinstance(x, torch.Tensor) else x for k, x in c.items()})
    check_verified(got, want, c["uniform"].shape[1])
    return want


def below(x, dtype):
    """The next entry of the type below x > 0."""
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    return (torch.tensor([x], dtype=dtype).view(bits) - 1).view(dtype)[0]


def ties(gen, v, seqs, dtype, q, temperatures, tops):
    """Sequences of a draft each, its row of one to three equal largest entries and as many
    one step below them; the draft one of either, the random number either side of what it
    takes."""
    x = torch.randn(2 * seqs, v, generator=gen) - 6
    tokens = torch.zeros(2 * seqs, dtype=torch.int64)
    u = torch.rand(seqs, 2, generator=gen)
    dp = torch.full((seqs, 1, v), 1 / v)
    x = x.to(dtype)
    for b in range(seqs):
        k, top = 1 + b % 3, torch.tensor(tops[b % len(tops)], dtype=dtype)
        at = torch.randperm(v, generator=gen)[:2 * k]
        for r in (2 * b, 2 * b + 1):
            x[r, at[:k]] = top
            x[r, at[k:]] = below(float(top), dtype)
        tokens[2 * b + 1] = at[0] if b % 4 else at[k]
        u[b, 0] = (1 / k + (1e-3 if b % 2 else -1e-3)) if b % 8 else 0.5
        dp[b, 0, tokens[2 * b + 1]] = 1.0
    u.clamp_(0, 1 - 2 ** -24)
    t = torch.tensor([temperatures[b % len(temperatures)] for b in range(seqs)])
    return dict(target=x, tokens=tokens, query_start_loc=torch.arange(0, 2 * seqs + 1, 2), uniform=u,
                draft_probs=dp if q else None, temperature=t)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [True, False])
@pytest.mark.parametrize("v,seqs", SIZES)
def test_equal_and_almost_equal_entries(dev, dtype, q, v, seqs):
    gen = torch.Generator().manual_seed(v)
    tops = (30.375, 20.125, 8.0, 39.75, 20.1, 1.5, 12.3)
    for shift in range(0, len(COLD), 3):  # (every top and number of ties at each temperature)
        for turn in range(3):
            some = COLD[shift:shift + 3]
            c = ties(gen, v, seqs, dtype, q, some[turn:] + some[:turn], tops[turn:] + tops[:turn])
            want = compare(dev, c)
            assert {len(w) for w in want} == {1, 2}  # refused and accepted ones


@pytest.mark.parametrize("v,seqs", SIZES)
def test_two_entries_at_a_very_low_temperature(dev, v, seqs):
    """p = 1/2 of each: refused at 0.9, accepted at 0.4; one step below the largest (p =
    10^-83 in float32): refused."""
    x = torch.full((2 * seqs, v), 3.0)
    x[:, [0, v - 1]] = 30.375
    x[:, v // 2] = below(30.375, torch.float32)
    for t in COLD[3:]:
        for u, token, kept in ((0.9, 0, False), (0.4, 0, True), (0.5, v // 2, False),
                               (1e-6, v // 2, False)):
            c = dict(target=x, tokens=torch.tensor([0, token] * seqs),
                     query_start_loc=torch.arange(0, 2 * seqs + 1, 2),
                     uniform=torch.tensor([[u, 0.3]] * seqs), draft_probs=None,
                     temperature=torch.full((seqs,), t))
            want = compare(dev, c)
            assert all((len(w) == 2) == kept for w in want), (t, u, token)


@pytest.mark.parametrize("v,seqs", SIZES)
def test_entries_of_any_size(dev, v, seqs):
    """The type's lowest and largest value in one row, at a temperature of as much and at
    an infinite one; subnormal entries at subnormal temperatures."""
    big = torch.finfo(torch.float32).max
    for low, high, t in ((-big, big, 3e38), (-big, big, INF), (-big, big, 1e38), (1e-40, 2e-40, 1e-40),
                         (0.0, 1e-43, 2e-43), (-1e-40, 1e-40, 3e-41), (0.0, 1e-40, 1e-36)):
        x = torch.full((2 * seqs, v), low)
        x[:, ::2] = high
        for u in (0.2, 0.9):
            for token in (0, 1):  # a share of w / Z each, times v
                dp = torch.full((seqs, 1, v), 1.5 / v)
                c = dict(target=x, tokens=torch.tensor([0, token] * seqs),
                         query_start_loc=torch.arange(0, 2 * seqs + 1, 2),
                         uniform=torch.tensor([[u, 0.3]] * seqs), draft_probs=dp,
                         temperature=torch.full((seqs,), t))
                compare(dev, c)
