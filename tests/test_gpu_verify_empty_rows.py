"""GPU: ``verify_drafts`` where the row that judges a draft has no entry: no draft is
accepted there, token 0 neither."""

import pytest
import torch

from tests.test_gpu_verify_cold import DTYPES, INF, SIZES, compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("v,seqs", SIZES)
@pytest.mark.parametrize("last", [0, 1])
def test_rows_without_entries(dev, dtype, probs, v, seqs, last):
    """Greedy and drawn sequences, the first or the second draft's row of nothing but -inf
    or NaN; the drafts token 0."""
    gen = torch.Generator().manual_seed(v)
    x = torch.randn(3 * seqs, v, generator=gen)
    if probs:
        x = torch.softmax(x, -1)
    x = x.to(dtype)
    x[:, 0] = 20.0  # token 0 where there are entries
    for b in range(seqs):
        x[3 * b + last] = -INF if b % 2 else float("nan")
    t = torch.tensor([0.0, 0.0, 1.0, -1.0, float("nan")] * seqs)[:seqs]
    c = dict(target=x, tokens=torch.zeros(3 * seqs, dtype=torch.int64),
             query_start_loc=torch.arange(0, 3 * seqs + 1, 3),
             uniform=torch.rand(seqs, 3, generator=gen) * 0.5, draft_probs=None, temperature=t,
             probs=probs)
    want = compare(dev, c)
    greedy = ~(t > 0)
    assert all(len(w) == last for w, g in zip(want, greedy) if g)
