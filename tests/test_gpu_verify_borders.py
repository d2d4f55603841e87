"""GPU: ``verify_drafts`` with a draft within what the sums in 32 bits may be off by
(2.5e-6) of its border: accepted on one side of it, refused on the other."""

import pytest
import torch

from tests.test_gpu_verify_cold import DTYPES, SIZES, compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("v,seqs", SIZES)
def test_both_sides_of_a_border(dev, dtype, probs, v, seqs):
    """u q = p(d) (1 + off): u in 32 bits is off by 2^-24 of itself, 6e-8, the least offset
    5e-7.  q(d) = 2 p(d), so that nothing of d is left where it is refused."""
    gen = torch.Generator().manual_seed(v)
    x = torch.randn(seqs, v, generator=gen)
    x[:, 5] = 4.0
    x = (torch.softmax(x, -1) if probs else x).to(dtype)
    w = x.double() if probs else torch.exp(x.double() - x.double().amax(1, keepdim=True))
    p = w[:, 5] / w.sum(1)
    dp = torch.zeros(seqs, 1, v)
    dp[:, 0, 5] = 2 * p
    for off in (5e-7, 1e-6, 2e-6):
        side = torch.tensor([-1.0, 1.0] * seqs)[:seqs].double()
        u = torch.full((seqs, 2), 0.3)
        u[:, 0] = p * (1 + side * off) / dp[:, 0, 5].double()
        c = dict(target=x.repeat_interleave(2, 0), tokens=torch.tensor([0, 5] * seqs),
                 query_start_loc=torch.arange(0, 2 * seqs + 1, 2), uniform=u, draft_probs=dp,
                 temperature=None, probs=probs)
        want = compare(dev, c)
        assert [t[0] == 5 for t in want] == (side < 0).tolist()
