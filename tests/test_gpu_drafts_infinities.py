"""GPU: ``decode_drafts`` over keys with an infinity that every row scores -inf: they have
no weight, at head dims that the kernel pads too."""

import pytest
import torch

from hcp_vllm_plugin_amd import decode_drafts
from tests._drafts_util import empty_cache
from tests._util import randn, scale_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["v031", "v023"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [8, 24, 64, 72, 96, 128, 136, 160, 200, 248, 256])
@pytest.mark.parametrize("bs", [1, 4, 8, 16, 64])
def test_keys_that_score_minus_infinity(dev, kind, dtype, d, bs):
    """The same as with the lowest finite score, whose weight is 0; a sequence of nothing
    else gets 0 and an LSE of -inf."""
    from hcp_vllm_plugin_amd.kv_cache import reshape_and_cache

    gen = torch.Generator().manual_seed(d * bs)
    n, far = 150, [0, 3, 40, 70, 149]
    q = randn(gen, (4, 8, d), dtype)
    k, v = randn(gen, (n, 2, d), dtype), randn(gen, (n, 2, d), dtype)
    alone = 5  # keys of a second sequence, all with an infinity
    for at in {0, 7, d - 1}:  # the row's first 16 bytes, and its last
        qa, ka, kb = q.clone(), k.clone(), k.clone()
        qa[:, :, at] = -1.0
        ka[far, :, at] = float("inf")
        kb[far, :, at] = torch.finfo(dtype).max / 2
        first = k[:alone].clone()
        first[:, :, at] = float("inf")
        outs = []
        for x in (ka, kb):
            nb = -(-n // bs) + -(-alone // bs)
            cache = empty_cache(kind, nb, 2, bs, d, dtype, dev)
            bt = torch.zeros(2, -(-n // bs), dtype=torch.int32)
            bt[0] = torch.arange(bt.shape[1])
            bt[1, :-(-alone // bs)] = torch.arange(bt.shape[1], nb)
            slots = torch.cat([torch.arange(n), bt.shape[1] * bs + torch.arange(alone)])
            reshape_and_cache(torch.cat([x, first]).to(dev), torch.cat([v, v[:alone]]).to(dev), cache,
                              slots.to(dev))
            outs.append(decode_drafts(qa.to(dev), cache, bt.to(dev), torch.tensor([n, alone], device=dev),
                                      torch.tensor([0, 2, 4], device=dev), 2, scale_for(d),
                                      with_lse=True))
        (a, la), (b, lb) = outs
        assert torch.isfinite(b[:2].float()).all()
        assert torch.equal(a, b) and torch.equal(la, lb)
        assert (a[2:] == 0).all() and (la[:, 2:] == float("-inf")).all()
