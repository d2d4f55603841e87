"""GPU: verification of drafted tokens (``verify_drafts``) against its definition in 64
bits; whole numbers, so equal."""

import pytest
import torch

from hcp_vllm_plugin_amd import verify_drafts
from tests._drafts_util import check_verified, verify

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


def case(gen, counts, v, dtype, most, q=True, probs=False, greedy=0.0, spread=2.0):
    """Targets of ``counts`` rows each and drafts drawn from a noisy copy of them."""
    t, s = sum(counts), len(counts)
    x = torch.randn(t, v, generator=gen) * spread
    starts = torch.tensor([0, *counts]).cumsum(0)
    tokens = torch.randint(0, v, (t,), generator=gen)
    dp = torch.zeros(s, max(most - 1, 1), v)
    for b, n in enumerate(counts):
        for i in range(min(n, most) - 1):
            row = int(starts[b]) + i
            dp[b, i] = torch.softmax(x[row] + torch.randn(v, generator=gen), 0)
            tokens[row + 1] = torch.multinomial(dp[b, i], 1, generator=gen)
            if torch.rand((), generator=gen) < 0.4:
                tokens[row + 1] = x[row].argmax()
    temperature = 0.5 + torch.rand(s, generator=gen)
    temperature[torch.rand(s, generator=gen) < greedy] = 0
    target = (torch.softmax(x, -1) if probs else x).to(dtype)
    return dict(target=target, tokens=tokens, query_start_loc=starts,
                uniform=torch.rand(s, most, generator=gen), draft_probs=dp if q else None,
                temperature=temperature, probs=probs)


def run(dev, c):
    return verify_drafts(**{k: x.to(dev) if isinstance(x, torch.Tensor) else x for k, x in c.items()})


def compare_(dev, c):
    want = verify(c["target"], c["tokens"], c["query_start_loc"], c["uniform"], c["draft_probs"],
                  c["temperature"], c["probs"])
    got = run(dev, c)
    assert got.tokens.dtype == c["tokens"].dtype and got.num_tokens.dtype == torch.int32
    check_verified(got, want, c["uniform"].shape[1])
    return want


compare = compare_


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [True, False])
@pytest.mark.parametrize("v", [1, 2, 7, 8, 9, 100, 2047, 2048, 2049, 8191, 8200, 50257])
def test_vocabularies(dev, dtype, q, v):
    gen = torch.Generator().manual_seed(v)
    want = compare(dev, case(gen, [1, 4, 5, 2, 3, 5, 4, 1, 5], v, dtype, 5, q=q, greedy=0.2))
    # (without q a draft is accepted with the target's probability, seldom in a large vocabulary)
    assert not q or any(len(w) > 1 for w in want)


@pytest.mark.parametrize("q", [True, False])
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("most", [1, 2, 3, 9, 64])
def test_drafts(dev, q, probs, most):
    gen = torch.Generator().manual_seed(most)
    counts = [1 + (i * 7) % most for i in range(12)]
    compare(dev, case(gen, counts, 1000, torch.float32, most, q=q, probs=probs, greedy=0.2))


@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("q", [True, False])
@pytest.mark.parametrize("v", [1, 9, 513, 8192, 9000, 33000, 65536, 65537])
def test_many_sequences(dev, v, q, probs):
    """As many as get a workgroup each, and vocabularies on either side of what one takes."""
    gen = torch.Generator().manual_seed(v)
    counts = [1 + i % 3 for i in range(70)]
    compare(dev, case(gen, counts, v, torch.float32, 3, q=q, probs=probs, greedy=0.2))
    flat = case(gen, [1] * 70, v, torch.bfloat16, 1, q=False, spread=0.0)
    flat["temperature"] = None
    compare(dev, flat)


def test_a_long_flat_row(dev):
    """150000 tokens of about the same weight: a sum in 32 bits would be off by whole
    tokens."""
    gen = torch.Generator().manual_seed(5)
    for q in (True, False):
        c = case(gen, [1, 2, 3, 2], 150001, torch.float32, 3, q=q, spread=0.01)
        compare(dev, c)


def test_rows_of_odd_places(dev):
    """Rows that begin at no multiple of 16 bytes, strided draft probabilities and
    uniforms, int32 tokens and starts, a padded batch."""
    gen = torch.Generator().manual_seed(6)
    for dtype in DTYPES:
        c = case(gen, [2, 4, 3], 1001, dtype, 4)
        c["tokens"], c["query_start_loc"] = c["tokens"].int(), c["query_start_loc"].int()
        want = verify(c["target"], c["tokens"], c["query_start_loc"], c["uniform"], c["draft_probs"],
                      c["temperature"])
        wide = torch.full((12, 1103), 50.0).to(dtype)
        wide[:9, 3:1004] = c["target"]
        dp = torch.full((3, 5, 1010), 9.0)
        dp[:, 1:4, 1:1002] = c["draft_probs"]
        u = torch.full((3, 7), 0.5)
        u[:, 2:6] = c["uniform"]
        tokens = torch.cat([c["tokens"], torch.full((3,), 7, dtype=torch.int32)])
        got = verify_drafts(wide.to(dev)[:, 3:1004], tokens.to(dev), c["query_start_loc"].to(dev),
                            u.to(dev)[:, 2:6], draft_probs=dp.to(dev)[:, 1:4, 1:1002],
                            temperature=c["temperature"].to(dev))
        assert got.tokens.dtype == torch.int32
        check_verified(got, want, 4)


def test_sequences_without_rows(dev):
    """Empty sequences, starts that fall or leave the target, more rows than max_tokens."""
    gen = torch.Generator().manual_seed(7)
    c = case(gen, [3, 3, 3, 3], 50, torch.float32, 3)
    for starts in ([0, 0, 3, 3, 12], [0, 3, 2, 9, 40], [-2, 1, 4, 12, 12], [12, 13, 14, 15, 16],
                   [0, 12, 12, 12, 12]):
        compare(dev, {**c, "query_start_loc": torch.tensor(starts)})


def test_equal_entries_go_to_the_lowest_index(dev):
    x = torch.zeros(4, 20000)
    x[0, [17, 19999, 8200]] = 3.0
    x[1, [9000, 12000]] = 1.0
    x[2, 5:] = 2.0
    tokens = torch.tensor([0, 17, 12000, 5])
    c = dict(target=x, tokens=tokens, query_start_loc=torch.tensor([0, 4]), uniform=torch.zeros(1, 4),
             draft_probs=None, temperature=torch.zeros(1), probs=False)
    assert compare(dev, c) == [[17, 9000]]
    c["tokens"] = torch.tensor([0, 17, 9000, 5])
    assert compare(dev, c) == [[17, 9000, 5, 0]]


def test_borders(dev):
    """Numbers that lie on a border: a draft is refused at equality, and a token begins
    where the sum before it equals u times the whole."""
    w = torch.tensor([1.0, 0.0, 1.0, 2.0, 0.0, 4.0]) / 8
    for u, want in ((0.0, 0), (0.125, 2), (0.25, 3), (0.5, 5), (0.4999, 3), (0.99999994, 5), (1.0, 5)):
        c = dict(target=w[None], tokens=torch.tensor([0]), query_start_loc=torch.tensor([0, 1]),
                 uniform=torch.tensor([[u]]), draft_probs=None, temperature=None, probs=True)
        assert compare(dev, c) == [[want]], u
    for u, first in ((0.5, None), (0.4999, 3), (0.0, 3)):  # p(3) = q(3) u at u = 1/2
        q = torch.tensor([0.0, 0.25, 0.25, 0.5, 0.0, 0.0])
        c = dict(target=torch.stack([w, w]), tokens=torch.tensor([0, 3]),
                 query_start_loc=torch.tensor([0, 2]), uniform=torch.tensor([[u, 0.0]]),
                 draft_probs=q[None, None], temperature=None, probs=True)
        got = compare(dev, c)
        assert got == ([[0]] if first is None else [[3, 0]]), (u, got)


def test_near_borders(dev):
    """Drafts within 32-bit sums' error of the border, on either side of it."""
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(1, 5000, generator=gen)
    w = torch.exp(x[0].double() - x.max().double())
    p = w / w.sum()
    d = int(x.argmax())
    q = torch.full((1, 1, 5000), 0.01)
    for off in (-3e-7, 3e-7):
        # u q = p(d) (1 + off), as near as 32-bit u comes: 2^-24 of it is 6e-8
        u = torch.tensor([[float(p[d] * (1 + off) / float(q[0, 0, d])), 0.3]])
        assert u[0, 0] < 1
        c = dict(target=x.expand(2, -1), tokens=torch.tensor([0, d]),
                 query_start_loc=torch.tensor([0, 2]), uniform=u, draft_probs=q, temperature=None,
                 probs=False)
        assert (compare(dev, c)[0][0] == d) == (off < 0) or off > 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [True, False])
@pytest.mark.parametrize("more", [0, 60])
def test_infinities_and_nan(dev, dtype, q, more):
    """Entries cut off by -inf or the type's lowest value, NaN, infinities; rows of
    nothing else.  With sequences of one row behind them, another kernel's share."""
    gen = torch.Generator().manual_seed(9)
    c = case(gen, [3] * 9 + [1] * more, 3000, dtype, 3, q=q)
    x = c["target"]
    x[0:3, 100:] = -INF
    x[3:6, 7:] = torch.finfo(dtype).min
    x[6:9, ::3] = float("nan")
    x[9] = -INF
    x[10:12] = float("nan")
    x[12:15, [5, 2999]] = INF
    x[15:18] = -INF
    x[15:18, 1234] = -5.0
    x[18:21, :] = torch.finfo(dtype).min
    x[22] = -INF
    x[24:27, 40] = torch.finfo(dtype).max
    for temperature in (None, torch.tensor([1.0, 0.0] * 4 + [0.25] + [1.0] * more)):
        for warm in (1.0, 1e-3, INF):
            t = None if temperature is None else temperature * warm
            t = t if t is None else torch.nan_to_num(t, nan=0.0, posinf=INF)
            compare(dev, {**c, "temperature": t})
    c["probs"] = True
    x[x == INF] = torch.finfo(dtype).max / 1e4
    compare(dev, {**c, "target": torch.where(x.abs() > 1e4, 0.5, x).to(dtype)})


def test_drafts_that_are_no_tokens(dev):
    gen = torch.Generator().manual_seed(10)
    for q in (True, False):
        c = case(gen, [3, 3, 3, 3], 64, torch.float32, 3, q=q)
        c["tokens"][[1, 4, 8, 11]] = torch.tensor([-1, 64, 1 << 40, -(1 << 40)])
        compare(dev, c)


@pytest.mark.parametrize("n", [1, 64])
def test_nothing_left_of_the_residual(dev, n):
    """q nowhere below p: the token is drawn from p itself."""
    def compare(dev, c):  # n sequences of the same
        many = {k: x.repeat(n, *[1] * (x.dim() - 1)) if isinstance(x, torch.Tensor) else x
                for k, x in c.items()}
        many["query_start_loc"] = torch.arange(0, 2 * n + 1, 2)
        want = compare_(dev, many)
        assert all(w == want[0] for w in want)
        return want[:1]

    p = torch.softmax(torch.arange(10.0), 0)
    for q, u in ((2 * p, 0.75), (torch.full((10,), INF), 0.5), (torch.full((10,), float("nan")), 0.5)):
        c = dict(target=p.expand(2, -1), tokens=torch.tensor([0, 9]), query_start_loc=torch.tensor([0, 2]),
                 uniform=torch.tensor([[u, 0.2]]), draft_probs=q[None, None], temperature=None,
                 probs=True)
        compare(dev, c)
    # one token has all the weight, and its draft is refused by u = 1
    one = torch.full((2, 10), -INF)
    one[:, 4] = 1.0
    c = dict(target=one, tokens=torch.tensor([0, 4]), query_start_loc=torch.tensor([0, 2]),
             uniform=torch.tensor([[1.0, 0.2]]), draft_probs=None, temperature=None, probs=False)
    assert compare(dev, c) == [[4]]


def test_tokens_are_as_the_target_draws_them(dev):
    """Over 40000 sequences with drafts from q, the first token's frequencies are p: within
    six deviations of a binomial count."""
    gen = torch.Generator().manual_seed(11)
    n, v = 40000, 8
    p = torch.softmax(torch.randn(v, generator=gen), 0)
    q = torch.softmax(torch.randn(v, generator=gen), 0)
    tokens = torch.zeros(n, 2, dtype=torch.int64)
    tokens[:, 1] = torch.multinomial(q, n, replacement=True, generator=gen)
    got = verify_drafts(p.expand(2 * n, v).contiguous().to(dev), tokens.view(-1).to(dev),
                        torch.arange(0, 2 * n + 1, 2, device=dev),
                        torch.rand(n, 2, generator=gen).to(dev),
                        draft_probs=q.expand(n, 1, v).contiguous().to(dev), probs=True)
    count = torch.bincount(got.tokens[:, 0].cpu(), minlength=v).double()
    assert ((count - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all()
    kept = (got.num_tokens == 2).double().mean().item()
    rate = float(torch.minimum(p, q).sum())
    assert abs(kept - rate) <= 6 * (rate * (1 - rate) / n) ** 0.5


def test_captured_replayed_and_on_two_streams(dev):
    gen = torch.Generator().manual_seed(12)
    cases = [case(gen, [4, 2, 1, 5], 9000, torch.bfloat16, 5, greedy=0.3) for _ in range(5)]
    d = {k: x.to(dev) if isinstance(x, torch.Tensor) else x for k, x in cases[0].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        verify_drafts(**d)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = verify_drafts(**d)
        graphs.append((g, out))
    for c in cases:
        for k, x in c.items():
            if isinstance(x, torch.Tensor):
                d[k].copy_(x)
        want = verify(c["target"], c["tokens"], c["query_start_loc"], c["uniform"], c["draft_probs"],
                      c["temperature"])
        for g, out in graphs:
            g.replay()
            check_verified(run(dev, c), want, 5)
            torch.cuda.synchronize()
            check_verified(out, want, 5)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(verify_drafts(**d))
    torch.cuda.synchronize()
    for o in outs:
        check_verified(o, want, 5)


@pytest.mark.parametrize("front,back", [(0, 40000), (33001, 0), (9000, 31000)])
@pytest.mark.parametrize("edges", [
    test_borders, test_near_borders, test_drafts_that_are_no_tokens, test_sequences_without_rows,
    test_equal_entries_go_to_the_lowest_index])
def test_edges_in_large_vocabularies(dev, monkeypatch, edges, front, back):
    """The same among tokens without weight, so many that a sequence's row takes several
    workgroups: the tokens of the small ones, `front` further on."""
    def wider(dev, c):
        pad = torch.nn.functional.pad
        more = {**c, "target": pad(c["target"], (front, back), value=0.0 if c["probs"] else -INF)}
        if c["draft_probs"] is not None:
            more["draft_probs"] = pad(c["draft_probs"], (front, back))
        d, v = c["tokens"], c["target"].shape[1]
        more["tokens"] = torch.where((d >= 0) & (d < v), d + front, torch.full_like(d, -1))
        want, small = compare_(dev, more), verify(
            c["target"], c["tokens"], c["query_start_loc"], c["uniform"], c["draft_probs"],
            c["temperature"], c["probs"])
        assert [[t - front for t in w] for w in want] == small
        return small

    monkeypatch.setitem(globals(), "compare", wider)
    edges(dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [True, False])
@pytest.mark.parametrize("v", [20000, 70001])
def test_infinities_and_nan_in_large_vocabularies(dev, dtype, q, v):
    gen = torch.Generator().manual_seed(13)
    c = case(gen, [3] * 9 + [1] * 3, v, dtype, 3, q=q)
    x = c["target"]
    x[0:3, 100:] = -INF
    x[3:6, :v - 7] = torch.finfo(dtype).min
    x[6:9, ::3] = float("nan")
    x[9] = -INF
    x[10:12] = float("nan")
    x[12:15, [5, v - 1]] = INF
    x[15:18] = -INF
    x[15:18, v - 1234] = -5.0
    x[18:21] = torch.finfo(dtype).min
    x[21:24, 8192:] = float("nan")
    compare(dev, c)
    c["temperature"][:] = 0
    compare(dev, c)
    if q:
        c["temperature"][:] = 0.9
        c["draft_probs"][0] = 0.0
        c["draft_probs"][1, :, ::2] = float("nan")
        compare(dev, c)


@pytest.mark.parametrize("v", [100, 3000, 40000])
def test_probabilities_of_any_size(dev, v):
    """Weights whose sum passes 32 bits' range, and subnormal ones."""
    for w in (3e38, 1e-42):
        x = torch.full((6, v), w)
        x[:, ::7] = 0.0
        x[2:4, 3] = w / 4
        dp = torch.full((3, 1, v), 1.0 / v)
        for u in (0.1, 0.9):
            c = dict(target=x, tokens=torch.tensor([0, 1, 0, 3, 0, 7]),
                     query_start_loc=torch.arange(0, 7, 2), uniform=torch.tensor([[u, 0.37]] * 3),
                     draft_probs=dp, temperature=None, probs=True)
            compare(dev, c)
            compare(dev, {**c, "draft_probs": None})
