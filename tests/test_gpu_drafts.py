"""GPU: attention of several tokens to a sequence over a paged cache
(``decode_drafts``) against the same values in 64 bits."""

import pytest
import torch

from hcp_vllm_plugin_amd import decode_drafts, decode_fp4, merge_attn_states
from hcp_vllm_plugin_amd.kv_cache import fp4_cache_shape, reshape_and_cache
from tests import _fp4_util as f4
from tests._drafts_util import KINDS, batch, check, empty_cache, slots_of
from tests._util import randn, scale_for

pytestmark = pytest.mark.gpu

LENS = [1, 2, 15, 16, 17, 31, 32, 33, 0, 100, 129, 511, 3, 700]
COUNTS = [1, 2, 1, 4, 5, 3, 1, 5, 2, 0, 5, 4, 5, 3]


def run(dev, b, lens, most, scale, **kw):
    q, cache, bt, starts, kvs = b
    t = torch.tensor(lens, dtype=torch.int32, device=dev)
    return decode_drafts(q.to(dev), cache, bt.to(dev), t, starts.to(dev), most, scale,
                         with_lse=True, **kw)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hkv,d,bs", [(28, 4, 128, 16), (14, 2, 64, 16), (16, 8, 256, 32),
                                        (6, 6, 96, 64), (40, 2, 32, 16), (5, 1, 160, 128),
                                        (33, 1, 192, 16)])
def test_ragged(dev, kind, dtype, h, hkv, d, bs):
    gen = torch.Generator().manual_seed(h * d)
    b = batch(gen, dev, LENS, COUNTS, h, hkv, d, bs, dtype, kind)
    check(run(dev, b, LENS, 5, scale_for(d)), b[0], COUNTS, b[4], scale_for(d), dtype)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group", [1, 4, 7, 16])
@pytest.mark.parametrize("most", [1, 2, 3, 8, 17, 64])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_tokens_and_groups(dev, kind, group, most, d):
    """Every number of tiles to a workgroup, and chunks of rows past them."""
    gen = torch.Generator().manual_seed(group * most + d)
    lens, counts = [most + 40, 70, 200], [most, min(most, 3), (most + 1) // 2]
    b = batch(gen, dev, lens, counts, 2 * group, 2, d, 16, torch.bfloat16, kind)
    check(run(dev, b, lens, most, scale_for(d)), b[0], counts, b[4], scale_for(d), torch.bfloat16)


@pytest.mark.parametrize("kind", ["v031", "v023"])
@pytest.mark.parametrize("bs", [1, 2, 4, 8])
@pytest.mark.parametrize("d", [64, 128, 200])
def test_small_blocks(dev, kind, bs, d):
    gen = torch.Generator().manual_seed(bs + d)
    b = batch(gen, dev, LENS, COUNTS, 8, 2, d, bs, torch.float16, kind)
    check(run(dev, b, LENS, 5, scale_for(d)), b[0], COUNTS, b[4], scale_for(d), torch.float16)
    got = run(dev, b, LENS, 5, scale_for(d), window=20)
    check(got, b[0], COUNTS, b[4], scale_for(d), torch.float16, 20)


@pytest.mark.parametrize("d", [8, 24, 72, 136, 248])
def test_head_dims(dev, d):
    gen = torch.Generator().manual_seed(d)
    b = batch(gen, dev, LENS, COUNTS, 6, 3, d, 16, torch.bfloat16, "v031")
    check(run(dev, b, LENS, 5, scale_for(d)), b[0], COUNTS, b[4], scale_for(d), torch.bfloat16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,counts", [([1], [1]), ([2000], [4]), ([9000], [6]), ([20000, 3], [2, 3]),
                                         ([0], [1]), ([0, 0, 5], [3, 0, 2])])
@pytest.mark.parametrize("h,hkv,d", [(28, 4, 128), (16, 8, 256), (14, 2, 64)])
def test_few_sequences(dev, kind, lens, counts, h, hkv, d):
    gen = torch.Generator().manual_seed(sum(lens) + d)
    b = batch(gen, dev, lens, counts, h, hkv, d, 16, torch.bfloat16, kind)
    q, cache, bt, starts, kvs = b
    t = torch.tensor(lens, dtype=torch.int64, device=dev)
    args = (q.to(dev), cache, bt.to(dev), t, starts.long().to(dev), 6, scale_for(d))
    got = decode_drafts(*args, with_lse=True)
    check(got, q, counts, kvs, scale_for(d), torch.bfloat16)
    assert torch.equal(decode_drafts(*args), got[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 2, 16, 31, 33, 100, 5000, 1 << 40])
def test_window(dev, kind, window):
    gen = torch.Generator().manual_seed(window)
    lens, counts = [1, 17, 40, 64, 333, 1000, 2500], [1, 5, 8, 1, 7, 8, 3]
    b = batch(gen, dev, lens, counts, 28, 4, 128, 16, torch.bfloat16, kind)
    got = run(dev, b, lens, 8, scale_for(128), window=window)
    check(got, b[0], counts, b[4], scale_for(128), torch.bfloat16, window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", KINDS)
def test_rising_scores(dev, kind, dtype):
    """Scores that rise by more than 2^8 from one 32 keys to the next, and a late spike."""
    gen = torch.Generator().manual_seed(21)
    n, h, d = 700, 4, 64
    k = torch.zeros(n, 2, d)
    k[:, 0, 0] = torch.arange(n) * 0.25
    k[650, 1, 0] = 60.0
    k[:, :, 1:] = torch.randn(n, 2, d - 1, generator=gen) * 0.25
    k, v = k.to(dtype), randn(gen, (n, 2, d), dtype)
    cache = empty_cache(kind, 45, 2, 16, d, dtype, dev)
    reshape_and_cache(k.to(dev), v.to(dev), cache, torch.arange(n, device=dev))
    q = torch.randn(4, h, d, generator=gen) * 0.25
    q[:, :, 0] = 8.0
    q = q.to(dtype)
    kvs = [(f4.stand_for(k), f4.stand_for(v)) if kind == "fp4" else (k.double(), v.double())]
    got = decode_drafts(q.to(dev), cache, torch.arange(45, dtype=torch.int32, device=dev)[None],
                        torch.tensor([n], dtype=torch.int32, device=dev),
                        torch.tensor([0, 4], dtype=torch.int32, device=dev), 4, 0.5, with_lse=True)
    check(got, q, [4], kvs, 0.5, dtype)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [None, 40])
def test_what_a_row_does_not_see(dev, kind, d, window):
    """Whatever stands past a sequence's last key, before its windows and in blocks that no
    table names: the result is the same."""
    gen = torch.Generator().manual_seed(3)
    lens, counts = [1, 5, 18, 47, 300], [1, 4, 3, 4, 4]
    b = batch(gen, dev, lens, counts, 28, 4, d, 16, torch.bfloat16, kind)
    q, cache, bt, starts, kvs = b
    want = run(dev, b, lens, 4, scale_for(d), window=window)
    check(want, q, counts, kvs, scale_for(d), torch.bfloat16, window)
    dirty = torch.full_like(cache, 255 if kind == "fp4" else float("nan"))
    reach = [(n, n if window is None else min(n, window + c - 1)) for n, c in zip(lens, counts)]
    slots = torch.cat([slots_of(bt[r], torch.arange(n - m, n), 16) for r, (n, m) in enumerate(reach)])
    k, v = (torch.cat([x[i][n - m:] for x, (n, m) in zip(kvs, reach)]).to(torch.bfloat16)
            for i in (0, 1))
    reshape_and_cache(k.to(dev), v.to(dev), dirty, slots.to(dev))  # (a code's value has that code)
    got = run(dev, (q, dirty, bt, starts, kvs), lens, 4, scale_for(d), window=window)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [70, 200, 96])
def test_later_tokens_do_not_reach_earlier_ones(dev, kind, d, n):
    """NaN and infinities in K and V of drafted tokens: rows before them are as without,
    rows that see them are not finite."""
    gen = torch.Generator().manual_seed(4)
    b = batch(gen, dev, [n], [6], 14, 2, d, 16, torch.bfloat16, kind)
    q, cache, bt, starts, kvs = b
    want = run(dev, b, [n], 6, scale_for(d))
    one = torch.zeros(1, 2, d, dtype=torch.bfloat16)
    for is_v in (False, True):
        for bad in (float("nan"), float("inf"), float("-inf")):
            spoilt = cache.clone()
            x = one.clone()
            x[0, 0, 5] = bad
            slot = slots_of(bt[0], torch.tensor([n - 3]), 16)  # token 3's own key
            reshape_and_cache((one if is_v else x).to(dev), (x if is_v else one).to(dev), spoilt,
                              slot.to(dev))
            out, lse = run(dev, (q, spoilt, bt, starts, kvs), [n], 6, scale_for(d))
            assert torch.equal(out[:3], want[0][:3]) and torch.equal(lse[:, :3], want[1][:, :3])
            # the other KV head's rows have a key of zeros there
            assert torch.isfinite(out[:, 7:].float()).all()
            if is_v:
                col = out[3:, :7, 5].float().cpu()
                assert not torch.isfinite(col).any(), (bad, col)
                if kind != "fp4":  # (whose 32 columns are NaN)
                    assert torch.isnan(col).all() if bad != bad else (col == bad).all()
                    rest = torch.arange(d) != 5
                    assert torch.isfinite(out[3:, :7][..., rest.to(dev)].float()).all()
                assert torch.isfinite(lse).all()
            elif bad != bad or kind == "fp4":
                assert torch.isnan(out[3:, :7].float()).all() and torch.isnan(lse[:7, 3:]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_nan_in_the_context(dev, kind):
    """A NaN value far behind the tokens: its columns of every row; an infinite one too."""
    gen = torch.Generator().manual_seed(5)
    b = batch(gen, dev, [900], [3], 8, 2, 64, 16, torch.float16, kind)
    q, cache, bt, starts, kvs = b
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    x[0, 0, 40] = float("inf")
    reshape_and_cache(torch.zeros_like(x).to(dev), x.to(dev), cache,
                      slots_of(bt[0], torch.tensor([100]), 16).to(dev))
    out, lse = run(dev, b, [900], 3, scale_for(64))
    assert torch.isfinite(lse).all() and torch.isfinite(out[:, 4:].float()).all()
    assert not torch.isfinite(out[:, :4, 40].float()).any()
    assert torch.isfinite(out[:, :4, :32].float()).all()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_are_not_run(dev, kind):
    """Rows of no sequence, tokens past max_tokens and rows past q are left as they were;
    a strided q and out."""
    gen = torch.Generator().manual_seed(7)
    lens, counts = [50, 200, 90], [2, 9, 3]
    b = batch(gen, dev, lens, counts, 4, 2, 64, 16, torch.float16, kind)
    q, cache, bt, starts, kvs = b
    qd = torch.zeros(20, 9, 64, dtype=torch.float16, device=dev)
    qd[3:17, 2:6] = q.to(dev)
    hold = torch.full((20, 6, 64), 7.0, dtype=torch.float16, device=dev)
    t = torch.tensor(lens, dtype=torch.int32, device=dev)
    out, lse = decode_drafts(qd[:, 2:6], cache, bt.to(dev), t, (starts + 3).to(dev), 9, scale_for(64),
                             out=hold[:, 1:5], with_lse=True)
    check((out[3:17], lse[:, 3:17]), q, counts, kvs, scale_for(64), torch.float16)
    assert (hold[:3] == 7).all() and (hold[17:] == 7).all()
    assert (hold[:, 0] == 7).all() and (hold[:, 5] == 7).all()
    # four tokens at most: of nine the first four, as if the last five did not exist
    hold.fill_(7.0)
    decode_drafts(qd[:, 2:6], cache, bt.to(dev), t - torch.tensor([0, 5, 0], device=dev,
                                                                 dtype=torch.int32),
                  (starts + 3).to(dev), 4, scale_for(64), out=hold[:, 1:5])
    assert (hold[9:14] == 7).all() and not (hold[5:9, 1:5] == 7).all(-1).any()
    # starts that lie outside q, fall, or are negative
    for s in ([18, 25, 25, 30], [5, 3, 2, 1], [-4, -2, -2, 0], [30, 40, 50, 60]):
        hold.fill_(7.0)
        decode_drafts(qd[:, 2:6], cache, bt.to(dev), t, torch.tensor(s, dtype=torch.int32, device=dev),
                      9, scale_for(64), out=hold[:, 1:5])
        ran = (hold != 7).any(-1).any(-1).nonzero().flatten().tolist()
        assert ran == ([18, 19] if s[0] == 18 else []), (s, ran)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [None, 40])
def test_the_first_tokens_of_many(dev, kind, window):
    """max_tokens below a sequence's tokens, and rows past q: those that run see what they
    would with the others beside them."""
    gen = torch.Generator().manual_seed(13)
    lens, counts = [300, 200, 30, 5, 90], [9, 3, 5, 7, 6]
    q, cache, bt, starts, kvs = batch(gen, dev, lens, counts, 8, 2, 64, 16, torch.bfloat16, kind)
    for most, rows in ((4, 30), (9, 26), (1, 30)):
        out, lse = decode_drafts(q[:rows].to(dev), cache, bt.to(dev),
                                 torch.tensor(lens, dtype=torch.int32, device=dev), starts.to(dev),
                                 most, scale_for(64), window=window, with_lse=True)
        for r, n in enumerate(counts):
            ran, at = min(n, most, max(0, rows - int(starts[r]))), int(starts[r])
            left = max(0, lens[r] - (n - ran))  # (five keys of seven tokens: the first see none)
            kv = tuple(x[:left] for x in kvs[r])
            check((out[at:at + ran], lse[:, at:at + ran]), q[at:at + ran], [ran], [kv], scale_for(64),
                  torch.bfloat16, window)


@pytest.mark.parametrize("kind", KINDS)
def test_lengths_past_the_table_and_ids_past_the_cache(dev, kind):
    gen = torch.Generator().manual_seed(6)
    b = batch(gen, dev, [64, 64], [3, 2], 8, 2, 128, 16, torch.bfloat16, kind)
    q, cache, bt, starts, kvs = b
    got = run(dev, b, [64 + 999, -3], 3, scale_for(128))
    check(got, q, [3, 2], [kvs[0], (kvs[1][0][:0], kvs[1][1][:0])], scale_for(128), torch.bfloat16)
    wild, last = bt.clone(), bt.clone()
    wild[0, 2], wild[1, 1] = 1 << 30, -5  # either reads the last block
    last[0, 2] = last[1, 1] = cache.shape[0] - 1
    a, c = (run(dev, (q, cache, x, starts, kvs), [64, 64], 3, scale_for(128)) for x in (wild, last))
    assert torch.equal(a[0], c[0])


@pytest.mark.parametrize("kind", KINDS)
def test_far_blocks(dev, kind):
    """Keys more than 4 GiB into the cache."""
    gen = torch.Generator().manual_seed(8)
    h, hkv, d, bs = 16, 8, 128, 16
    row = fp4_cache_shape(1, hkv, bs, d)[3] if kind == "fp4" else 4 * d
    nb = (5 << 30) // (hkv * bs * row)
    cache = empty_cache(kind, nb, hkv, bs, d, torch.bfloat16, dev)
    bt = torch.tensor([[nb - 1, 0, nb // 2, nb - 2]], dtype=torch.int32)
    k, v = (randn(gen, (60, hkv, d), torch.bfloat16) for _ in "kv")
    reshape_and_cache(k.to(dev), v.to(dev), cache, slots_of(bt[0], torch.arange(60), bs).to(dev))
    q = randn(gen, (4, h, d), torch.bfloat16)
    kv = (f4.stand_for(k), f4.stand_for(v)) if kind == "fp4" else (k.double(), v.double())
    got = decode_drafts(q.to(dev), cache, bt.to(dev), torch.tensor([60], device=dev),
                        torch.tensor([0, 4], device=dev), 4, scale_for(d), with_lse=True)
    check(got, q, [4], [kv], scale_for(d), torch.bfloat16)


def test_a_strided_cache(dev):
    """Blocks of a larger tensor, and heads of a cache that holds more."""
    gen = torch.Generator().manual_seed(9)
    lens, counts = [40, 90], [4, 2]
    q, cache, bt, starts, kvs = b = batch(gen, dev, lens, counts, 4, 2, 64, 16, torch.bfloat16, "v031")
    wide = torch.full((cache.shape[0], 5, 16, 128), float("nan"), dtype=torch.bfloat16, device=dev)
    wide[:, 1:3] = cache
    want = run(dev, b, lens, 4, scale_for(64))
    got = run(dev, (q, wide[:, 1:3], bt, starts, kvs), lens, 4, scale_for(64))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kind", ["v031", "fp4"])
def test_many_sequences(dev, kind):
    """More than one launch takes."""
    gen = torch.Generator().manual_seed(10)
    lens = [1 + (i * 37) % 70 for i in range(1100)]
    counts = [i % 4 for i in range(1100)]
    b = batch(gen, dev, lens, counts, 4, 2, 64, 16, torch.float16, kind)
    check(run(dev, b, lens, 3, scale_for(64)), b[0], counts, b[4], scale_for(64), torch.float16)


@pytest.mark.parametrize("kind", KINDS)
def test_captured_and_replayed(dev, kind):
    """Two graphs over one cache, lengths and rows changed between replays, eager calls in
    between."""
    gen = torch.Generator().manual_seed(11)
    q, cache, bt, starts, kvs = batch(gen, dev, [300, 500, 64], [4, 3, 5], 28, 4, 128, 16,
                                      torch.bfloat16, kind)
    qd, btd, sd = q.to(dev), bt.to(dev), starts.to(dev)
    lens = [torch.tensor(x, dtype=torch.int32, device=dev) for x in ([300, 500, 64], [1, 33, 0])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode_drafts(qd, cache, btd, lens[0], sd, 5, scale_for(128))
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for t in lens:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = decode_drafts(qd, cache, btd, t, sd, 5, scale_for(128), with_lse=True)
        graphs.append((g, t, out))
    for step in range(4):
        sd.copy_(torch.tensor([0, 4 - step, 7, 12], dtype=torch.int32))
        for g, t, out in graphs:
            t.copy_(torch.tensor([300 - 70 * step, 500 - step, 64 - 20 * step], dtype=torch.int32))
            g.replay()
            eager = decode_drafts(qd, cache, btd, t, sd, 5, scale_for(128), with_lse=True)
            torch.cuda.synchronize()
            ran = torch.ones(12, dtype=torch.bool)
            ran[4 - step + 5:7] = False  # tokens past the fifth of the second sequence
            assert torch.equal(out[0][ran], eager[0][ran]), step
            assert torch.equal(out[1][:, ran], eager[1][:, ran]), step


@pytest.mark.parametrize("kind", KINDS)
def test_two_streams(dev, kind):
    gen = torch.Generator().manual_seed(12)
    b = batch(gen, dev, [900, 200], [4, 2], 28, 4, 128, 16, torch.bfloat16, kind)
    q, cache, bt, starts, kvs = b
    args = (q.to(dev), cache, bt.to(dev), torch.tensor([900, 200], device=dev),
            starts.long().to(dev), 4, scale_for(128))
    want = decode_drafts(*args)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(decode_drafts(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_single_tokens_as_decode_fp4(dev):
    """One token to a sequence is what ``decode_fp4`` runs; both against 64 bits."""
    gen = torch.Generator().manual_seed(13)
    lens = [5, 700, 64]
    q, cache, bt, starts, kvs = b = batch(gen, dev, lens, [1, 1, 1], 28, 4, 128, 16, torch.bfloat16,
                                          "fp4")
    check(run(dev, b, lens, 1, scale_for(128)), q, [1, 1, 1], kvs, scale_for(128), torch.bfloat16)
    t = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = decode_fp4(q.to(dev), cache, bt.to(dev), t, scale_for(128), with_lse=True)
    check(got, q, [1, 1, 1], kvs, scale_for(128), torch.bfloat16)


def test_merged_with_staged_keys(dev):
    """The local keys' result and that of keys held elsewhere, merged by their LSE, are the
    attention over both."""
    gen = torch.Generator().manual_seed(14)
    n, c, far = 80, 3, 50
    q, cache, bt, starts, kvs = b = batch(gen, dev, [n], [c], 8, 2, 64, 16, torch.bfloat16, "v031")
    k, v = (randn(gen, (far, 2, 64), torch.bfloat16) for _ in "kv")
    from hcp_vllm_plugin_amd import ring_attn_with_lse
    po, pl = ring_attn_with_lse(q.to(dev), k.to(dev), v.to(dev), scale_for(64), None)
    so, sl = run(dev, b, [n], c, scale_for(64))
    out = torch.empty_like(so)
    merge_attn_states(out, po, pl, so, sl)
    lk, lv = kvs[0]
    want, _ = f4.attend(q, torch.cat([k.double(), lk]), torch.cat([v.double(), lv]), scale_for(64),
                        first=far + n - c)
    # three roundings to bf16 of a value, and P of the far pass rounded to bf16 (2^-8 of the
    # largest value)
    tol = 2.0 ** -8 * (3 * want.abs() + torch.cat([v.double(), lv]).abs().max())
    assert ((out.cpu().double() - want).abs() <= tol).all()


def placed(dev, kind, k, v, dtype, kv=None):
    """One sequence with these keys and values: (cache, table, what they (or kv) stand for)."""
    n, hkv, d = k.shape
    nb = -(-n // 16) + 1
    cache = empty_cache(kind, nb, hkv, 16, d, dtype, dev)
    reshape_and_cache(k.to(dev), v.to(dev), cache, torch.arange(n, device=dev))
    k, v = kv or (k, v)
    kv = (f4.stand_for(k), f4.stand_for(v)) if kind == "fp4" else (k.double(), v.double())
    return cache, torch.arange(nb, dtype=torch.int32, device=dev)[None], kv


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", KINDS)
def test_many_small_weights(dev, kind, dtype):
    """A key in the first 32 of each wave far above 32764 others, 2^-14 of it each:
    together they weigh half as much, so a bias of their weights shows.  (As many KV
    heads, with the same keys, as leave a workgroup to each.)"""
    gen, n, heads = torch.Generator().manual_seed(17), 32768, 512
    k = (torch.randn(n, 1, 32, generator=gen) * 0.05).to(dtype)
    v = (1 + 0.1 * torch.randn(n, 1, 32, generator=gen)).to(dtype)
    k[5:128:32], v[5:128:32] = 0.375, -1.0
    q = torch.ones(2, heads, 32, dtype=dtype)
    cache, bt, kv = placed(dev, kind, k.to(dev).expand(n, heads, 32), v.to(dev).expand(n, heads, 32),
                           dtype, (k, v))
    out, lse = decode_drafts(q.to(dev), cache, bt, torch.tensor([n], device=dev),
                             torch.tensor([0, 2], device=dev), 2, 0.81, with_lse=True)
    assert (out == out[:, :1]).all() and (lse == lse[:1]).all()
    check((out[:, :1], lse[:1]), q[:, :1], [2], [kv], 0.81, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["v031", "fp4"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("slope", [0.01, 0.04, -0.04, 0.3, 3.0])
def test_scores_that_rise_and_fall(dev, kind, dtype, d, slope):
    """Scores (of half of the query heads) that climb by ``slope`` a key, past the
    maximum so far by less or by more than it is let stand, or fall."""
    gen = torch.Generator().manual_seed(d)
    n = 900
    k = randn(gen, (n, 2, d), dtype) * 0.1
    k[:, :, :32] = (slope * torch.arange(n) / 32)[:, None, None].to(dtype)
    v = randn(gen, (n, 2, d), dtype)
    q = randn(gen, (3, 8, d), dtype)
    q[:, ::2, :32] = 1.0
    cache, bt, kv = placed(dev, kind, k.to(dtype), v, dtype)
    got = decode_drafts(q.to(dev), cache, bt, torch.tensor([n], device=dev),
                        torch.tensor([0, 3], device=dev), 3, 1.0, with_lse=True)
    check(got, q, [3], [kv], 1.0, dtype)


def test_rows_of_out_on_top_of_each_other_are_refused(dev):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev)
    cache = torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16, device=dev)
    bt, lens = torch.zeros(2, 1, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int64, device=dev)
    starts = torch.tensor([0, 1, 2], device=dev)
    room = torch.zeros(4096, dtype=torch.bfloat16, device=dev)
    for strides in ((255, 64, 1), (256, 63, 1), (64, 127, 1), (0, 64, 1), (256, 0, 1)):
        with pytest.raises(ValueError, match="out"):
            decode_drafts(q, cache, bt, lens, starts, 1, 0.1, out=room.as_strided((2, 4, 64), strides))
    heads_first = room.as_strided((2, 4, 64), (64, 128, 1))
    assert decode_drafts(q, cache, bt, lens, starts, 1, 0.1, out=heads_first) is heads_first
    assert decode_drafts(q[:0], cache, bt, lens, starts, 1, 0.1).shape == (0, 4, 64)
    assert decode_drafts(q, cache, bt, lens[:0], starts[:1], 1, 0.1).shape == (2, 4, 64)
