"""GPU: single-token attention over the 4-bit cache (``decode_fp4``) against the
same values in 64 bits."""

import pytest
import torch

from hcp_vllm_plugin_amd import decode_fp4
from hcp_vllm_plugin_amd.kv_cache import fp4_cache_shape, reshape_and_cache
from tests import _fp4_util as f4
from tests._util import outlier_k, randn, scale_for

pytestmark = pytest.mark.gpu


def batch(gen, dev, lens, h, hkv, d, bs, dtype, spare=2, width=0):
    """Keys of sequences of ``lens``, written into a cache through a shuffled table:
    (q, cache, table, [(k, v) as the cache stands for them])."""
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + spare
    ids = torch.randperm(nb, generator=gen)
    bt = torch.full((len(lens), max([1, width, *need])), nb - 1, dtype=torch.int32)
    cache = torch.zeros(fp4_cache_shape(nb, hkv, bs, d), dtype=torch.uint8, device=dev)
    at, kvs = 0, []
    for r, n in enumerate(lens):
        bt[r, :need[r]] = ids[at:at + need[r]]
        at += need[r]
        k = outlier_k(randn(gen, (n, hkv, d), dtype), gen).to(dtype)
        v = randn(gen, (n, hkv, d), dtype)
        x = torch.arange(n)
        slots = bt[r].long()[x // bs] * bs + x % bs
        reshape_and_cache(k.to(dev), v.to(dev), cache, slots.to(dev))
        kvs.append((f4.stand_for(k), f4.stand_for(v)))
    q = randn(gen, (len(lens), h, d), dtype)
    return q, cache, bt, kvs


def check(got, q, kvs, scale, dtype, window=None, starts=None):
    """Output and LSE rows against 64 bits.  A score is a sum of d products in 32 bits,
    each half a step off: (d + 8) 2^-24 of the sum of their magnitudes, times the
    scale; its exponent loses 2^-22 of the score and the exponential 2^-21.  P is held
    in two 16-bit terms, 2^-15 at worst.  So an output moves by twice that score error
    and 2^-15 of the largest value, and is rounded once."""
    out, lse = (x.cpu().double() for x in got)
    half = torch.finfo(dtype).eps / 2
    for r, (k, v) in enumerate(kvs):
        lo = 0 if starts is None else min(max(int(starts[r]), 0), k.shape[0])
        if window:
            lo = max(lo, k.shape[0] - window)
        k, v = k[lo:], v[lo:]
        o, l = f4.attend(q[r:r + 1], k, v, scale)
        if k.shape[0] == 0:
            assert not out[r].any() and (lse[:, r] == float("-inf")).all()
            continue
        g = q.shape[1] // k.shape[1]
        qa = q[r].double().abs().view(k.shape[1], g, -1)
        mags = (qa @ k.abs().permute(1, 2, 0)).amax().item() * scale
        delta = (q.shape[2] + 8) * 2.0 ** -24 * mags + mags * 2.0 ** -22 + 2.0 ** -21
        top = v.abs().max().item()
        tol = half * o[0].abs() + top * (2 * delta + 2.0 ** -15) + 2.0 ** -25
        assert ((out[r] - o[0]).abs() <= tol).all(), (r, (out[r] - o[0]).abs().max())
        ltol = delta + 2.0 ** -20 + 2.0 ** -22 * l[:, 0].abs()
        assert ((lse[:, r] - l[:, 0]).abs() <= ltol).all(), (r, (lse[:, r] - l[:, 0]).abs().max())


LENS = [1, 2, 15, 16, 17, 31, 32, 33, 0, 100, 129, 511, 700]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hkv,d,bs", [(28, 4, 128, 16), (14, 2, 64, 16), (16, 8, 256, 32),
                                        (6, 6, 96, 64), (40, 2, 32, 16), (5, 1, 160, 128),
                                        (33, 1, 192, 16)])
def test_ragged(dev, dtype, h, hkv, d, bs):
    gen = torch.Generator().manual_seed(h * d)
    q, cache, bt, kvs = batch(gen, dev, LENS, h, hkv, d, bs, dtype)
    lens = torch.tensor(LENS, dtype=torch.int32, device=dev)
    got = decode_fp4(q.to(dev), cache, bt.to(dev), lens, scale_for(d), with_lse=True)
    check(got, q, kvs, scale_for(d), dtype)


def test_more_heads_than_workgroups(dev):
    """KV heads that leave one workgroup to each of them."""
    gen = torch.Generator().manual_seed(13)
    lens = [5, 70]
    q, cache, bt, kvs = batch(gen, dev, lens, 700, 700, 64, 16, torch.bfloat16)
    t = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = decode_fp4(q.to(dev), cache, bt.to(dev), t, scale_for(64), with_lse=True)
    check(got, q, kvs, scale_for(64), torch.bfloat16)


@pytest.mark.parametrize("lens", [[1], [2000], [9000], [20000, 3], [0], [0, 0, 5]])
@pytest.mark.parametrize("h,hkv,d", [(28, 4, 128), (16, 8, 256), (14, 2, 64)])
def test_few_sequences(dev, lens, h, hkv, d):
    gen = torch.Generator().manual_seed(sum(lens) + d)
    q, cache, bt, kvs = batch(gen, dev, lens, h, hkv, d, 16, torch.bfloat16)
    t = torch.tensor(lens, dtype=torch.int64, device=dev)
    got = decode_fp4(q.to(dev), cache, bt.to(dev), t, scale_for(d), with_lse=True)
    check(got, q, kvs, scale_for(d), torch.bfloat16)
    again = decode_fp4(q.to(dev), cache, bt.to(dev), t, scale_for(d))
    assert torch.equal(again, got[0])


@pytest.mark.parametrize("window", [1, 2, 16, 31, 33, 100, 5000, 1 << 40])
@pytest.mark.parametrize("with_starts", [False, True])
def test_window_and_starts(dev, window, with_starts):
    gen = torch.Generator().manual_seed(window)
    lens = [1, 17, 40, 64, 333, 1000]
    q, cache, bt, kvs = batch(gen, dev, lens, 28, 4, 128, 16, torch.bfloat16)
    starts = [0, 5, 40, 33, 332, -4] if with_starts else None
    t = torch.tensor(lens, dtype=torch.int32, device=dev)
    s = torch.tensor(starts, dtype=torch.int32, device=dev) if with_starts else None
    got = decode_fp4(q.to(dev), cache, bt.to(dev), t, scale_for(128), window=window,
                     with_lse=True, starts=s)
    check(got, q, kvs, scale_for(128), torch.bfloat16, window, starts)


def test_many_sequences(dev):
    """More than one launch takes; rows of a strided q and a given strided out."""
    gen = torch.Generator().manual_seed(7)
    lens = [1 + (i * 37) % 70 for i in range(1100)]
    q, cache, bt, kvs = batch(gen, dev, lens, 4, 2, 64, 16, torch.float16)
    qd = torch.zeros(1100, 9, 64, dtype=torch.float16, device=dev)
    qd[:, 2:6] = q.to(dev)
    hold = torch.full((1101, 6, 64), 7.0, dtype=torch.float16, device=dev)
    t = torch.tensor(lens, dtype=torch.int32, device=dev)
    out, lse = decode_fp4(qd[:, 2:6], cache, bt.to(dev), t, scale_for(64), out=hold[:1100, 1:5],
                          with_lse=True)
    check((out, lse), q, kvs, scale_for(64), torch.float16)
    assert (hold[1100] == 7).all() and (hold[:, 0] == 7).all() and (hold[:, 5] == 7).all()


def test_bytes_behind_the_keys_do_not_count(dev):
    """Whatever stands past a sequence's last key, before its window and in blocks that no
    table names -- NaN scales among it -- the result is the same."""
    gen = torch.Generator().manual_seed(3)
    lens = [1, 5, 18, 47, 300]
    q, cache, bt, kvs = batch(gen, dev, lens, 28, 4, 128, 16, torch.bfloat16)
    t = torch.tensor(lens, dtype=torch.int32, device=dev)
    want = decode_fp4(q.to(dev), cache, bt.to(dev), t, scale_for(128), window=40, with_lse=True)
    dirty = torch.full_like(cache, 255)
    x = [torch.arange(max(0, n - 40), n) for n in lens]
    slots = torch.cat([bt[r].long()[i // 16] * 16 + i % 16 for r, i in enumerate(x)])
    from hcp_vllm_plugin_amd.kv_cache import gather_kv
    k, v = gather_kv(cache, slots.to(dev), torch.bfloat16)
    reshape_and_cache(k, v, dirty, slots.to(dev))  # what a code stands for has that code
    got = decode_fp4(q.to(dev), dirty, bt.to(dev), t, scale_for(128), window=40, with_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("keep_nan", [False, True])
def test_nan_keys_and_values(dev, keep_nan):
    """A NaN key makes its row NaN, or (as over a 16-bit cache) its split is left out; a
    NaN value makes its 32 columns NaN."""
    gen = torch.Generator().manual_seed(4)
    lens = [40, 40, 40]
    q, cache, bt, kvs = batch(gen, dev, lens, 8, 2, 64, 16, torch.bfloat16)
    one = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    bad = one.clone()
    bad[0, 0, 40] = float("inf")
    for r, (k, v) in ((1, (bad, one)), (2, (one, bad))):
        slot = int(bt[r, 1]) * 16 + 3
        reshape_and_cache(k.to(dev), v.to(dev), cache, torch.tensor([slot], device=dev))
    t = torch.tensor(lens, dtype=torch.int32, device=dev)
    out, lse = decode_fp4(q.to(dev), cache, bt.to(dev), t, scale_for(64), with_lse=True,
                          keep_nan=keep_nan)
    out = out.cpu()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, 4:]).all()
    if keep_nan:
        assert torch.isnan(out[1, :4]).all()
    else:
        assert torch.isfinite(out[1, :4]).all()
    assert torch.isnan(out[2, :4, 32:]).all() and torch.isfinite(out[2, :4, :32]).all()
    assert torch.isfinite(out[2, 4:]).all()


def test_lengths_past_the_table_and_ids_past_the_cache(dev):
    gen = torch.Generator().manual_seed(6)
    q, cache, bt, kvs = batch(gen, dev, [64, 64], 8, 2, 128, 16, torch.bfloat16)
    t = torch.tensor([64 + 999, -3], dtype=torch.int64, device=dev)
    got = decode_fp4(q.to(dev), cache, bt.to(dev), t, scale_for(128), with_lse=True)
    check(got, q, [kvs[0], (kvs[1][0][:0], kvs[1][1][:0])], scale_for(128), torch.bfloat16)
    wild = bt.clone()
    wild[0, 2], wild[1, 1] = 1 << 30, -5  # either reads the last block
    last = bt.clone()
    last[0, 2] = last[1, 1] = cache.shape[0] - 1
    t = torch.tensor([64, 64], device=dev)
    a = decode_fp4(q.to(dev), cache, wild.to(dev), t, scale_for(128))
    b = decode_fp4(q.to(dev), cache, last.to(dev), t, scale_for(128))
    assert torch.equal(a, b)


def test_far_blocks(dev):
    """Keys more than 4 GiB into the cache."""
    gen = torch.Generator().manual_seed(8)
    h, hkv, d, bs = 16, 8, 128, 16
    nb = (5 << 30) // (hkv * bs * (d + d // 16))
    cache = torch.empty(fp4_cache_shape(nb, hkv, bs, d), dtype=torch.uint8, device=dev)
    bt = torch.tensor([[nb - 1, 0, nb // 2, nb - 2]], dtype=torch.int32)
    k, v = (randn(gen, (60, hkv, d), torch.bfloat16) for _ in "kv")
    x = torch.arange(60)
    reshape_and_cache(k.to(dev), v.to(dev), cache, (bt[0].long()[x // bs] * bs + x % bs).to(dev))
    q = randn(gen, (1, h, d), torch.bfloat16)
    got = decode_fp4(q.to(dev), cache, bt.to(dev), torch.tensor([60], device=dev), scale_for(d),
                     with_lse=True)
    check(got, q, [(f4.stand_for(k), f4.stand_for(v))], scale_for(d), torch.bfloat16)


def test_captured_and_replayed(dev):
    """Two graphs over one cache, lengths changed between replays, eager calls in between."""
    gen = torch.Generator().manual_seed(11)
    q, cache, bt, kvs = batch(gen, dev, [300, 500, 64], 28, 4, 128, 16, torch.bfloat16)
    qd, btd = q.to(dev), bt.to(dev)
    lens = [torch.tensor(x, dtype=torch.int32, device=dev) for x in ([300, 500, 64], [1, 33, 0])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode_fp4(qd, cache, btd, lens[0], scale_for(128))
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for t in lens:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = decode_fp4(qd, cache, btd, t, scale_for(128), with_lse=True)
        graphs.append((g, t, out))
    for step in range(4):
        for g, t, out in graphs:
            t.copy_(torch.tensor([300 - 70 * step, 500 - step, 64 - 20 * step], dtype=torch.int32))
            g.replay()
            eager = decode_fp4(qd, cache, btd, t, scale_for(128), with_lse=True)
            torch.cuda.synchronize()
            assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1]), step


def test_two_streams(dev):
    gen = torch.Generator().manual_seed(12)
    q, cache, bt, kvs = batch(gen, dev, [900, 200], 28, 4, 128, 16, torch.bfloat16)
    qd, btd = q.to(dev), bt.to(dev)
    t = torch.tensor([900, 200], device=dev)
    want = decode_fp4(qd, cache, btd, t, scale_for(128))
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(decode_fp4(qd, cache, btd, t, scale_for(128)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def _placed(dev, k, v, dtype, kv=None):
    """One sequence with these keys and values: (cache, table, what they (or kv) stand
    for in it)."""
    n, hkv, d = k.shape
    nb = -(-n // 16) + 1
    cache = torch.zeros(fp4_cache_shape(nb, hkv, 16, d), dtype=torch.uint8, device=dev)
    reshape_and_cache(k.to(dev), v.to(dev), cache, torch.arange(n, device=dev))
    k, v = kv or (k, v)
    return cache, torch.arange(nb, dtype=torch.int32)[None], (f4.stand_for(k), f4.stand_for(v))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_small_weights(dev, dtype):
    """A key in the first 32 of each wave far above 32764 others, 2^-14 of it each:
    together they weigh half as much, so a bias of their weights shows.  (As many KV
    heads, with the same keys, as leave a workgroup to each.)"""
    gen, n, heads = torch.Generator().manual_seed(17), 32768, 1024
    k = (torch.randn(n, 1, 32, generator=gen) * 0.05).to(dtype)
    v = (1 + 0.1 * torch.randn(n, 1, 32, generator=gen)).to(dtype)
    k[5:128:32], v[5:128:32] = 0.375, -1.0
    q = torch.ones(1, heads, 32, dtype=dtype)
    cache, bt, (ks, vs) = _placed(dev, k.to(dev).expand(n, heads, 32),
                                  v.to(dev).expand(n, heads, 32), dtype, (k, v))
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    out, lse = decode_fp4(q.to(dev), cache, bt.to(dev), lens, 0.81, with_lse=True)
    assert (out == out[:, :1]).all() and (lse == lse[:1]).all()
    check((out[:, :1], lse[:1]), q[:, :1], [(ks, vs)], 0.81, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("slope", [0.01, 0.04, -0.04, 0.3, 3.0])
def test_scores_that_rise_and_fall(dev, dtype, d, slope):
    """Scores (of half of the query heads) that climb by ``slope`` a key, past the
    maximum so far by less or by more than it is let stand, or fall."""
    gen = torch.Generator().manual_seed(d)
    n = 900
    k = randn(gen, (n, 2, d), dtype) * 0.1
    k[:, :, :32] = (slope * torch.arange(n) / 32)[:, None, None].to(dtype)
    v = randn(gen, (n, 2, d), dtype)
    q = randn(gen, (1, 8, d), dtype)
    q[:, ::2, :32] = 1.0
    cache, bt, kv = _placed(dev, k.to(dtype), v, dtype)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    got = decode_fp4(q.to(dev), cache, bt.to(dev), lens, 1.0, with_lse=True)
    check(got, q, [kv], 1.0, dtype)


def test_rows_of_out_on_top_of_each_other_are_refused(dev):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev)
    cache = torch.zeros(fp4_cache_shape(2, 2, 16, 64), dtype=torch.uint8, device=dev)
    bt, lens = torch.zeros(2, 1, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int64, device=dev)
    for out in (q[:1].expand(2, 4, 64), q[:, :1].expand(2, 4, 64)):
        with pytest.raises(ValueError, match="out"):
            decode_fp4(q, cache, bt, lens, 0.1, out=out)


def test_rows_of_out_that_share_bytes_in_part_are_refused(dev):
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=dev)
    cache = torch.zeros(fp4_cache_shape(2, 2, 16, 64), dtype=torch.uint8, device=dev)
    bt, lens = torch.zeros(2, 1, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int64, device=dev)
    room = torch.zeros(4096, dtype=torch.bfloat16, device=dev)
    for strides in ((255, 64, 1), (256, 63, 1), (64, 127, 1)):
        with pytest.raises(ValueError, match="out"):
            decode_fp4(q, cache, bt, lens, 0.1, out=room.as_strided((2, 4, 64), strides))
    heads_first = room.as_strided((2, 4, 64), (64, 128, 1))
    assert decode_fp4(q, cache, bt, lens, 0.1, out=heads_first) is heads_first
