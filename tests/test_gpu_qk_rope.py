"""GPU: norms of the heads, rotation and cache write (``qk_norm_rope``) against the
formulas in 64 bits."""

import pytest
import torch

from hcp_vllm_plugin_amd import qk_norm_rope
from hcp_vllm_plugin_amd.kv_cache import fp4_cache_shape, gather_kv, reshape_and_cache
from oracle import ring_oracle as orc
from tests import _fp4_util as f4
from tests._util import outlier_k, randn

pytestmark = pytest.mark.gpu


def _table(rows, rot, dtype, base=10000.0):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * \
        base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    return torch.cat([a.cos(), a.sin()], 1).to(dtype)


def _ref(x, w, pos, table, interleaved, eps=1e-6):
    """(float64 result, magnitudes summed in it)."""
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * w.double()
    rot = table.shape[1]
    c, s = (t[:, None] for t in table.double()[pos].chunk(2, 1))
    i = torch.arange(rot // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    out, mag = y.clone(), y.abs()
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
    mag[..., a] = (y[..., a] * c).abs() + (y[..., b] * s).abs()
    mag[..., b] = (y[..., b] * c).abs() + (y[..., a] * s).abs()
    return out, mag


def _check(got, ref, dtype):
    """In 32 bits the mean of d squares is off by (d + 2) 2^-24 of itself, its root by half of
    that, and the eight products and sums behind it by 2^-24 of the magnitudes each; the
    result is rounded once (the fp16 step is at least 2^-24)."""
    out, mag = ref
    d = out.shape[-1]
    tol = torch.finfo(dtype).eps / 2 * out.abs() + (d / 2 + 16) * 2.0 ** -24 * mag + 2.0 ** -25
    assert ((got.cpu().double() - out).abs() <= tol).all()


def _inputs(gen, t, h, hkv, d, dtype):
    q, v = randn(gen, (t, h, d), dtype), randn(gen, (t, hkv, d), dtype)
    k = outlier_k(randn(gen, (t, hkv, d), dtype), gen).to(dtype)
    return q, k, v


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("h,hkv,d,rot", [(28, 4, 128, 128), (14, 2, 64, 32), (16, 8, 256, 256),
                                         (3, 1, 80, 16), (5, 5, 8, 0), (7, 7, 248, 240),
                                         (2, 1, 112, 48), (1, 1, 16, 16)])
def test_norm_and_rotation(dev, dtype, interleaved, h, hkv, d, rot):
    gen = torch.Generator().manual_seed(h * d + rot)
    t = 37
    q, k, _ = _inputs(gen, t, h, hkv, d, dtype)
    pos = torch.randint(0, 500, (t,), generator=gen)
    for norm, wide in ((True, False), (True, True), (False, False)):
        table = _table(500, rot, torch.float32 if wide else dtype)
        wq, wk = ((1 + 0.2 * torch.randn(d, generator=gen)).to(torch.float32 if wide else dtype)
                  for _ in "qk") if norm else (None, None)
        put = lambda x: None if x is None else x.to(dev)  # noqa: E731
        gq, gk = qk_norm_rope(put(q), put(k), put(pos), put(table), q_weight=put(wq),
                              k_weight=put(wk), interleaved=interleaved)
        _check(gq, _ref(q, wq, pos, table, interleaved), dtype)
        _check(gk, _ref(k, wk, pos, table, interleaved), dtype)


@pytest.mark.parametrize("layout", ["v031", "v023"])
@pytest.mark.parametrize("t", [1, 5, 700])
def test_into_a_16_bit_cache(dev, layout, t):
    """The cache gets the key that would come back, and the value as it is; one weight only."""
    gen = torch.Generator().manual_seed(t)
    h, hkv, d, bs, nb = 28, 4, 128, 16, 60
    q, k, v = (x.to(dev) for x in _inputs(gen, t, h, hkv, d, torch.bfloat16))
    pos = torch.arange(1000, 1000 + t, dtype=torch.int32, device=dev)
    table, wk = _table(2000, d, torch.float32).to(dev), randn(gen, (d,), torch.bfloat16).to(dev)
    slots = torch.randperm(nb * bs, generator=gen)[:t]
    slots[t // 2] = -1
    shape = (nb, 2, bs, hkv, d) if layout == "v023" else (nb, hkv, bs, 2 * d)
    cache = randn(gen, shape, torch.bfloat16)
    want = cache.clone()
    gq, gk = qk_norm_rope(q, k, pos, table, k_weight=wk)
    orc.kv_cache_update(gk.cpu(), v.cpu(), want, slots, layout)
    got = cache.to(dev)
    hold = torch.empty_like(k)
    qq, kk = qk_norm_rope(q, k, pos, table, k_weight=wk, value=v, kv_cache=got,
                          slot_mapping=slots.to(dev), key_out=hold)
    assert kk is hold and torch.equal(kk, gk) and torch.equal(qq, gq)
    assert torch.equal(got.cpu(), want)
    got = cache.to(dev)
    qq, kk = qk_norm_rope(q, k, pos, table, k_weight=wk, value=v, kv_cache=got,
                          slot_mapping=slots.to(dev, torch.int32)[:t])
    assert kk is None and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,hkv,d,rot,bs,t", [(28, 4, 128, 128, 16, 50), (64, 8, 128, 64, 32, 3),
                                              (14, 2, 64, 32, 16, 1), (16, 8, 256, 256, 64, 20),
                                              (6, 3, 96, 96, 16, 33), (2, 2, 32, 16, 16, 9)])
@pytest.mark.parametrize("norm", [True, False])
def test_into_the_4_bit_cache(dev, dtype, h, hkv, d, rot, bs, t, norm):
    """The cache holds the formula's key, rounded to the type, then coded: exactly."""
    gen = torch.Generator().manual_seed(d + t)
    q, k, v = _inputs(gen, t, h, hkv, d, dtype)
    pos = torch.randint(0, 3000, (t,), generator=gen)
    table = _table(3000, rot, torch.float32)
    w = (1 + 0.2 * torch.randn(d, generator=gen)).to(dtype) if norm else None
    nb = -(-t // bs) + 3
    slots = torch.randperm(nb * bs, generator=gen)[:t]
    slots[t // 2] = -1 if t > 1 else slots[0]
    cache = torch.randint(0, 256, fp4_cache_shape(nb, hkv, bs, d), generator=gen,
                          dtype=torch.uint8)
    key = _ref(k, w, pos, table, False)[0].to(dtype)
    want = cache.clone()
    f4.write(want, key, v, slots)
    got, hold = cache.to(dev), torch.empty_like(k, device=dev)
    put = lambda x: None if x is None else x.to(dev)  # noqa: E731
    gq, gk = qk_norm_rope(put(q), put(k), put(pos), put(table), q_weight=put(w), k_weight=put(w),
                          value=put(v), kv_cache=got, slot_mapping=put(slots), key_out=hold)
    assert torch.equal(hold.cpu(), key) and torch.equal(got.cpu(), want)
    _check(gq, _ref(q, w, pos, table, False), dtype)
    other = cache.to(dev)
    reshape_and_cache(hold, put(v), other, put(slots))
    assert torch.equal(other, got)  # as the two calls one after the other


def test_in_place_views_and_padding(dev):
    """q, k and v as views of one projection, results in place, fewer slots than tokens,
    positions outside the table."""
    gen = torch.Generator().manual_seed(21)
    t, h, hkv, d, bs = 45, 28, 4, 128, 16
    qkv = randn(gen, (t, h + 2 * hkv, d), torch.bfloat16)
    pos = torch.arange(t)
    pos[7], pos[8] = -5, 10 ** 12
    table, w = _table(64, d, torch.float32), randn(gen, (d,), torch.float32)
    x = qkv.to(dev)
    q, k, v = x[:, :h], x[:, h:h + hkv], x[:, h + hkv:]
    cache = torch.zeros(fp4_cache_shape(6, hkv, bs, d), dtype=torch.uint8, device=dev)
    slots = torch.arange(40, device=dev)
    gq, gk = qk_norm_rope(q, k, pos.to(dev), table.to(dev), q_weight=w.to(dev),
                          k_weight=w.to(dev), value=v, kv_cache=cache, slot_mapping=slots,
                          query_out=q, key_out=k)
    assert gq is q and gk is k
    clamped = pos.clamp(0, 63)
    _check(gq, _ref(qkv[:, :h], w, clamped, table, False), torch.bfloat16)
    key = _ref(qkv[:, h:h + hkv], w, clamped, table, False)[0].to(torch.bfloat16)
    assert torch.equal(gk.cpu(), key) and torch.equal(v.cpu(), qkv[:, h + hkv:])
    kk, vv = gather_kv(cache, torch.arange(48, device=dev), torch.bfloat16)
    assert torch.equal(kk[:40].cpu().double(), f4.stand_for(key[:40]))
    assert torch.equal(vv[:40].cpu().double(), f4.stand_for(qkv[:40, h + hkv:]))
    assert not cache[3:].any() and not kk[40:].any() and not vv[40:].any()


def test_no_tokens_zero_rows_and_nan(dev):
    d, table = 64, _table(8, 64, torch.float32).to(dev)
    q = torch.zeros(0, 4, d, dtype=torch.float16, device=dev)
    gq, gk = qk_norm_rope(q, q[:, :1], torch.zeros(0, dtype=torch.int64, device=dev), table)
    assert gq.shape == (0, 4, d) and gk.shape == (0, 1, d)
    q = torch.zeros(2, 4, d, dtype=torch.float16, device=dev)
    w = torch.ones(d, device=dev)
    q[1, 2, 5] = float("nan")
    pos = torch.tensor([3, 4], device=dev)
    gq, gk = qk_norm_rope(q, q[:, :1], pos, table, q_weight=w, k_weight=w)
    assert not gq[0].any() and not gk.any()  # a row of zeros: eps keeps it finite
    assert torch.isnan(gq[1, 2]).all() and not gq[1, [0, 1, 3]].any()  # a NaN stays in its head


def test_captured_and_replayed(dev):
    gen = torch.Generator().manual_seed(5)
    t, h, hkv, d = 16, 28, 4, 128
    q, k, v = (x.to(dev) for x in _inputs(gen, t, h, hkv, d, torch.bfloat16))
    pos, slots = torch.arange(t, device=dev), torch.arange(t, device=dev)
    table, w = _table(512, d, torch.float32).to(dev), torch.ones(d, device=dev)
    cache = torch.zeros(fp4_cache_shape(8, hkv, 16, d), dtype=torch.uint8, device=dev)
    kw = dict(q_weight=w, k_weight=w, value=v, kv_cache=cache, slot_mapping=slots)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gq, _ = qk_norm_rope(q, k, pos, table, **kw)
    for step in range(3):
        pos.copy_(torch.arange(t) + 31 * step)
        slots.copy_(torch.arange(t).flip(0) + 16 * step)
        cache.zero_()
        g.replay()
        torch.cuda.synchronize()
        first = cache.clone()
        cache.zero_()
        eq, _ = qk_norm_rope(q, k, pos, table, **kw)
        torch.cuda.synchronize()
        assert torch.equal(gq, eq) and torch.equal(first, cache) and first.any()


def test_outputs_on_top_of_each_other_are_refused(dev):
    q, k = (torch.zeros(3, h, 64, dtype=torch.bfloat16, device=dev) for h in (4, 2))
    pos, table = torch.zeros(3, dtype=torch.int64, device=dev), torch.zeros(4, 64, device=dev)
    for kw in ({"query_out": q[:1].expand(3, 4, 64)}, {"query_out": q[:, :1].expand(3, 4, 64)},
               {"key_out": k[:1].expand(3, 2, 64)}, {"key_out": k[:, :1].expand(3, 2, 64)}):
        with pytest.raises(ValueError, match="on top"):
            qk_norm_rope(q, k, pos, table, **kw)
    one = qk_norm_rope(q[:1], k[:1], pos[:1], table, query_out=q[:1], key_out=k[:1])
    assert one[0].shape == (1, 4, 64)


def test_outputs_that_share_bytes_in_part_are_refused(dev):
    q, k = (torch.zeros(3, h, 64, dtype=torch.bfloat16, device=dev) for h in (4, 2))
    pos, table = torch.zeros(3, dtype=torch.int64, device=dev), torch.zeros(4, 64, device=dev)
    room = torch.zeros(4096, dtype=torch.bfloat16, device=dev)
    for kw in ({"query_out": room.as_strided((3, 4, 64), (248, 64, 1))},
               {"query_out": room.as_strided((3, 4, 64), (64, 184, 1))},
               {"key_out": room.as_strided((3, 2, 64), (128, 56, 1))}):
        with pytest.raises(ValueError, match="on top"):
            qk_norm_rope(q, k, pos, table, **kw)
    heads_first = room.as_strided((3, 4, 64), (64, 192, 1))
    assert qk_norm_rope(q, k, pos, table, query_out=heads_first)[0] is heads_first


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("h,hkv,d,rot,bs,t", [
    (14, 2, 64, 32, 16, 1), (2, 2, 32, 16, 16, 9), (6, 3, 96, 96, 16, 33), (16, 8, 256, 128, 64, 20),
    # fewer waves than a token has jobs, then one: a wave goes from query jobs to several of
    # keys and values, through the same LDS
    (64, 8, 128, 128, 16, 700), (16, 8, 256, 256, 32, 700), (64, 8, 128, 64, 16, 2100),
    (16, 8, 256, 256, 16, 2100), (5, 12, 96, 96, 16, 2100)])
def test_into_the_4_bit_cache_at_length(dev, dtype, interleaved, h, hkv, d, rot, bs, t):
    """Neighbours or halves paired, at every number of waves to a token: the cache holds the
    formula's key, rounded to the type, then coded; bytes of no slot stay as they were."""
    gen = torch.Generator().manual_seed(d + t + h)
    q, k, v = _inputs(gen, t, h, hkv, d, dtype)
    pos = torch.randint(0, 3000, (t,), generator=gen)
    table = _table(3000, rot, torch.float32)
    w = (1 + 0.2 * torch.randn(d, generator=gen)).to(dtype)
    nb = -(-t // bs) + 3
    slots = torch.randperm(nb * bs, generator=gen)[:t]
    slots[t // 3] = -1 if t > 1 else slots[0]
    cache = torch.randint(0, 256, fp4_cache_shape(nb, hkv, bs, d), generator=gen,
                          dtype=torch.uint8)
    key = _ref(k, w, pos, table, interleaved)[0].to(dtype)
    want = cache.clone()
    f4.write(want, key, v, slots)
    got, hold = cache.to(dev), torch.empty_like(k, device=dev)
    gq, _ = qk_norm_rope(q.to(dev), k.to(dev), pos.to(dev), table.to(dev), q_weight=w.to(dev),
                         k_weight=w.to(dev), interleaved=interleaved, value=v.to(dev), kv_cache=got,
                         slot_mapping=slots.to(dev), key_out=hold)
    assert torch.equal(hold.cpu(), key) and torch.equal(got.cpu(), want)
    _check(gq, _ref(q, w, pos, table, interleaved), dtype)
