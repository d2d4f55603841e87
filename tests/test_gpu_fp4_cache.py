"""GPU: K and V into the 4-bit cache and back (``reshape_and_cache``, ``gather_kv``),
byte for byte against the format in plain operations."""

import ctypes

import numpy as np
import pytest
import torch

from hcp_vllm_plugin_amd import _lib
from hcp_vllm_plugin_amd.kv_cache import fp4_cache_shape, gather_kv, reshape_and_cache
from hcp_vllm_plugin_amd.varlen import ENTRY_DTYPE, fp4_desc
from tests import _fp4_util as f4
from tests._util import randn

pytestmark = pytest.mark.gpu


def _rows(gen, n, hkv, d, dtype, spread=6.0):
    """Rows whose groups of 32 have scales of their own, zeros and a few ties among them."""
    x = torch.randn(n, hkv, d, generator=gen) * torch.exp2(
        spread * torch.randn(n, hkv, d // 32, generator=gen)).repeat_interleave(32, -1)
    x[torch.rand(n, hkv, d, generator=gen) < 0.05] = 0
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    at = torch.rand(n, hkv, d, generator=gen) < 0.1
    x[at] = ties[torch.randint(0, 8, (int(at.sum()),), generator=gen)]
    return x.to(dtype)


def _same(got, want):
    """The values are the wanted ones, NaN where those are."""
    got = got.cpu().double()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and \
        torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hkv,bs", [(128, 4, 16), (64, 2, 32), (256, 3, 64), (96, 1, 16),
                                      (32, 5, 128), (160, 2, 16)])
def test_write_and_read(dev, dtype, d, hkv, bs):
    gen = torch.Generator().manual_seed(d + hkv)
    n, nb = 77, 9 * 16 // bs + 6
    k, v = _rows(gen, n, hkv, d, dtype), _rows(gen, n, hkv, d, dtype)
    slots = torch.randperm(nb * bs, generator=gen)[:n]
    slots[[3, 40]] = -1
    slots[5] = nb * bs + 7
    cache = torch.randint(0, 256, fp4_cache_shape(nb, hkv, bs, d), generator=gen,
                          dtype=torch.uint8)
    want = cache.clone()
    f4.write(want, k, v, slots)
    got = cache.to(dev)
    reshape_and_cache(k.to(dev), v.to(dev), got, slots.to(dev))
    assert torch.equal(got.cpu(), want)  # the bytes of the other slots are as they were
    kk, vv = gather_kv(got, slots.to(dev), dtype)
    inside = (slots >= 0) & (slots < nb * bs)
    for x, y in ((kk, k), (vv, v)):
        ref = torch.where(inside[:, None, None], f4.stand_for(y), 0.0)
        assert _same(x, ref)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_value(dev, dtype):
    """Each of the 65536 values as the largest of its 32, next to parts of itself."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    part = torch.tensor([1, -0.9, 0.7, 0.5, 0.4, -0.3, 0.2, 0.1, 0.05, 0, 1, -1, 0.6, 0.8, 0.95,
                         0.35] * 2, dtype=torch.float32)
    k = (x.float()[:, None] * part).to(dtype).view(512, 4, 1024 // 32 * 32).reshape(-1, 4, 128)
    slots = torch.arange(k.shape[0])
    cache = torch.zeros(fp4_cache_shape(k.shape[0] // 16, 4, 16, 128), dtype=torch.uint8,
                        device=dev)
    reshape_and_cache(k.to(dev), k.flip(0).to(dev), cache, slots.to(dev))
    kk, vv = gather_kv(cache, slots.to(dev), dtype)
    ref = f4.stand_for(k)
    for got, want in ((kk, ref), (vv, ref.flip(0))):
        assert _same(got, want)
    assert torch.isnan(ref).any()  # groups with an infinity or a NaN


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_error_is_half_a_step(dev, dtype):
    """A value is off by at most half the step between codes where it lies: a quarter
    of the scale's unit up to 2, half up to 4, one up to 7."""
    gen = torch.Generator().manual_seed(5)
    k = randn(gen, (160, 2, 128), dtype)
    cache = torch.zeros(fp4_cache_shape(10, 2, 16, 128), dtype=torch.uint8, device=dev)
    slots = torch.arange(160, device=dev)
    reshape_and_cache(k.to(dev), k.to(dev), cache, slots)
    got = gather_kv(cache, slots, dtype)[0].cpu().double()
    unit = torch.exp2(f4.scale_bytes(k).double() - 127).repeat_interleave(32, -1)
    a = k.double().abs() / unit
    step = torch.where(a <= 2, 0.25, torch.where(a <= 4, 0.5, 1.0))
    assert ((got - k.double()).abs() <= step * unit).all()
    assert a.max() <= 7


@pytest.mark.parametrize("slot_dtype", [torch.int32, torch.int64])
def test_views_offsets_and_fewer_slots(dev, slot_dtype):
    """Rows out of a packed projection, fewer slots than rows, a cache that is a view."""
    gen = torch.Generator().manual_seed(9)
    hkv, d, bs, nb, n = 4, 128, 16, 8, 50
    qkv = randn(gen, (n + 9, 28 + 2 * hkv, d), torch.bfloat16).to(dev)
    k, v = qkv[:, 28:28 + hkv], qkv[:, 28 + hkv:]
    slots = torch.randperm(nb * bs, generator=gen)[:n].to(slot_dtype)
    both = torch.zeros(2, *fp4_cache_shape(nb, hkv, bs, d), dtype=torch.uint8, device=dev)
    cache = both.transpose(0, 1)[:, 1]  # every second block
    reshape_and_cache(k, v, cache, slots.to(dev))
    want = torch.zeros(nb, hkv, bs, d + d // 16, dtype=torch.uint8)
    f4.write(want, k.cpu()[:n], v.cpu()[:n], slots)
    assert torch.equal(cache.cpu(), want) and not both[0].any()
    kk, _ = gather_kv(cache, slots.to(dev), torch.bfloat16)
    assert torch.equal(kk.cpu().double(), f4.stand_for(k.cpu()[:n]))
    reshape_and_cache(k, v, cache, slots[:0].to(dev))  # no slots: nothing is written
    assert gather_kv(cache, slots[:0].to(dev), torch.bfloat16)[0].shape == (0, hkv, d)
    assert torch.equal(cache.cpu(), want)


def test_far_blocks(dev):
    """Byte offsets past 4 GiB."""
    hkv, d, bs = 8, 256, 64
    nb = (5 << 30) // (hkv * bs * (d + d // 16))
    cache = torch.empty(fp4_cache_shape(nb, hkv, bs, d), dtype=torch.uint8, device=dev)
    gen = torch.Generator().manual_seed(2)
    k, v = randn(gen, (3, hkv, d), torch.float16), randn(gen, (3, hkv, d), torch.float16)
    slots = torch.tensor([nb * bs - 1, 5, (nb - 3) * bs + 17])
    reshape_and_cache(k.to(dev), v.to(dev), cache, slots.to(dev))
    kk, vv = gather_kv(cache, slots.to(dev), torch.float16)
    assert torch.equal(kk.cpu().double(), f4.stand_for(k))
    assert torch.equal(vv.cpu().double(), f4.stand_for(v))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,hkv,bs,lens", [
    (128, 4, 16, [37]), (64, 2, 32, [0, 1, 0, 0, 700, 33, 0]), (96, 3, 16, [5] * 70 + [900, 0, 2]),
    (256, 1, 16, [1] * 4300), (32, 1, 64, [300, 0, 0])])
def test_gather_of_ragged_entries(dev, dtype, d, hkv, bs, lens):
    """Entries' keys one after another (``hcp_fp4_gather``): what gather_kv reads at
    their slots, from any first key on; an entry without a block table, and rows past
    the last one's, stay as they were."""
    gen = torch.Generator().manual_seed(d + len(lens))
    n, start = len(lens), [(7 * i) % 41 for i in range(len(lens))]
    width = max((s + x + bs - 1) // bs for s, x in zip(start, lens))
    nb = 400
    cache = torch.randint(104, 140, fp4_cache_shape(nb, hkv, bs, d), generator=gen,
                          dtype=torch.uint8).to(dev)
    table = torch.randint(0, nb, (n, width), generator=gen, dtype=torch.int32)
    table_dev = table.to(dev)
    ent = np.zeros(n, dtype=ENTRY_DTYPE)
    ent["q_len"], ent["start"], ent["len"] = 3, start, lens
    ent["block_table"] = table_dev.data_ptr() + 4 * width * np.arange(n)
    skipped = n // 2 if n > 1 else -1
    if skipped >= 0:
        ent["block_table"][skipped] = 0
    at = np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)
    total, more = int(at[-1]), 3
    ent_dev = torch.from_numpy(ent.view(np.uint8).copy()).to(dev)
    at_dev = torch.from_numpy(at[:-1].copy()).to(dev)
    kv = torch.full((2, total + more, hkv, d), 5.0, dtype=dtype, device=dev)
    made = torch.zeros_like(ent_dev)
    desc, _, _ = fp4_desc(cache)
    _lib.check(_lib.lib().hcp_fp4_gather(
        ent_dev.data_ptr(), n, at_dev.data_ptr(), total, hkv, ctypes.addressof(desc),
        _lib.dtype_code(dtype), kv[0].data_ptr(), kv[1].data_ptr(), made.data_ptr(),
        _lib.stream_ptr(dev)), "hcp_fp4_gather")
    slots = torch.full((total + more,), -1, dtype=torch.int64)
    for r, (s, x) in enumerate(zip(start, lens)):
        pos = torch.arange(s, s + x)
        if r != skipped:
            slots[at[r]:at[r] + x] = table[r][pos // bs].long() * bs + pos % bs
    k, v = gather_kv(cache, slots.to(dev), dtype)
    named = (slots >= 0).to(dev)[:, None, None]
    for got, want in ((kv[0], k), (kv[1], v)):
        assert torch.equal(got, torch.where(named, want, 5.0))
    out = made.cpu().numpy().view(ENTRY_DTYPE)
    for f, x in (("start", at[:-1]), ("len", lens), ("q_len", 3), ("block_table", 0),
                 ("stride_tok", hkv * d), ("stride_head", d), ("k_addr", kv[0].data_ptr()),
                 ("v_addr", kv[1].data_ptr())):
        assert (out[f] == x).all(), f


@pytest.mark.parametrize("order", [(0, 1), (1, 0)])
def test_heads_or_blocks_outside(dev, order):
    """Caches whose heads lie outside their blocks, or the other way round; one with a head for
    all (its bytes shared) is read, not written."""
    gen = torch.Generator().manual_seed(12)
    nb, hkv, bs, d = 6, 3, 16, 64
    k, v = (randn(gen, (40, hkv, d), torch.bfloat16) for _ in "kv")
    slots = torch.randperm(nb * bs, generator=gen)[:40]
    want = torch.zeros(fp4_cache_shape(nb, hkv, bs, d), dtype=torch.uint8)
    f4.write(want, k, v, slots)
    sizes = (nb, hkv)
    cache = torch.zeros(sizes[order[0]], sizes[order[1]], bs, d + d // 16, dtype=torch.uint8,
                        device=dev).permute(*order, 2, 3)
    reshape_and_cache(k.to(dev), v.to(dev), cache, slots.to(dev))
    assert torch.equal(cache.cpu(), want)
    one = cache[:, :1].expand(nb, hkv, bs, d + d // 16)
    kk, _ = gather_kv(one, slots.to(dev), torch.bfloat16)
    assert torch.equal(kk[:, 2].cpu().double(), f4.stand_for(k[:, 0]))
    with pytest.raises(RuntimeError, match="on top"):
        reshape_and_cache(k.to(dev), v.to(dev), one, slots.to(dev))
    assert torch.equal(cache.cpu(), want)
