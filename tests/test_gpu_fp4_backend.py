"""GPU: ``HcpRingAttentionImpl(kv_cache_dtype="fp4")`` over steps of every kind, and the
operators of a serving step one after the other."""

import types

import pytest
import torch

from hcp_vllm_plugin_amd import build_step_tables, decode_fp4, qk_norm_rope
from hcp_vllm_plugin_amd import ring_backend as rb
from hcp_vllm_plugin_amd.kv_cache import fp4_cache_shape, gather_kv
from tests import _fp4_util as f4
from tests._util import outlier_k, randn, scale_for

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean(monkeypatch):
    monkeypatch.delenv("HCP_RING_SPLIT_TOKENS", raising=False)
    rb.clear_peer_kv()
    rb.invalidate_step_cache()
    yield
    rb.clear_peer_kv()
    rb.invalidate_step_cache()


class Step:
    """Requests (new tokens, keys after them, staged prefix) with their keys in a 4-bit cache."""

    def __init__(self, dev, reqs, h, hkv, d, dtype, bs=16, window=None, seed=0, layers=1):
        gen = torch.Generator().manual_seed(seed)
        self.dev, self.reqs, self.dtype, self.window = dev, reqs, dtype, window
        self.h, self.hkv, self.d = h, hkv, d
        self.impl = rb.HcpRingAttentionImpl(h, d, scale_for(d), hkv, sliding_window=window,
                                            kv_cache_dtype="fp4")
        need = [-(-tk // bs) for _, tk, _ in reqs]
        nb = sum(need) + 2
        ids = torch.randperm(nb, generator=gen)
        bt = torch.zeros(len(reqs), max(need), dtype=torch.int32)
        at = 0
        for r, n in enumerate(need):
            bt[r, :n] = ids[at:at + n]
            at += n
        self.rows = sum(n for n, _, _ in reqs)
        starts = [0]
        for n, _, _ in reqs:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.meta = types.SimpleNamespace(
            num_actual_tokens=self.rows,
            query_start_loc=torch.tensor(starts, dtype=torch.int32, device=dev),
            seq_lens=torch.tensor([tk for _, tk, _ in reqs], dtype=torch.int32, device=dev),
            block_table=bt.to(dev))
        self.layers = []
        for i in range(layers):
            layer = types.SimpleNamespace(layer_name=f"layer{i}")
            cache = torch.zeros(fp4_cache_shape(nb, hkv, bs, d), dtype=torch.uint8, device=dev)
            kvs = []
            for r, (_, tk, peer) in enumerate(reqs):
                k = outlier_k(randn(gen, (tk, hkv, d), dtype), gen).to(dtype)
                v = randn(gen, (tk, hkv, d), dtype)
                x = torch.arange(tk)
                slots = (bt[r].long()[x // bs] * bs + x % bs).to(dev)
                self.impl.do_kv_cache_update(layer, k.to(dev), v.to(dev), cache, slots)
                pk = pv = None
                if peer:
                    pk = outlier_k(randn(gen, (peer, hkv, d), dtype), gen).to(dtype)
                    pv = randn(gen, (peer, hkv, d), dtype)
                    rb.stage_peer_kv(f"chunk{r}", layer.layer_name, pk.to(dev), pv.to(dev))
                    rb.map_request_peer(int(bt[r, 0]), [f"chunk{r}"])
                kvs.append((f4.stand_for(k), f4.stand_for(v), pk, pv))
            self.layers.append((layer, cache, kvs, randn(gen, (self.rows, h, d), dtype)))

    def run(self):
        return [self.impl.forward(layer, q.to(self.dev), None, None, cache, self.meta,
                                  torch.full((self.rows + 3, self.h, self.d), 9.0,
                                             dtype=self.dtype, device=self.dev))
                for layer, cache, _, q in self.layers]

    def check(self, outs):
        """A prefill launch rounds P to 16 bits (half a step of each key's weight), a result
        may be merged with a peer's after its own rounding and is rounded again: two half
        steps of the largest value, one of the result, one of a merged partial, and the
        scores' own error (test_gpu_decode_fp4)."""
        half = torch.finfo(self.dtype).eps / 2
        for out, (_, _, kvs, q) in zip(outs, self.layers):
            out = out.cpu().double()
            assert (out[self.rows:] == 9).all()
            for r, (n, tk, peer) in enumerate(self.reqs):
                a = self.starts[r]
                k, v, pk, pv = kvs[r]
                qr = q[a:a + n]
                first, see = tk - n, torch.arange(tk)[None] <= tk - n + torch.arange(n)[:, None]
                if self.window:  # (of the local keys; a staged prefix is seen whole)
                    see &= torch.arange(tk)[None] > tk - n - self.window + torch.arange(n)[:, None]
                if peer:
                    # queries past the prefix see it whole, and the local keys behind it
                    past = (first + torch.arange(n) >= peer)[:, None]
                    see = torch.where(past, see & (torch.arange(tk)[None] >= peer), see)
                    k, v = torch.cat([k, pk.double()]), torch.cat([v, pv.double()])
                    see = torch.cat([see, past.expand(n, peer)], 1)
                ref = torch.zeros(n, self.h, self.d, dtype=torch.float64)
                mags = 0.0
                for head in range(self.h):
                    kh = head // (self.h // self.hkv)
                    sc = qr[:, head].double() @ k[:, kh].t() * scale_for(self.d)
                    mags = max(mags, (qr[:, head].double().abs() @ k[:, kh].abs().t()).max().item())
                    ref[:, head] = torch.softmax(sc.masked_fill(~see, float("-inf")), 1) @ v[:, kh]
                mags *= scale_for(self.d)
                delta = (self.d + 8) * 2.0 ** -24 * mags + mags * 2.0 ** -22 + 2.0 ** -21
                top = v.abs().max().item()
                tol = 2 * half * ref.abs() + top * (2 * half + 2 * delta) + 2.0 ** -25
                assert ((out[a:a + n] - ref).abs() <= tol).all(), (r, (out[a:a + n] - ref).abs().max())


SHAPES = [(28, 4, 128, torch.bfloat16), (14, 2, 64, torch.float16), (16, 8, 256, torch.bfloat16),
          (6, 2, 96, torch.float16)]


@pytest.mark.parametrize("h,hkv,d,dtype", SHAPES)
@pytest.mark.parametrize("window", [None, 40])
@pytest.mark.parametrize("reqs", [
    [(1, 300, 0), (1, 1, 0), (1, 77, 0)],             # decode
    [(50, 50, 0)],                                    # a prompt
    [(130, 400, 0), (1, 1, 0), (17, 17, 0)],          # chunks
    [(1, 500, 0), (1, 33, 0), (90, 200, 0)],          # decode rows first
    [(60, 60, 0), (1, 900, 0), (33, 70, 0), (1, 20, 0)],  # and in between
])
def test_without_peers(dev, h, hkv, d, dtype, window, reqs):
    s = Step(dev, reqs, h, hkv, d, dtype, window=window, seed=d, layers=2)
    s.check(s.run())


@pytest.mark.parametrize("h,hkv,d,dtype", SHAPES[:2])
@pytest.mark.parametrize("reqs", [
    [(1, 300, 128), (1, 40, 0), (1, 200, 160)],       # decode behind prefixes
    [(1, 100, 128), (1, 129, 128)],                   # inside a prefix, just behind one
    [(70, 300, 128)],                                 # a chunk behind its prefix
    [(90, 180, 128), (1, 250, 64), (20, 20, 0)],      # across a prefix's end; mixed
])
def test_with_staged_peers(dev, h, hkv, d, dtype, reqs):
    s = Step(dev, reqs, h, hkv, d, dtype, seed=d + 1, layers=3)
    s.check(s.run())


def test_two_chunks_and_a_window_behind_peers(dev):
    """A prefix of two chunks; a window that ends inside the local keys."""
    for window in (None, 30):
        s = Step(dev, [(1, 400, 130), (1, 90, 0), (1, 260, 64)], 28, 4, 128, torch.bfloat16,
                 window=window, seed=9, layers=2)
        first = int(s.meta.block_table[0, 0])
        for layer, _, kvs, _ in s.layers:
            pk, pv = kvs[0][2].to(dev), kvs[0][3].to(dev)
            rb.stage_peer_kv("a", layer.layer_name, pk[:50], pv[:50])
            rb.stage_peer_kv("b", layer.layer_name, pk[50:], pv[50:])
        rb.map_request_peer(first, ["a", "b"])
        s.check(s.run())
        rb.clear_peer_kv()


def test_decode_rows_apart(dev, monkeypatch):
    """Mixed batches whose single-token rows leave the prefill launch, neighbours or not."""
    monkeypatch.setattr(rb.HcpRingAttentionImpl, "_decode_rows_apart", lambda *a, **k: True)
    for reqs in ([(1, 300, 0), (1, 90, 0), (40, 80, 0)], [(40, 80, 0), (1, 300, 0), (9, 9, 0),
                                                          (1, 90, 0)]):
        s = Step(dev, reqs, 28, 4, 128, torch.bfloat16, seed=2)
        s.check(s.run())


def test_launches_that_share_the_scratch(dev, monkeypatch):
    """Chunks whose keys do not fit the scratch together run in launches of their own."""
    monkeypatch.setattr(rb, "_FP4_SCRATCH", 200 * 4 * 4 * 128)  # 200 keys
    s = Step(dev, [(20, 150, 0), (30, 90, 0), (5, 400, 0), (9, 9, 0)], 28, 4, 128, torch.bfloat16,
             seed=3)
    s.check(s.run())


def test_many_decode_rows(dev):
    s = Step(dev, [(1, 1 + i % 50, 0) for i in range(1040)], 4, 2, 64, torch.float16, seed=4)
    s.check(s.run())


def test_step_from_lengths_to_attention(dev):
    """A prompt chunk and decoding requests through tables, norms, rotation, write and
    attention over three steps; the cache's keys and the outputs against 64 bits."""
    gen = torch.Generator().manual_seed(30)
    h, hkv, d, bs, dtype, nb = 28, 4, 128, 16, torch.bfloat16, 40
    impl = rb.HcpRingAttentionImpl(h, d, scale_for(d), hkv, kv_cache_dtype="fp4")
    layer = types.SimpleNamespace(layer_name="layer")
    a = torch.arange(256, dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    table = torch.cat([a.cos(), a.sin()], 1).float()
    w = (1 + 0.1 * torch.randn(d, generator=gen)).to(dtype)
    cache = torch.full(fp4_cache_shape(nb, hkv, bs, d), 255, dtype=torch.uint8, device=dev)
    bt = torch.full((3, 12), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(nb, generator=gen).to(torch.int32).to(dev)
    ctx, keys = [0, 0, 0], [[], [], []]
    for new in ([50, 1, 17], [1, 1, 30], [1, 1, 1]):
        t = sum(new)
        tab = build_step_tables(torch.tensor(ctx, device=dev), torch.tensor(new, device=dev), bt,
                                free, bs, t)
        free = free[int(tab.blocks_used):]
        qkv = randn(gen, (t, h + 2 * hkv, d), dtype)
        x = qkv.to(dev)
        q, _ = qk_norm_rope(x[:, :h], x[:, h:h + hkv], tab.positions, table.to(dev),
                            q_weight=w.to(dev), k_weight=w.to(dev), value=x[:, h + hkv:],
                            kv_cache=cache, slot_mapping=tab.slot_mapping)
        meta = types.SimpleNamespace(num_actual_tokens=t, query_start_loc=tab.query_start_loc,
                                     seq_lens=tab.seq_lens, block_table=bt)
        out = impl.forward(layer, q, None, None, cache, meta, torch.empty_like(q)).cpu().double()
        kk, vv = gather_kv(cache, tab.slot_mapping, dtype)
        assert torch.equal(vv.cpu().double(), f4.stand_for(qkv[:, h + hkv:]))
        at = 0
        for r, n in enumerate(new):
            pos = torch.arange(ctx[r], ctx[r] + n)
            y = qkv[at:at + n, h:h + hkv].double()
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.double()
            c, s = (z[:, None] for z in table[pos].double().chunk(2, 1))
            y = torch.cat([y[..., :64] * c - y[..., 64:] * s, y[..., 64:] * c + y[..., :64] * s], -1)
            k = f4.stand_for(y.to(dtype))
            assert torch.equal(kk[at:at + n].cpu().double(), k)
            keys[r].append((k, f4.stand_for(qkv[at:at + n, h + hkv:])))
            ka, va = (torch.cat([z[i] for z in keys[r]]) for i in (0, 1))
            ref, _ = f4.attend(q[at:at + n].cpu(), ka, va, scale_for(d), ctx[r])
            half = torch.finfo(dtype).eps / 2  # as Step.check; scores under 100 here
            tol = 2 * half * ref.abs() + va.abs().max() * (2 * half + 2.0 ** -12)
            assert ((out[at:at + n] - ref).abs() <= tol).all()
            at += n
            ctx[r] += n
    if ctx:  # the decode rows alone, through the operator itself
        lens = torch.tensor(ctx, dtype=torch.int32, device=dev)
        assert torch.equal(decode_fp4(q, cache, bt, lens, scale_for(d)).cpu().double(), out)


def test_layers_share_a_step_on_two_streams(dev):
    s = Step(dev, [(1, 300, 0), (1, 41, 0)], 28, 4, 128, torch.bfloat16, seed=6, layers=3)
    want = s.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = s.run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    s.check(want)


def test_refusals(dev, monkeypatch):
    s = Step(dev, [(1, 300, 0), (1, 41, 0)], 28, 4, 128, torch.bfloat16)
    layer, cache, _, q = s.layers[0]
    out = torch.empty(2, 28, 128, dtype=torch.bfloat16, device=dev)
    plain = rb.HcpRingAttentionImpl(28, 128, 0.1, 4)
    with pytest.raises(ValueError, match="cache for kv_cache_dtype"):
        plain.forward(layer, q.to(dev), None, None, cache, s.meta, out)
    wide = torch.zeros(40, 4, 16, 256, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="cache for kv_cache_dtype"):
        s.impl.forward(layer, q.to(dev), None, None, wide, s.meta, out)
    with pytest.raises(ValueError, match="does not match"):
        s.impl.forward(layer, q.to(dev), None, None, cache[:, :2], s.meta, out)
    monkeypatch.setenv("HCP_RING_SPLIT_TOKENS", "16")
    with pytest.raises(NotImplementedError, match="16-bit cache"):
        s.impl.forward(layer, q.to(dev), None, None, cache, s.meta, out)
    monkeypatch.delenv("HCP_RING_SPLIT_TOKENS")
    first = int(s.meta.block_table[0, 0])
    rb.register_decode_ring(first, [("c", "u")], 16, transport=object())
    try:
        with pytest.raises(NotImplementedError, match="16-bit cache"):
            s.impl.forward(layer, q.to(dev), None, None, cache, s.meta, out)
    finally:
        rb.clear_decode_ring(first)
    s.meta.seq_lens = torch.tensor([300, 400], dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="past the block-table row"):
        s.impl.forward(layer, q.to(dev), None, None, cache, s.meta, out)
    with pytest.raises(NotImplementedError, match="4-bit cache"):
        rb.HcpRingAttentionImpl(28, 80, 0.1, 4, kv_cache_dtype="fp4")
