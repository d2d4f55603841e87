"""GPU: a step's block table, slots and positions (``build_step_tables``), equal to the
same made on the host."""

import types

import pytest
import torch

from hcp_vllm_plugin_amd import build_step_tables
from hcp_vllm_plugin_amd import ring_backend as rb

pytestmark = pytest.mark.gpu


def _host(ctx, new, table, free, bs, rows):
    """(query starts, lengths, positions, slots, blocks used), table updated."""
    width = table.shape[1]
    starts, lens, pos, slots, used = [0], [], [], [], 0
    for r, (c, m) in enumerate(zip(ctx, new)):
        c, m = max(c, 0), max(m, 0)
        for b in range(min(-(-c // bs), width), min(-(-(c + m) // bs), width)):
            table[r, b] = free[used] if used < len(free) else -1
            used += 1
        starts.append(starts[-1] + m)
        lens.append(c + m)
        for p in range(c, c + m):
            pos.append(p)
            b = int(table[r, p // bs]) if p // bs < width else -1
            slots.append(b * bs + p % bs if b >= 0 else -1)
    pos, slots = pos + [0] * (rows - len(pos)), slots + [-1] * (rows - len(slots))
    return starts, lens, pos[:rows], slots[:rows], used


def _run(dev, ctx, new, bs, width, free, rows, dtype=torch.int32, spare_rows=0, seed=0, strided=False):
    gen = torch.Generator().manual_seed(seed)
    table = torch.randint(0, 1 << 20, (len(ctx) + spare_rows, width), generator=gen).to(torch.int32)
    want_table = table.clone()
    want = _host(ctx, new, want_table, free, bs, rows)
    both = torch.tensor([ctx, new], dtype=dtype, device=dev)
    if strided:
        both = both.t().contiguous().t()
    wide = torch.full((len(ctx) + spare_rows, width + 3), 77, dtype=torch.int32, device=dev)
    wide[:, :width] = table.to(dev)
    got = build_step_tables(both[0], both[1], wide[:, :width],
                            torch.tensor(free, dtype=torch.int32, device=dev), bs, rows)
    assert got.query_start_loc.tolist() == want[0] and got.seq_lens.tolist() == want[1]
    assert got.positions.tolist() == want[2] and got.slot_mapping.tolist() == want[3]
    assert got.blocks_used.tolist() == [want[4]]
    assert torch.equal(wide[:, :width].cpu(), want_table) and (wide[:, width:] == 77).all()
    return got


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 256, 257, 1000, 4096])
@pytest.mark.parametrize("bs", [1, 16, 64])
def test_sizes(dev, n, bs):
    gen = torch.Generator().manual_seed(n * bs)
    ctx = torch.randint(0, 200, (n,), generator=gen).tolist()
    new = torch.randint(0, 20 if n < 1000 else 4, (n,), generator=gen).tolist()
    free = torch.randperm(30000, generator=gen)[:20 * n + 5].tolist()
    _run(dev, ctx, new, bs, 220 // bs + 1, free, sum(new) + 9, spare_rows=2, strided=n % 2 == 1,
         dtype=torch.int64 if n % 3 == 0 else torch.int32)


def test_decode_step_and_block_borders(dev):
    """One token each: a new block exactly where the cached tokens fill theirs."""
    ctx = [0, 1, 15, 16, 17, 31, 32, 33]
    _run(dev, ctx, [1] * 8, 16, 4, [9, 8, 7, 6, 5], 8)


def test_nothing_to_do(dev):
    _run(dev, [5, 0, 40], [0, 0, 0], 16, 4, [], 0)
    _run(dev, [5, 0, 40], [0, 0, 0], 16, 4, [3], 6)
    t = build_step_tables(*(torch.zeros(0, dtype=torch.int32, device=dev) for _ in "cn"),
                          torch.zeros(0, 4, dtype=torch.int32, device=dev),
                          torch.zeros(0, dtype=torch.int32, device=dev), 16, 3)
    assert t.query_start_loc.tolist() == [0] and t.seq_lens.tolist() == []
    assert t.positions.tolist() == [0, 0, 0] and t.slot_mapping.tolist() == [-1, -1, -1]
    assert t.blocks_used.tolist() == [0]


def test_out_of_blocks_and_past_the_table(dev):
    _run(dev, [10, 30, 0], [40, 3, 20], 16, 4, [11, 12], 63)       # one block short, then none
    _run(dev, [10, 60, 70], [80, 9, 5], 16, 4, [1, 2, 3, 4, 5], 94)  # rows name 64 keys
    _run(dev, [0, 5], [30, 30], 16, 8, [1, 2, 3, 4], 40)           # fewer rows than tokens
    _run(dev, [-4, 5, 2], [3, -7, 2], 16, 2, [1, 2, 3], 8)         # lengths below 0


def test_entries_without_a_block(dev):
    """A cached position whose entry is -1 (out of blocks a step before): slot -1."""
    table = torch.tensor([[-1, 5]], dtype=torch.int32, device=dev)
    t = build_step_tables(torch.tensor([3], device=dev), torch.tensor([2], device=dev), table,
                          torch.zeros(0, dtype=torch.int32, device=dev), 16, 2)
    assert t.slot_mapping.tolist() == [-1, -1] and t.positions.tolist() == [3, 4]


def test_long_lengths(dev):
    """Positions and slots past 2^31 / block_size, lengths past their limit."""
    c = (1 << 30) - 3
    table = torch.full((1, 1 << 14), 3, dtype=torch.int32, device=dev)
    free = torch.tensor([(1 << 31) - 1], dtype=torch.int32, device=dev)
    t = build_step_tables(torch.tensor([c], device=dev), torch.tensor([5], device=dev), table, free,
                          1 << 17, 5)
    assert t.positions.tolist() == [c + i for i in range(5)] and t.seq_lens.tolist() == [c + 5]
    free_id = ((1 << 31) - 1) * (1 << 17)
    cached = [3 * (1 << 17) + (1 << 17) - 3 + i for i in range(3)]
    assert t.slot_mapping.tolist() == cached + [free_id, free_id + 1]
    t = build_step_tables(torch.tensor([0], device=dev), torch.tensor([2], device=dev), table, free,
                          1 << 17, 2)
    assert t.slot_mapping.tolist() == [free_id, free_id + 1]
    t = build_step_tables(torch.tensor([1 << 40, 2], device=dev), torch.tensor([1 << 40, 1], device=dev),
                          table.expand(2, -1).contiguous(), free, 1 << 17, 4)
    assert t.query_start_loc.tolist() == [0, 1 << 30, (1 << 30) + 1]
    assert t.seq_lens.tolist() == [(1 << 31) - 1, 3]


def test_captured_and_replayed(dev):
    gen = torch.Generator().manual_seed(1)
    ctx = torch.zeros(40, dtype=torch.int32, device=dev)
    new = torch.zeros(40, dtype=torch.int32, device=dev)
    table = torch.zeros(40, 8, dtype=torch.int32, device=dev)
    free = torch.arange(100, 400, dtype=torch.int32, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = build_step_tables(ctx, new, table, free, 16, 256)
    for step in range(3):
        ctx.copy_(torch.randint(0, 60, (40,), generator=gen))
        new.copy_(torch.randint(0, 7, (40,), generator=gen))
        table.fill_(step)
        g.replay()
        torch.cuda.synchronize()
        first = [x.clone() for x in (*out, table)]
        table.fill_(step)
        again = build_step_tables(ctx, new, table, free, 16, 256)
        assert all(torch.equal(a, b) for a, b in zip(first, (*again, table)))


class _Forward:
    """One request's attention over a 16-bit cache with the metadata object that its caller
    keeps from step to step."""

    def __init__(self, dev, rows, lens, starts, table):
        gen = torch.Generator().manual_seed(3)
        rb.invalidate_step_cache()
        self.impl = rb.HcpRingAttentionImpl(4, 64, 0.125, 2)
        self.layers = [types.SimpleNamespace(layer_name=f"layer{i}") for i in range(2)]
        self.cache = torch.randn(8, 2, 16, 128, generator=gen).to(dev, torch.bfloat16)
        self.q = torch.randn(rows, 4, 64, generator=gen).to(dev, torch.bfloat16)
        self.meta = types.SimpleNamespace(num_actual_tokens=rows, query_start_loc=starts,
                                          seq_lens=lens, block_table=table)

    def run(self, meta=None):
        return [self.impl.forward(layer, self.q, None, None, self.cache, meta or self.meta,
                                  torch.zeros_like(self.q)) for layer in self.layers]

    def check(self):
        """The kept object's result is that of an object that no step has seen."""
        got = self.run()
        want = self.run(types.SimpleNamespace(**vars(self.meta)))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        rb.invalidate_step_cache()
        assert all(torch.equal(a, b) for a, b in zip(got, self.run()))
        return got


@pytest.mark.parametrize("inference", [False, True])
@pytest.mark.parametrize("new", [1, 4])
def test_forward_sees_the_table_that_a_call_has_written(dev, inference, new):
    """A table made anew (here after the first one had run out of blocks) under the same
    metadata object, lengths and starts; the table a view that the forward copies."""
    with torch.inference_mode(inference):
        table = torch.zeros(2, 6, dtype=torch.int32, device=dev)[:, :2]
        free = torch.tensor([5, 6], dtype=torch.int32, device=dev)
        ctx, fresh = (torch.tensor([x, x], device=dev) for x in (16, new))
        f = _Forward(dev, 2 * new, torch.tensor([16 + new] * 2, dtype=torch.int32, device=dev),
                     torch.tensor([0, new, 2 * new], dtype=torch.int32, device=dev), table)
        first = f.run()
        build_step_tables(ctx, fresh, table, free, 16, 2 * new)
        assert table[:, 1].tolist() == [5, 6]
        second = f.check()
        assert not torch.equal(first[0], second[0])


def test_forward_sees_the_tables_of_a_replayed_graph(dev):
    """The tables captured, the attention not: every replay writes the same tensors."""
    ctx = torch.tensor([3], dtype=torch.int32, device=dev)
    new = torch.tensor([1], dtype=torch.int32, device=dev)
    table = torch.zeros(1, 4, dtype=torch.int32, device=dev)
    free = torch.tensor([2, 3, 4, 5], dtype=torch.int32, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        t = build_step_tables(ctx, new, table, free, 16, 4)
    g.replay()
    f, outs = _Forward(dev, 1, t.seq_lens, t.query_start_loc, table), []
    for n in (3, 17, 40, 15):
        ctx.fill_(n)
        g.replay()
        outs.append(f.check()[0])
    assert not any(torch.equal(outs[0], o) for o in outs[1:])
