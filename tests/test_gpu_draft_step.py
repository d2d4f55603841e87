"""GPU: decode steps with drafted tokens, the operators one after the other as a program
runs them: tables of the step, position table, head norms and rotation into the cache,
attention of the new tokens, logits, verification, and the next step from what was
accepted.  Every stage against 64 bits on what the stage before it gave."""

import pytest
import torch

from hcp_vllm_plugin_amd import (build_step_tables, decode_drafts, qk_norm_rope, rope_table,
                                 verify_drafts)
from hcp_vllm_plugin_amd.kv_cache import gather_kv, reshape_and_cache
from tests._drafts_util import check, check_verified, empty_cache, slots_of, verify
from tests._util import randn, scale_for

pytestmark = pytest.mark.gpu

H, HKV, D, BS, VOCAB, DRAFTS = 14, 2, 64, 16, 1003, 3
SCALING = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}


class Program:
    """One attention layer with random weights over requests of ``ctx`` cached tokens."""

    def __init__(self, gen, dev, kind, ctx, blocks=64):
        self.dev, self.kind, self.n = dev, kind, len(ctx)
        self.cache = empty_cache(kind, blocks, HKV, BS, D, torch.bfloat16, dev)
        self.bt = torch.zeros(self.n, 12, dtype=torch.int32, device=dev)
        self.free = torch.randperm(blocks, generator=gen).to(torch.int32).to(dev)
        self.table = rope_table(12 * BS, D, base=10000.0, scaling=SCALING, device=dev)
        self.emb = (torch.randn(VOCAB, (H + 2 * HKV) * D, generator=gen)).to(torch.bfloat16).to(dev)
        self.head = (torch.randn(H * D, VOCAB, generator=gen) * 0.3).to(dev)
        self.wq, self.wk = ((1 + 0.1 * torch.randn(D, generator=gen)).to(torch.bfloat16).to(dev)
                            for _ in "qk")
        self.ctx = torch.zeros(self.n, dtype=torch.int32, device=dev)
        new = torch.tensor(ctx, dtype=torch.int32, device=dev)
        t = build_step_tables(self.ctx, new, self.bt, self.free, BS, sum(ctx))
        k, v = (randn(gen, (sum(ctx), HKV, D), torch.bfloat16).to(dev) for _ in "kv")
        reshape_and_cache(k, v, self.cache, t.slot_mapping)
        self.free = self.free[int(t.blocks_used):].contiguous()
        self.ctx.copy_(new)

    def step(self, tokens, counts, uniform, temperature, draft_probs, rows):
        """(tables, q, attention, logits, verified) of a step that runs ``tokens`` [rows],
        ``counts`` of them for each request."""
        t = build_step_tables(self.ctx, counts, self.bt, self.free, BS, rows)
        qkv = self.emb[tokens].view(rows, H + 2 * HKV, D)
        q, _ = qk_norm_rope(qkv[:, :H], qkv[:, H:H + HKV], t.positions, self.table, q_weight=self.wq,
                            k_weight=self.wk, value=qkv[:, H + HKV:], kv_cache=self.cache,
                            slot_mapping=t.slot_mapping)
        o = decode_drafts(q, self.cache, self.bt, t.seq_lens, t.query_start_loc, DRAFTS + 1,
                          scale_for(D), with_lse=True)
        logits = o[0].view(rows, -1).float() @ self.head
        got = verify_drafts(logits, tokens, t.query_start_loc, uniform, draft_probs=draft_probs,
                            temperature=temperature)
        return t, q, o, logits, got


def keys_of(p, lens):
    """What the cache stands for, float64 (k, v) of each request."""
    out = []
    for r, n in enumerate(lens):
        slots = slots_of(p.bt[r].cpu(), torch.arange(n), BS).to(p.dev)
        if p.kind == "fp4":
            k, v = gather_kv(p.cache, slots, torch.bfloat16)
        elif p.kind == "v031":
            k, v = p.cache[slots // BS, :, slots % BS].chunk(2, -1)
        else:
            k, v = p.cache[slots // BS, 0, slots % BS], p.cache[slots // BS, 1, slots % BS]
        out.append((k.double().cpu(), v.double().cpu()))
    return out


@pytest.mark.parametrize("kind", ["v031", "v023", "fp4"])
@pytest.mark.parametrize("with_q", [True, False])
def test_steps(dev, kind, with_q):
    gen = torch.Generator().manual_seed(5)
    ctx = [40, 3, 100, 17]
    p = Program(gen, dev, kind, ctx)
    last = torch.randint(0, VOCAB, (4,), generator=gen).tolist()
    temperature = torch.tensor([1.0, 0.0, 0.7, 1.3])
    advanced = 0
    for step in range(3):
        counts = [1 + int(torch.randint(0, DRAFTS + 1, (), generator=gen)) for _ in ctx]
        dp = torch.softmax(2 * torch.randn(4, DRAFTS, VOCAB, generator=gen), -1)
        drafted = torch.multinomial(dp.view(-1, VOCAB), 1, generator=gen).view(4, DRAFTS)
        tokens = torch.cat([torch.cat([torch.tensor([x]), d[:n - 1]])
                            for x, d, n in zip(last, drafted, counts)])
        uniform = torch.rand(4, DRAFTS + 1, generator=gen) * 0.02  # (so that some are accepted)
        uniform[:, -1] *= 50
        rows = sum(counts) + 2  # padded
        padded = torch.cat([tokens, torch.zeros(2, dtype=tokens.dtype)])
        t, q, o, logits, got = p.step(padded.to(dev), torch.tensor(counts, dtype=torch.int32, device=dev),
                                      uniform.to(dev), temperature.to(dev),
                                      dp.to(dev) if with_q else None, rows)
        lens = [c + n for c, n in zip(ctx, counts)]
        assert t.seq_lens.tolist() == lens
        check(o, q.cpu(), counts, keys_of(p, lens), scale_for(D), torch.bfloat16)
        want = verify(logits.cpu(), padded, t.query_start_loc.cpu(), uniform, dp if with_q else None,
                      temperature)
        check_verified(got, want, DRAFTS + 1)
        # the next step: rejected keys stay behind the length and are written over
        p.free = p.free[int(t.blocks_used):].contiguous()
        num = got.num_tokens
        p.ctx += num
        ctx = [c + len(w) for c, w in zip(ctx, want)]
        assert p.ctx.tolist() == ctx
        # blocks past the new length go back to the list's front, as an engine returns them
        for r, (c, n) in enumerate(zip(ctx, lens)):
            extra = p.bt[r, -(-c // BS):-(-n // BS)]
            p.free = torch.cat([extra, p.free])
        last = got.tokens.gather(1, (num.long() - 1)[:, None])[:, 0].tolist()
        advanced += sum(len(w) > 1 for w in want)
    assert advanced > 0 or not with_q


def test_a_captured_step(dev):
    """The whole step in one graph, replayed with other tokens, numbers and lengths, eager
    steps of the same in between."""
    gen = torch.Generator().manual_seed(6)
    p = Program(gen, dev, "v031", [40, 3, 100])
    rows = 3 * (DRAFTS + 1)
    tokens = torch.zeros(rows, dtype=torch.int64, device=dev)
    counts = torch.full((3,), DRAFTS + 1, dtype=torch.int32, device=dev)
    uniform = torch.zeros(3, DRAFTS + 1, device=dev)
    dp = torch.full((3, DRAFTS, VOCAB), 1 / VOCAB, device=dev)
    args = (tokens, counts, uniform, torch.tensor([1.0, 0.8, 0.0], device=dev), dp, rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        p.step(*args)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, _, o, logits, got = p.step(*args)
    for i in range(4):
        tokens.copy_(torch.randint(0, VOCAB, (rows,), generator=gen))
        counts.copy_(torch.tensor([1 + i % 4, 4, 1 + (2 * i) % 4], dtype=torch.int32))
        uniform.copy_(torch.rand(3, DRAFTS + 1, generator=gen) * 0.5)
        p.ctx.copy_(torch.tensor([40 + i, 3 + 2 * i, 100], dtype=torch.int32))
        g.replay()
        ran = int(counts.sum())
        eager = p.step(*args)
        torch.cuda.synchronize()
        assert torch.equal(o[0][:ran], eager[2][0][:ran]), i
        assert torch.equal(got.tokens, eager[4].tokens) and torch.equal(got.num_tokens,
                                                                        eager[4].num_tokens), i
