"""The operators of a step over a KV cache held in 4 bits, one case per kind of call.

A case is a dict of plain values; its "kind" names the operator:

* ``tables``  a step's block table, slots and positions from the requests' lengths
              (``build_step_tables``).
* ``rope``    norms of the query and key heads, the position rotation and the cache write in one pass
              (``qk_norm_rope``), into a 16-bit or a 4-bit cache or into none.
* ``write``   K and V rows into the 4-bit cache (``reshape_and_cache``) and back (``gather_kv``): what
              the cache then stands for.
* ``decode``  attention of single-token queries over the 4-bit cache (``decode_fp4``).
* ``forward`` ``HcpRingAttentionImpl.forward`` with ``kv_cache_dtype="fp4"`` over the layers of one
              engine step: prefill chunks, and decode rows beside them.
* ``step``    the operators in the order of a decode step: tables, then each layer's norms, rotation
              and write, and its attention.

The 4-bit cache is a uint8 tensor [blocks, KV heads, block_size, D + D / 16].  The bytes of one
(block, head) hold, in this order: the K codes [block_size][D / 2]; the V codes [block_size / 4][D / 8]
[4 keys][4 bytes]; the K scales [block_size / 4][D / 32][4 keys]; the V scales likewise.  A code is
sign, two bits of exponent, one of mantissa (0, 0.5, 1, 1.5, 2, 3, 4, 6), the even column in a byte's
low half; 32 columns share a scale byte b that stands for 2^(b - 127): the least power of two for
which the largest magnitude is at most 7 times it, and a code is the nearest one, ties to the even.

Attention shapes are those of this repository's benchmark and tests: 28 / 4 heads x 128, 14 / 2 x 64,
64 / 8 x 128 and 16 / 8 x 256.  Values are N(0, 1) with a few K channels scaled up (logit outliers).
"""

from __future__ import annotations

import math
import random
import types

import torch

own = False

SHAPES = {"28/4x128": (28, 4, 128), "14/2x64": (14, 2, 64),
          "64/8x128": (64, 8, 128), "16/8x256": (16, 8, 256)}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EXPONENTS = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}  # of a scale, by the model's type
LARGEST_FLOPS = 4.77e11  # a drawn case stays below the largest listed ones
LARGEST_BYTES = 8.5e8
LARGEST_SCORES = 3 << 30  # values of the plain form's padded score matrix
EPS = 1e-6


def _tables(name, seqs, new_lo, new_hi, ctx_lo, ctx_hi, block=16, pad=0):
    return {"name": name, "kind": "tables", "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi,
            "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "block": block, "pad": pad}


def _rope(name, shape, dtype, tokens, cache, block=16, rot=0, interleaved=False, norm=True,
          table="f32"):
    return {"name": name, "kind": "rope", "shape": shape, "dtype": dtype, "tokens": tokens,
            "cache": cache, "block": block, "rot": rot or SHAPES[shape][2],
            "interleaved": interleaved, "norm": norm, "table": table}


def _decode(name, shape, dtype, seqs, ctx_lo, ctx_hi, block=16, window=0):
    return {"name": name, "kind": "decode", "shape": shape, "dtype": dtype, "seqs": seqs,
            "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "block": block, "window": window}


def _forward(name, shape, dtype, prefills, new_lo, new_hi, before_lo, before_hi, decodes=0,
             ctx_lo=1, ctx_hi=1, layers=2, block=16, window=0, kind="forward"):
    return {"name": name, "kind": kind, "shape": shape, "dtype": dtype, "layers": layers,
            "prefills": prefills, "new_lo": new_lo, "new_hi": new_hi, "before_lo": before_lo,
            "before_hi": before_hi, "decodes": decodes, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi,
            "block": block, "window": window}


def listed():
    return [
        # the tables of an ordinary decode step: the smallest call
        _tables("tables-64", 64, 1, 1, 512, 8192),
        # a crowded step of short prompts and decoding requests, rows padded to a fixed count
        _tables("tables-1000", 1000, 1, 96, 0, 2048, block=32, pad=700),
        # one user's decode row into a 16-bit cache: latency
        _rope("rope-1", "28/4x128", "bf16", 1, "v031"),
        # an 8k prefill step into a 16-bit cache
        _rope("rope-8k", "28/4x128", "bf16", 8192, "v031"),
        # a long prompt of a partly rotated small model without norms, no cache, neighbours paired
        _rope("rope-odd", "14/2x64", "fp16", 5003, "none", rot=32, interleaved=True, norm=False),
        # the same prefill step into the 4-bit cache
        _rope("rope-fp4", "64/8x128", "bf16", 4096, "fp4", table="16"),
        # a prefill's K and V into the 4-bit cache and back, as for a prefill that follows
        {"name": "write-8k", "kind": "write", "shape": "28/4x128", "dtype": "bf16",
         "tokens": 8192, "block": 16},
        # one user's decode step at a short context: the smallest attention
        _decode("decode-1", "28/4x128", "bf16", 1, 2000, 2000),
        # an ordinary ragged decode batch of the small model
        _decode("decode-16", "14/2x64", "fp16", 16, 1024, 8192),
        # a long-context decode batch: the largest cache
        _decode("decode-64", "28/4x128", "bf16", 64, 16384, 32768),
        # chunked prefill: a 512-token chunk near the end of a 32k prompt
        _forward("chunk-512", "28/4x128", "bf16", 1, 512, 512, 32256, 32256),
        # a decode step of 32 requests from its lengths to its attention, two layers
        _forward("step-32", "28/4x128", "bf16", 0, 1, 1, 0, 0, decodes=32, ctx_lo=512, ctx_hi=8192,
                 kind="step"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(["tables", "rope", "rope", "write", "decode", "decode", "forward", "step"])
        shape, dtype = rng.choice(list(SHAPES)), rng.choice(list(DTYPES))
        block, window = rng.choice([16, 16, 32, 64]), rng.choice([0, 0, 0, _log(rng, 100, 5000)])
        h, hkv, d = SHAPES[shape]
        if kind == "tables":
            new, ctx = _log(rng, 1, 512), _log(rng, 1, 16384)
            seqs = min(_log(rng, 1, 2000), max(1, 65536 // new))
            c = _tables("", seqs, rng.choice([0, 1, 1]), new, ctx // 8, ctx,
                        block=rng.choice([1, 8, 16, 32, 128]), pad=rng.choice([0, 0, 100]))
        elif kind == "rope":
            cache = rng.choice(["none", "v031", "v023", "fp4", "fp4"])
            c = _rope("", shape, dtype, _log(rng, 1, 8192), cache, block=block,
                      rot=rng.choice([d, d, d // 2]), interleaved=rng.random() < 0.3,
                      norm=rng.random() < 0.7, table=rng.choice(["f32", "16"]))
        elif kind == "write":
            c = {"kind": "write", "shape": shape, "dtype": dtype, "tokens": _log(rng, 1, 16384),
                 "block": block}
        elif kind == "decode":
            ctx = _log(rng, 100, 32768)
            c = _decode("", shape, dtype, _log(rng, 1, 128), max(1, ctx // 8), ctx, block=block,
                        window=window)
        elif kind == "forward":
            new, before = _log(rng, 16, 1024), _log(rng, 100, 32768)
            n, m = rng.randint(1, 4), rng.choice([0, 0, _log(rng, 1, 16)])
            c = _forward("", shape, dtype, n, max(1, new // 4), new, before // 8, before, decodes=m,
                         ctx_lo=max(1, before // 16), ctx_hi=max(1, before // 2), block=block,
                         window=window)
        else:
            ctx = _log(rng, 64, 16384)
            c = _forward("", shape, dtype, 0, 1, 1, 0, 0, decodes=_log(rng, 1, 64),
                         ctx_lo=max(1, ctx // 8), ctx_hi=ctx, block=block, window=window,
                         kind="step")
        c.pop("name", None)
        w = work(c)
        if w["flops"] > LARGEST_FLOPS or w["bytes"] > LARGEST_BYTES:
            continue
        if kind == "tables" and not sum(n for n, _ in _requests(c)):
            continue
        if kind in ("decode", "forward", "step"):
            reqs = _requests(c)
            if len(reqs) * h * max(n for n, _ in reqs) * max(k for _, k in reqs) > LARGEST_SCORES:
                continue
        return c


# -- sizes --------------------------------------------------------------------
def _sizes(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _requests(case):
    """(new tokens, keys after them) of each request, the same for every seed."""
    r = _sizes(case)
    if case["kind"] == "decode":
        return [(1, r.randint(case["ctx_lo"], case["ctx_hi"])) for _ in range(case["seqs"])]
    if case["kind"] == "tables":
        out = [(r.randint(case["new_lo"], case["new_hi"]), r.randint(case["ctx_lo"], case["ctx_hi"]))
               for _ in range(case["seqs"])]
        return [(n, n + c) for n, c in out]
    out = []
    for _ in range(case["prefills"]):
        n = r.randint(case["new_lo"], case["new_hi"])
        out.append((n, n + r.randint(case["before_lo"], case["before_hi"])))
    return out + [(1, r.randint(case["ctx_lo"], case["ctx_hi"])) for _ in range(case["decodes"])]


def _pairs(new, keys, window):
    """Visible (query, key) pairs of the last ``new`` of ``keys`` positions."""
    last = torch.arange(keys - new, keys, dtype=torch.int64) + 1
    return int((last.clamp(max=window) if window else last).sum())


def _seen(new, keys, window):
    """Keys that any of the last ``new`` positions sees."""
    return min(keys, window + new - 1) if window else keys


def work(case):
    if case["kind"] == "tables":
        reqs, bs = _requests(case), case["block"]
        tokens = sum(n for n, _ in reqs) + case["pad"]
        blocks = sum(-(-k // bs) + -(-(k - n) // bs) * -1 for n, k in reqs)
        # lengths, a table entry or free block per touched block; starts, lengths, positions, slots
        touched = sum(-(-k // bs) - (k - n) // bs for n, k in reqs if n)
        return {"bytes": 8 * len(reqs) + 4 * touched + 4 * blocks + 8 * len(reqs) + 16 * tokens,
                "flops": 0}
    h, hkv, d = SHAPES[case["shape"]]
    kv4 = hkv * (d + d // 16)  # bytes of a token's K and V in 4 bits
    if case["kind"] == "rope":
        t, rot = case["tokens"], case["rot"]
        kv = {"none": hkv * d * 4, "fp4": 2 * hkv * d * 2 + kv4}.get(case["cache"], 8 * hkv * d)
        row = rot * (4 if case["table"] == "f32" else 2)
        return {"bytes": t * (4 * h * d + kv + row + 8 + (0 if case["cache"] == "none" else 8)),
                "flops": t * (h + hkv) * (4 * d + 3 * rot)}
    if case["kind"] == "write":
        return {"bytes": case["tokens"] * (2 * (4 * hkv * d + kv4) + 8), "flops": 0}
    reqs, w, layers = _requests(case), case["window"], case.get("layers", 1)
    rows, keys = sum(n for n, _ in reqs), sum(_seen(n, k, w) for n, k in reqs)
    pairs = sum(_pairs(n, k, w) for n, k in reqs)
    per = 4 * rows * h * d + keys * kv4
    if case["kind"] == "decode":
        per += 4 * rows * h
    if case["kind"] == "step":  # q, k, v in, the rotated q out and in again
        per += rows * (4 * h * d + 4 * hkv * d + kv4 + 4 * d)
    return {"bytes": layers * per, "flops": layers * 4 * d * h * pairs}


# -- the 4-bit format in elementary operations ---------------------------------
def _scales(x):
    """Exponent of each group's scale: x [..., D] -> int32 [..., D / 32]."""
    lo, hi = EXPONENTS[x.dtype]
    top = x.float().unflatten(-1, (-1, 32)).abs().amax(-1)
    # 7 = 1.75 * 4: two below the largest value's own exponent, or one where it is past 1.75
    e = ((top.view(torch.int32) + 0x1fffff) >> 23) - 129
    return e.clamp(lo, hi)


def _power(e):
    return ((e + 127) << 23).view(torch.float32)


def _codes(x, e):
    """Codes of x [..., D] at the scales' exponents e, uint8 of one code each."""
    a = x.float().unflatten(-1, (-1, 32)) * _power(-e)[..., None]
    m = a.abs()
    c = (m > 0.25).byte() + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5)
    return (c | torch.signbit(a).byte() << 3).flatten(-2)


def _values(codes, scale_bytes):
    """float32 values of codes [..., D] with the scale bytes [..., D / 32]."""
    mags = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6],
                        device=codes.device)
    v = mags[codes.int()].unflatten(-1, (-1, 32))
    return (v * (scale_bytes.int() << 23).view(torch.float32)[..., None]).flatten(-2)


def _pack(k, v):
    """The cache bytes [blocks, Hkv, bs, D + D / 16] of k, v [blocks, Hkv, bs, D]."""
    nb, hkv, bs, d = k.shape
    ek, ev = _scales(k), _scales(v)
    ck, cv = _codes(k, ek), _codes(v, ev)
    bk, bv = ck[..., ::2] | ck[..., 1::2] << 4, cv[..., ::2] | cv[..., 1::2] << 4
    bv = bv.view(nb, hkv, bs // 4, 4, d // 8, 4).transpose(3, 4)
    sk, sv = ((e + 127).byte().view(nb, hkv, bs // 4, 4, d // 32).transpose(3, 4) for e in (ek, ev))
    return torch.cat([x.reshape(nb, hkv, -1) for x in (bk, bv, sk, sv)], -1) \
        .view(nb, hkv, bs, d + d // 16)


def _unpack(blocks):
    """(k, v) [..., bs, D] in float32 of cache bytes [..., bs, D + D / 16]."""
    bs, d = blocks.shape[-2], blocks.shape[-1] // 17 * 16
    f = blocks.flatten(-2)
    at = (bs * d // 2, bs * d, bs * d + bs * d // 32)
    bk = f[..., :at[0]].unflatten(-1, (bs, d // 2))
    bv = f[..., at[0]:at[1]].unflatten(-1, (bs // 4, d // 8, 4, 4)).transpose(-3, -2) \
        .flatten(-2).flatten(-3, -2)
    sk, sv = (s.unflatten(-1, (bs // 4, d // 32, 4)).transpose(-2, -1).flatten(-3, -2)
              for s in (f[..., at[1]:at[2]], f[..., at[2]:]))
    return tuple(_values(torch.stack([b & 15, b >> 4], -1).flatten(-2), s)
                 for b, s in ((bk, sk), (bv, sv)))


def _slot_index(cache, slots, head_dim):
    """For rows at ``slots``: flat positions in the cache bytes of the K codes [n, Hkv, D / 2], the V
    codes, the K scales [n, Hkv, D / 32] and the V scales."""
    nb, hkv, bs, _ = cache.shape
    d, dev = head_dim, cache.device
    blk, off = (slots // bs)[:, None, None], (slots % bs)[:, None, None]
    base = (blk * hkv + torch.arange(hkv, device=dev)[:, None]) * (bs * (d + d // 16))
    i, g = torch.arange(d // 2, device=dev), torch.arange(d // 32, device=dev)
    kc = base + off * (d // 2) + i
    vc = base + bs * d // 2 + ((off // 4 * (d // 8) + i // 4) * 4 + off % 4) * 4 + i % 4
    ks = base + bs * d + (off // 4 * (d // 32) + g) * 4 + off % 4
    return kc, vc, ks, ks + bs * d // 32


def _write_rows(cache, k, v, slots):
    """k, v [n, Hkv, D] into the cache bytes at ``slots``."""
    f, (kc, vc, ks, vs) = cache.view(-1), _slot_index(cache, slots, k.shape[2])
    ek, ev = _scales(k), _scales(v)
    ck, cv = _codes(k, ek), _codes(v, ev)
    f[kc], f[vc] = ck[..., ::2] | ck[..., 1::2] << 4, cv[..., ::2] | cv[..., 1::2] << 4
    f[ks], f[vs] = (ek + 127).byte(), (ev + 127).byte()


def _read_rows(cache, slots, dtype):
    """(k, v) [n, Hkv, D] that the cache stands for at ``slots``."""
    d = cache.shape[3] // 17 * 16
    f, (kc, vc, ks, vs) = cache.view(-1), _slot_index(cache, slots, d)
    return tuple(_values(torch.stack([f[c] & 15, f[c] >> 4], -1).flatten(-2), f[s]).to(dtype)
                 for c, s in ((kc, ks), (vc, vs)))


# -- inputs -------------------------------------------------------------------
class _Draw:
    """Seeded values on the GPU: N(0, 1) rounded to the case's dtype, four K channels scaled by 8 as
    the outlier channels of trained models are."""

    def __init__(self, case, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = DTYPES[case.get("dtype", "bf16")]
        if "shape" in case:
            self.ch = torch.randperm(SHAPES[case["shape"]][2], device="cuda", generator=self.gen)[:4]

    def randn(self, *shape, dtype=None):
        return torch.empty(*shape, dtype=dtype or self.dtype, device="cuda").normal_(generator=self.gen)

    def keys(self, *shape):
        k = self.randn(*shape)
        k[..., self.ch] *= 8
        return k

    def perm(self, n):
        return torch.randperm(n, device="cuda", generator=self.gen)

    def cache(self, nb, hkv, bs, d):
        return _pack(self.keys(nb, hkv, bs, d), self.randn(nb, hkv, bs, d))

    def weight(self, d):
        return 1 + 0.1 * self.randn(d, dtype=torch.float32)


class _State:
    """A case's inputs."""


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _tables_state(s, d, reqs, bs, spare=3):
    """Lengths, a table that names the cached blocks and a list of free ones; the blocks that the
    step will take come from that list's start."""
    held = [-(-(k - n) // bs) for n, k in reqs]
    need = [-(-k // bs) - x for (_, k), x in zip(reqs, held)]
    s.blocks = sum(held) + sum(need) + spare
    ids = d.perm(s.blocks).to(torch.int32)
    width = max(1, max(-(-k // bs) for _, k in reqs))
    s.bt = torch.zeros(len(reqs), width, dtype=torch.int32, device="cuda")
    have = torch.arange(width, device="cuda") < _ints(held)[:, None]
    s.bt[have] = ids[:sum(held)]
    s.free = ids[sum(held):].contiguous()
    s.ctx, s.new = _ints([k - n for n, k in reqs]), _ints([n for n, _ in reqs])


def _angles(case, rows, rot):
    """cos | sin of ``rows`` positions [rows, rot]; the angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    t = torch.cat([a.cos(), a.sin()], 1)
    return t.to(DTYPES[case["dtype"]] if case.get("table") == "16" else torch.float32)


def prepare(case, seed):
    s, d = _State(), _Draw(case, seed)
    s.case, kind = case, case["kind"]
    if kind == "tables":
        reqs = _requests(case)
        _tables_state(s, d, reqs, case["block"])
        s.rows = sum(n for n, _ in reqs) + case["pad"]
        return s
    h, hkv, dim = SHAPES[case["shape"]]
    bs = case["block"]
    if kind in ("rope", "write"):
        n = case["tokens"]
        nb = -(-n // bs) + -(-n // (4 * bs)) + 1
        # a prefill writes whole blocks: runs of neighbouring slots
        slots = d.perm(nb)[:-(-n // bs)][:, None] * bs + torch.arange(bs, device="cuda")
        s.slots = slots.reshape(-1)[:n].contiguous()
        # q, k and v as the projection leaves them: one row per token
        qkv = d.randn(n, h + 2 * hkv, dim)
        qkv[:, h:h + hkv, d.ch] *= 8
        s.q, s.k, s.v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
        cache = case.get("cache", "fp4")
        if cache == "fp4":
            s.cache = torch.zeros(nb, hkv, bs, dim + dim // 16, dtype=torch.uint8, device="cuda")
        elif cache != "none":
            shape = (nb, hkv, bs, 2 * dim) if cache == "v031" else (nb, 2, bs, hkv, dim)
            s.cache = torch.zeros(*shape, dtype=d.dtype, device="cuda")
        if kind == "rope":
            first = int(torch.randint(0, 32768, (), generator=torch.Generator().manual_seed(seed)))
            s.pos = torch.arange(first, first + n, device="cuda")
            s.table = _angles(case, first + n + 7, case["rot"])
            s.wq, s.wk = (d.weight(dim).to(d.dtype) for _ in "qk") if case["norm"] else (None, None)
        return s
    reqs = _requests(case)
    _tables_state(s, d, reqs, bs)
    s.rows = sum(n for n, _ in reqs)
    s.lens, s.most = _ints([k for _, k in reqs]), max(n for n, _ in reqs)
    s.scale = 1 / math.sqrt(dim)
    layers = case.get("layers", 1)
    s.caches = [d.cache(s.blocks, hkv, bs, dim) for _ in range(layers)]
    if kind == "step":
        s.qkv = [d.randn(s.rows, h + 2 * hkv, dim) for _ in range(layers)]
        s.w = [(d.weight(dim).to(d.dtype), d.weight(dim).to(d.dtype)) for _ in range(layers)]
        s.table = _angles(case, max(k for _, k in reqs) + 1, dim)
    else:  # the step's blocks are in the table already
        held, need = (s.ctx + bs - 1) // bs, (s.lens + bs - 1) // bs
        at = torch.arange(s.bt.shape[1], device="cuda")
        s.bt[(at >= held[:, None]) & (at < need[:, None])] = s.free[:int((need - held).sum())]
        s.qs = [d.randn(s.rows, h, dim) for _ in range(layers)]
        s.starts = torch.nn.functional.pad(s.new.cumsum(0), (1, 0)).to(torch.int32)
    s.layers = [types.SimpleNamespace(layer_name="model.layers.%d.self_attn.attn" % i)
                for i in range(layers)]
    s.shape, s.impl = (h, hkv, dim), None
    return s


# -- one pass, in elementary operations -----------------------------------------
def _plain_tables(ctx, new, bt, free, bs, rows):
    held, need = (ctx + bs - 1) // bs, (ctx + new + bs - 1) // bs
    take = need - held
    first = take.cumsum(0) - take
    at = torch.arange(bt.shape[1], device=bt.device)
    fresh = (at >= held[:, None]) & (at < need[:, None])
    which = (first[:, None] + at - held[:, None]).clamp(0, free.shape[0] - 1)
    bt.copy_(torch.where(fresh, free[which], bt))
    ends = new.cumsum(0)
    starts = torch.nn.functional.pad(ends, (1, 0))
    t = torch.arange(rows, device=bt.device)
    r = torch.searchsorted(ends, t, right=True)
    inside = r < new.shape[0]
    r = r.clamp(max=new.shape[0] - 1)
    pos = torch.where(inside, ctx[r] + t - starts[r], 0)
    slots = torch.where(inside, bt[r, pos // bs].long() * bs + pos % bs, -1)
    return starts.to(torch.int32), (ctx + new).to(torch.int32), pos, slots, \
        take.sum().to(torch.int32).reshape(1)


def _plain_rope(x, w, pos, table, interleaved, wide):
    """Norm (with a weight) and rotation of x [T, heads, D], rounded once; ``wide``: in 64 bits, for
    values that a 4-bit code's border may lie next to."""
    real = torch.float64 if wide else torch.float32
    y = x.to(real)
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.to(real)
    rot = table.shape[1]
    c, sn = table[pos].to(real)[:, None].chunk(2, -1)
    a, b = (y[..., :rot:2], y[..., 1:rot:2]) if interleaved else \
        (y[..., :rot // 2], y[..., rot // 2:rot])
    u, v = a * c - b * sn, b * c + a * sn
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _write16(cache, k, v, slots):
    bs = cache.shape[2]
    blk, off = slots // bs, slots % bs
    if cache.dim() == 4:
        cache[blk, :, off] = torch.cat([k, v], -1)
    else:
        cache[blk, 0, off], cache[blk, 1, off] = k, v


def _plain_attention(q, cache, bt, new, most, lens, scale, window):
    """(out [T, H, D], lse [H, T] float32) of queries that are the last ``new`` of each request's
    ``lens`` keys; all requests at once, padded to the ``most`` new tokens of one."""
    n, width = bt.shape
    (t, h, d), hkv = q.shape, cache.shape[1]
    k, v = (x.transpose(1, 2).reshape(n, hkv, -1, d) for x in _unpack(cache[bt.long()]))
    ends = new.cumsum(0)
    rows = torch.arange(t, device=q.device)
    r = torch.searchsorted(ends, rows, right=True)
    i = rows - (ends - new)[r]
    padded = torch.zeros(n, most, h, d, device=q.device)
    padded[r, i] = q.float()
    x = padded.view(n, most, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    sc = (x @ k.transpose(-1, -2)).view(n, hkv, h // hkv, most, -1) * scale
    key = torch.arange(sc.shape[-1], device=q.device)
    last = (lens - new)[:, None] + torch.arange(most, device=q.device)
    see = key <= last[..., None]
    if window:
        see &= key > last[..., None] - window
    sc.masked_fill_(~see[:, None, None], float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = sc.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(n, hkv, -1, p.shape[-1]) @ v).view(n, hkv, -1, most, d) / total
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, h, d)[r, i]
    return out.to(q.dtype), lse.permute(1, 2, 0, 3).reshape(h, n, most)[:, r, i]


def _plain(s):
    case = s.case
    kind = case["kind"]
    if kind == "tables":
        return *_plain_tables(s.ctx, s.new, s.bt, s.free, case["block"], s.rows), s.bt
    if kind == "rope":
        wide = case["cache"] == "fp4"
        q = _plain_rope(s.q, s.wq, s.pos, s.table, case["interleaved"], False)
        k = _plain_rope(s.k, s.wk, s.pos, s.table, case["interleaved"], wide)
        if wide:
            _write_rows(s.cache, k, s.v, s.slots)
            return q, *_read_rows(s.cache, s.slots, q.dtype)
        if case["cache"] == "none":
            return q, k
        _write16(s.cache, k, s.v, s.slots)
        return q, s.cache
    if kind == "write":
        _write_rows(s.cache, s.k, s.v, s.slots)
        return _read_rows(s.cache, s.slots, s.k.dtype)
    if kind == "decode":
        return _plain_attention(s.qs[0], s.caches[0], s.bt, s.new, s.most, s.lens, s.scale, case["window"])
    if kind == "forward":
        return [_plain_attention(q, c, s.bt, s.new, s.most, s.lens, s.scale, case["window"])[0]
                for q, c in zip(s.qs, s.caches)]
    starts, lens, pos, slots, _ = _plain_tables(s.ctx, s.new, s.bt, s.free, case["block"], s.rows)
    return slots, [_plain_layer(s, pos, slots, *x) for x in zip(s.qkv, s.w, s.caches)]


def _plain_layer(s, pos, slots, qkv, w, cache):
    h, hkv, _ = s.shape
    q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
    q = _plain_rope(q, w[0], pos, s.table, False, True)
    k = _plain_rope(k, w[1], pos, s.table, False, True)
    _write_rows(cache, k, v, slots)
    out = _plain_attention(q, cache, s.bt, s.new, s.most, s.lens, s.scale, s.case["window"])[0]
    return out, *_read_rows(cache, slots, q.dtype)


# -- one pass, by the framework's calls -------------------------------------------
def _impl(s):
    if s.impl is None:  # a program keeps it with its layers
        from hcp_vllm_plugin_amd.ring_backend import HcpRingAttentionImpl
        h, hkv, d = s.shape
        s.impl = HcpRingAttentionImpl(h, d, s.scale, hkv, sliding_window=s.case["window"] or None,
                                      kv_cache_dtype="fp4")
    return s.impl


def _framework(s):
    from hcp_vllm_plugin_amd import build_step_tables, decode_fp4, qk_norm_rope
    from hcp_vllm_plugin_amd.kv_cache import gather_kv, reshape_and_cache
    case = s.case
    kind = case["kind"]
    if kind == "tables":
        t = build_step_tables(s.ctx, s.new, s.bt, s.free, case["block"], s.rows)
        return t.query_start_loc, t.seq_lens, t.positions, t.slot_mapping, t.blocks_used, s.bt
    if kind == "rope":
        into = {} if case["cache"] == "none" else \
            {"value": s.v, "kv_cache": s.cache, "slot_mapping": s.slots}
        q, k = qk_norm_rope(s.q, s.k, s.pos, s.table, q_weight=s.wq, k_weight=s.wk, eps=EPS,
                            interleaved=case["interleaved"], **into)
        if case["cache"] == "fp4":
            return q, *gather_kv(s.cache, s.slots, q.dtype)
        return q, (k if case["cache"] == "none" else s.cache)
    if kind == "write":
        reshape_and_cache(s.k, s.v, s.cache, s.slots)
        return gather_kv(s.cache, s.slots, s.k.dtype)
    if kind == "decode":
        return decode_fp4(s.qs[0], s.caches[0], s.bt, s.lens, s.scale, window=case["window"] or None,
                          with_lse=True)
    impl = _impl(s)
    if kind == "forward":
        meta = types.SimpleNamespace(num_actual_tokens=s.rows, query_start_loc=s.starts,
                                     seq_lens=s.lens, block_table=s.bt)
        return [impl.forward(layer, q, None, None, c, meta, torch.empty_like(q))
                for layer, q, c in zip(s.layers, s.qs, s.caches)]
    t = build_step_tables(s.ctx, s.new, s.bt, s.free, case["block"], s.rows)
    meta = types.SimpleNamespace(num_actual_tokens=s.rows, query_start_loc=t.query_start_loc,
                                 seq_lens=t.seq_lens, block_table=s.bt)
    (h, hkv, _), outs = s.shape, []
    for layer, qkv, w, cache in zip(s.layers, s.qkv, s.w, s.caches):
        q, k, v = qkv[:, :h], qkv[:, h:h + hkv], qkv[:, h + hkv:]
        q, _ = qk_norm_rope(q, k, t.positions, s.table, q_weight=w[0], k_weight=w[1], eps=EPS,
                            value=v, kv_cache=cache, slot_mapping=t.slot_mapping)
        out = impl.forward(layer, q, None, None, cache, meta, torch.empty_like(q))
        outs.append((out, *gather_kv(cache, t.slot_mapping, q.dtype)))
    return t.slot_mapping, outs


def run(s):
    return _framework(s) if own else _plain(s)


# -- the same in 64 bits ------------------------------------------------------
_MAGNITUDE = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest(x):
    """What the cache stands for where x [..., D] (rounded to the model's type) was written: the
    scale by comparing, the code by the distance to each, the even one where two are as near."""
    lo, hi = EXPONENTS[x.dtype]
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1, keepdim=True)
    e = torch.log2(top.clamp(min=1e-300) / 7).ceil()
    e = torch.where(top <= 7 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top > 7 * torch.exp2(e), e + 1, e).clamp(lo, hi)
    unit = torch.exp2(e)
    best, off = torch.zeros_like(g), g.abs()
    for c in range(1, 8):
        far = (g.abs() - _MAGNITUDE[c] * unit).abs()
        nearer = (far < off) | ((far == off) & (c % 2 == 0))
        best, off = torch.where(nearer, _MAGNITUDE[c] * unit, best), torch.where(nearer, far, off)
    return (best * g.sign()).flatten(-2)


def _at(cache, blk, off, head_dim):
    """K and V rows [n, Hkv, D] of keys (block, place in it), a byte address for each column."""
    nb, hkv, bs, _ = cache.shape
    d = torch.arange(head_dim, device=cache.device)
    size = bs * head_dim + 2 * (bs * head_dim // 32)
    home = (blk.long()[:, None] * hkv + torch.arange(hkv, device=cache.device))[..., None] * size
    o = off.long()[:, None, None]
    flat, mags = cache.reshape(-1), torch.tensor(_MAGNITUDE, dtype=torch.float64, device=cache.device)
    rows = []
    for v in (0, 1):
        code = (o // 4 * head_dim * 2 + d // 8 * 16 + o % 4 * 4 + d % 8 // 2 + bs * head_dim // 2) if v \
            else o * (head_dim // 2) + d // 2
        c = (flat[home + code].long() >> (4 * (d % 2))) % 16
        sc = bs * head_dim + v * (bs * head_dim // 32) + o // 4 * (head_dim // 8) + d // 32 * 4 + o % 4
        unit = torch.exp2(flat[home + sc].double() - 127)
        rows.append(mags[c % 8] * unit * (1 - 2.0 * (c // 8)))
    return rows


def _attend(q, k, v, scale, first, window):
    """float64 (out, lse) of q [T, H, D], row i at key ``first + i``, over k, v [N, Hkv, D]."""
    t, h, d = q.shape
    n, hkv, _ = k.shape
    out = torch.empty(t, h, d, dtype=torch.float64, device=q.device)
    lse = torch.empty(h, t, dtype=torch.float64, device=q.device)
    at = torch.arange(n, device=q.device)
    last = first + torch.arange(t, device=q.device)[:, None]
    hide = at > last
    if window:
        hide |= at <= last - window
    for head in range(h):
        kh = head // (h // hkv)
        sc = q[:, head].double() @ k[:, kh].t().contiguous() * scale
        sc.masked_fill_(hide, float("-inf"))
        lse[head] = torch.logsumexp(sc, 1)
        out[:, head] = torch.exp(sc - lse[head][:, None]) @ v[:, kh]
    return out, lse


def _exact_rope(x, w, pos, table, interleaved):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.double()
    half = table.shape[1] // 2
    z = torch.complex(table[pos, :half].double(), table[pos, half:].double())[:, None]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    turned = torch.complex(y[..., a], y[..., b]) * z
    out = y.clone()
    out[..., a], out[..., b] = turned.real, turned.imag
    return out


def _exact_attention(s, q, cache, bt):
    bs, outs, lses, at = s.case["block"], [], [], 0
    for r, (n, keys) in enumerate(_requests(s.case)):
        j = torch.arange(keys, device="cuda")
        k, v = _at(cache, bt[r][j // bs], j % bs, q.shape[2])
        o, l = _attend(q[at:at + n], k, v, s.scale, keys - n, s.case["window"])
        outs.append(o)
        lses.append(l)
        at += n
    return torch.cat(outs), torch.cat(lses, 1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "tables":
        return None
    if kind == "write":
        return _nearest(s.k), _nearest(s.v)
    if kind == "rope":
        q = _exact_rope(s.q, s.wq, s.pos, s.table, case["interleaved"])
        k = _exact_rope(s.k, s.wk, s.pos, s.table, case["interleaved"])
        if case["cache"] == "none":
            return q, k
        k16 = k.to(s.k.dtype)
        if case["cache"] == "fp4":
            return q, _nearest(k16), _nearest(s.v)
        c = s.cache.double()  # a token's rows lie next to each other, or a head's
        rows = c.permute(0, 2, 1, 3) if c.dim() == 4 else c.permute(0, 2, 3, 1, 4).flatten(-2)
        rows = rows.flatten(0, 1).clone()
        rows[s.slots] = torch.cat([k, s.v.double()], -1)
        rows = rows.unflatten(0, (c.shape[0], case["block"]))
        return q, (rows.permute(0, 2, 1, 3) if c.dim() == 4 else
                   rows.unflatten(-1, (2, -1)).permute(0, 3, 1, 2, 4)).contiguous()
    if kind == "decode":
        return _exact_attention(s, s.qs[0], s.caches[0], s.bt)
    if kind == "forward":
        return [_exact_attention(s, q, c, s.bt)[0] for q, c in zip(s.qs, s.caches)]
    reqs, bs = _requests(case), case["block"]
    free, slots, pos = s.free.tolist(), [], []
    for r, (_, keys) in enumerate(reqs):  # one new token each
        if (keys - 1) % bs == 0:
            s.bt[r, (keys - 1) // bs] = free.pop(0)
        slots.append(int(s.bt[r, (keys - 1) // bs]) * bs + (keys - 1) % bs)
        pos.append(keys - 1)
    where, outs, (h, hkv, _) = torch.tensor(pos, device="cuda"), [], s.shape
    for qkv, w, cache in zip(s.qkv, s.w, s.caches):
        q = _exact_rope(qkv[:, :h], w[0], where, s.table, False).to(qkv.dtype)
        k = _nearest(_exact_rope(qkv[:, h:h + hkv], w[1], where, s.table, False).to(qkv.dtype))
        v = _nearest(qkv[:, h + hkv:])
        got = []
        for r, (_, keys) in enumerate(reqs):
            j = torch.arange(keys, device="cuda")
            kk, vv = _at(cache, s.bt[r][j // bs], j % bs, q.shape[2])
            kk[-1], vv[-1] = k[r], v[r]
            got.append(_attend(q[r:r + 1], kk, vv, s.scale, keys - 1, case["window"])[0])
        outs.append((torch.cat(got), k, v))
    return None, outs
