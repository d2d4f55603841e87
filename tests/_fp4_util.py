"""The 4-bit KV cache in plain operations on the CPU: what a value becomes, where
its bytes lie, and attention over it in 64 bits."""

import torch

MAGS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
EXPONENTS = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}


def scale_bytes(x):
    """int64 [..., D / 32] of x [..., D]: the least power of two of which the
    largest magnitude is at most 7 times it; 255 next to an infinity or a NaN."""
    lo, hi = EXPONENTS[x.dtype]
    g = x.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    bad = ~torch.isfinite(g).all(-1)
    top = torch.where(bad, 1.0, top)
    e = torch.full(top.shape, hi, dtype=torch.int64)
    for k in range(hi, lo - 1, -1):
        e = torch.where(top <= 7 * 2.0 ** k, k, e)
    return torch.where(bad, 255, e + 127)


def codes(x, scale):
    """int64 [..., D]: sign bit and the nearest magnitude, the even one of two as near."""
    unit = torch.exp2(scale.double() - 127)[..., None]
    g = x.double().unflatten(-1, (-1, 32))
    off = (g.abs()[..., None] / unit[..., None] - MAGS).abs()
    best = off.amin(-1, keepdim=True)
    at = torch.where(off == best, torch.tensor([2, 1] * 4), 0).argmax(-1)
    c = at + 8 * torch.signbit(g)
    return torch.where(scale[..., None] == 255, 0, c).flatten(-2)


def values(code, scale):
    unit = torch.exp2(scale.double() - 127)
    unit = torch.where(scale == 255, float("nan"), unit)
    v = MAGS[code & 7] * (1 - 2.0 * (code >> 3))
    return (v.unflatten(-1, (-1, 32)) * unit[..., None]).flatten(-2)


def stand_for(x):
    """float64: what the cache stands for where x was written."""
    s = scale_bytes(x)
    return values(codes(x, s), s)


def write(cache, k, v, slots):
    """k, v [n, Hkv, D] into the bytes of a CPU cache, slot by slot."""
    nb, hkv, bs, row = cache.shape
    d = row // 17 * 16
    flat = cache.view(nb, hkv, -1)
    for is_v, x in ((0, k), (1, v)):
        s = scale_bytes(x)
        c = codes(x, s)
        b = (c[..., ::2] | c[..., 1::2] << 4).to(torch.uint8)
        for t, slot in enumerate(slots.tolist()):
            if not 0 <= slot < nb * bs:
                continue
            blk, o = divmod(slot, bs)
            if is_v:
                i = torch.arange(d // 2)
                at = bs * d // 2 + (o // 4 * (d // 8) + i // 4) * 16 + o % 4 * 4 + i % 4
            else:
                at = o * (d // 2) + torch.arange(d // 2)
            flat[blk][:, at] = b[t]
            sc = bs * d + is_v * (bs * d // 32) + (o // 4 * (d // 32) + torch.arange(d // 32)) * 4 \
                + o % 4
            flat[blk][:, sc] = s[t].to(torch.uint8)


def attend(q, k, v, scale, first=None, window=None):
    """float64 (out [T, H, D], lse [H, T]) of q over k, v [N, Hkv, D]; row i sees the
    keys up to ``first + i`` (all where None), the last ``window`` of them."""
    t, h, d = q.shape
    n, hkv, _ = k.shape
    g = h // hkv
    out = torch.zeros(t, h, d, dtype=torch.float64)
    lse = torch.full((h, t), float("-inf"), dtype=torch.float64)
    if n == 0:
        return out, lse
    at = torch.arange(n)
    see = torch.ones(t, n, dtype=torch.bool)
    if first is not None:
        last = first + torch.arange(t)[:, None]
        see = at <= last
        if window:
            see &= at > last - window
    for head in range(h):
        sc = (q[:, head].double() @ k[:, head // g].double().t()) * scale
        sc = sc.masked_fill(~see, float("-inf"))
        m = sc.amax(1, keepdim=True)
        m = torch.where(m == float("-inf"), 0.0, m)
        p = torch.exp(sc - m)
        total = p.sum(1, keepdim=True)
        some = (total != 0).squeeze(1)
        out[some, head] = ((p @ v[:, head // g].double()) / total)[some]
        lse[head, some] = (m + total.log()).squeeze(1)[some]
    return out, lse
