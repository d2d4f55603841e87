"""Batches with several query tokens to a sequence, in every kind of cache, and what
verification gives by its definition in 64 bits."""

import math

import torch

from hcp_vllm_plugin_amd.kv_cache import fp4_cache_shape, reshape_and_cache
from tests import _fp4_util as f4
from tests._util import outlier_k, randn

KINDS = ("v031", "v023", "fp4")


def empty_cache(kind, nb, hkv, bs, d, dtype, dev):
    if kind == "fp4":
        return torch.zeros(fp4_cache_shape(nb, hkv, bs, d), dtype=torch.uint8, device=dev)
    shape = (nb, hkv, bs, 2 * d) if kind == "v031" else (nb, 2, bs, hkv, d)
    return torch.zeros(shape, dtype=dtype, device=dev)


def batch(gen, dev, lens, counts, h, hkv, d, bs, dtype, kind, spare=2):
    """Keys of sequences of ``lens`` and the queries of their last ``counts`` tokens: (q,
    cache, table, row starts, [(k, v) float64 as the cache stands for them])."""
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + spare
    ids = torch.randperm(nb, generator=gen)
    bt = torch.full((len(lens), max([1, *need])), nb - 1, dtype=torch.int32)
    cache = empty_cache(kind, nb, hkv, bs, d, dtype, dev)
    at, kvs, slots, ks, vs = 0, [], [], [], []
    for r, n in enumerate(lens):
        bt[r, :need[r]] = ids[at:at + need[r]]
        at += need[r]
        k = outlier_k(randn(gen, (n, hkv, d), dtype), gen).to(dtype)
        v = randn(gen, (n, hkv, d), dtype)
        slots.append(slots_of(bt[r], torch.arange(n), bs))
        ks.append(k)
        vs.append(v)
        kvs.append((f4.stand_for(k), f4.stand_for(v)) if kind == "fp4" else (k.double(), v.double()))
    reshape_and_cache(torch.cat(ks).to(dev), torch.cat(vs).to(dev), cache, torch.cat(slots).to(dev))
    q = randn(gen, (sum(counts), h, d), dtype)
    starts = torch.tensor([0, *counts]).cumsum(0).to(torch.int32)
    return q, cache, bt, starts, kvs


def slots_of(row, positions, bs):
    return row.long()[positions // bs] * bs + positions % bs


def check(got, q, counts, kvs, scale, dtype, window=None):
    """Output and LSE rows against 64 bits.  A score is a sum of d products in 32 bits,
    each half a step off: (d + 8) 2^-24 of the sum of their magnitudes, times the scale;
    its exponent loses 2^-22 of the score and the exponential 2^-21.  P is held in two
    16-bit terms, 2^-15 at worst.  So an output moves by twice that score error and 2^-15
    of the largest value, and is rounded once."""
    out, lse = (x.cpu().double() for x in got)
    half, at = torch.finfo(dtype).eps / 2, 0
    for r, (n, (k, v)) in enumerate(zip(counts, kvs)):
        rows, keys = slice(at, at + n), k.shape[0]
        at += n
        if not n:
            continue
        o, l = f4.attend(q[rows], k, v, scale, first=keys - n, window=window)
        g = q.shape[1] // k.shape[1] if keys else 1
        mags = top = 0.0
        if keys:
            qa = q[rows].double().abs().view(n, k.shape[1], g, -1).transpose(0, 1).flatten(1, 2)
            mags = (qa @ k.abs().permute(1, 2, 0)).amax().item() * scale
            top = v.abs().max().item()
        delta = (q.shape[2] + 8) * 2.0 ** -24 * mags + mags * 2.0 ** -22 + 2.0 ** -21
        tol = half * o.abs() + top * (2 * delta + 2.0 ** -15) + 2.0 ** -25
        off = (out[rows] - o).abs()
        assert (off <= tol).all(), (r, off.max())
        none = l == float("-inf")
        assert (lse[:, rows][none] == float("-inf")).all(), r
        ltol = delta + 2.0 ** -20 + 2.0 ** -22 * l.abs()
        off = (lse[:, rows] - l).abs()
        assert (off <= ltol)[~none].all(), (r, off[~none].max())


# -- verification -----------------------------------------------------------------
def weights(x, temperature, probs):
    """(w float64 [V], index of the largest or None) of a row."""
    x = x.double()
    y = torch.where(torch.isnan(x), -math.inf, x)
    top = y.max()
    best = None if top == -math.inf else int((y == top).nonzero()[0])
    if probs:
        return torch.where((y > 0) & (y < math.inf), y, 0.0), best
    if best is None:
        return torch.zeros_like(y), None
    if top == math.inf:
        return (y == top).double(), best
    t = temperature if temperature > 0 else 1.0
    w = torch.exp((y - top) / t)
    return torch.where(y == -math.inf, 0.0, torch.where(y == top, 1.0, w)), best


def draw(r, u):
    """First index at which the running sum passes u times the whole; None without any."""
    c = r.cumsum(0)
    if not c[-1] > 0:
        return None
    past = (c > u * c[-1]).nonzero()
    return int(past[0]) if len(past) else int((r > 0).nonzero()[-1])


def verify(target, tokens, starts, uniform, draft_probs=None, temperature=None, probs=False):
    """([tokens of a sequence], ...) by the definition, on CPU tensors."""
    t, v = target.shape
    most, out = uniform.shape[1], []
    for b in range(len(starts) - 1):
        a, z = int(starts[b]), min(int(starts[b + 1]), t)
        n = 0 if a < 0 or z <= a else min(z - a, most)
        temp = 1.0 if temperature is None else float(temperature[b])
        greedy, got = not temp > 0, []
        for i in range(n):
            w, best = weights(target[a + i], temp, probs)
            z_ = w.sum()
            d = int(tokens[a + i + 1]) if i + 1 < n else None
            if d is not None and 0 <= d < v:
                q = 1.0 if draft_probs is None else float(draft_probs[b, i, d])
                ok = best == d if greedy else float(uniform[b, i]) * q * z_ < w[d]
                if ok:
                    got.append(d)
                    continue
            if greedy:
                token = best
            else:
                r = w.clone()
                if d is not None:
                    if draft_probs is not None:
                        r = w - draft_probs[b, i].double() * z_
                        r = torch.where(r > 0, r, 0.0)
                    elif 0 <= d < v:
                        r[d] = 0.0
                    if not r.sum() > 0:
                        r = w
                token = draw(r, float(uniform[b, -1]))
            if token is not None:
                got.append(token)
            break
        out.append(got)
    return out


def check_verified(got, want, most):
    tokens, num = got.tokens.cpu(), got.num_tokens.cpu()
    for b, w in enumerate(want):
        assert int(num[b]) == len(w), (b, int(num[b]), w)
        assert tokens[b].tolist() == w + [-1] * (most - len(w)), (b, tokens[b].tolist(), w)
