"""GPU: the table of cosines and sines (``rope_table``) against 64 bits."""

import math

import pytest
import torch

from hcp_vllm_plugin_amd import qk_norm_rope, rope_table

pytestmark = pytest.mark.gpu

LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}


def frequencies(rot, base, scaling, positions):
    """([f_i], factor of the values) by the definitions, one after the other."""
    s = scaling or {"rope_type": "default"}
    kind, x = s["rope_type"], s.get("factor")
    trained, a, fs = s.get("original_max_position_embeddings"), 1.0, []
    if kind == "dynamic" and positions > trained:
        base *= (x * positions / trained - (x - 1)) ** (rot / (rot - 2))
    for i in range(rot // 2):
        f = base ** (-2 * i / rot)
        if kind == "linear":
            f /= x
        elif kind == "llama3":
            wave = 2 * math.pi / f
            lo, hi = s["low_freq_factor"], s["high_freq_factor"]
            if wave > trained / lo:
                f /= x
            elif wave >= trained / hi:
                m = (trained / wave - lo) / (hi - lo)
                f = (1 - m) * f / x + m * f
        elif kind == "yarn":
            first, last = (rot / 2 * math.log(trained / (2 * math.pi * s.get(n, d))) / math.log(base)
                           for n, d in (("beta_fast", 32), ("beta_slow", 1)))
            first, last = max(math.floor(first), 0), min(math.ceil(last), rot - 1)
            m = min(max((i - first) / max(last - first, 1e-3), 0), 1)
            f = f * (1 - m) + f / x * m
        elif kind == "longrope":
            f /= s["long_factor" if positions > trained else "short_factor"][i]
        fs.append(f)
    if kind == "yarn":
        a = 0.1 * math.log(x) + 1
        if "mscale" in s:
            a = (1 + s["mscale"] * math.log(x) / 10) / (1 + s["mscale_all_dim"] * math.log(x) / 10)
    elif kind == "longrope":
        ratio = s.get("factor", positions / trained)
        a = math.sqrt(1 + math.log(ratio) / math.log(trained)) if ratio > 1 else 1.0
    return fs, s.get("attention_factor", a)


def check(table, rows, rot, base=10000.0, scaling=None, positions=None):
    """A value's own error is 2^-22 (a reduced angle in 32 bits, half a step of at most 0.79,
    and five operations of as much); the angle here, in 64 bits, is off by 2^-52 of itself."""
    fs, a = frequencies(rot, base, scaling, positions or table.shape[0])
    t = torch.tensor(rows, dtype=torch.float64)[:, None]
    f = torch.tensor(fs, dtype=torch.float64)
    want = torch.cat([torch.cos(t * f), torch.sin(t * f)], 1) * a
    half = torch.finfo(table.dtype).eps / 2
    got = table[torch.tensor(rows, device=table.device)].cpu().double()
    tol = abs(a) * (2.0 ** -22 + 2.0 ** -50 * t) + half * want.abs() + 2.0 ** -25
    off = (got - want).abs()
    assert (off <= tol).all(), off.max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rot", [16, 32, 64, 80, 128, 256])
@pytest.mark.parametrize("positions", [1, 2, 255, 4097])
def test_sizes(dev, dtype, rot, positions):
    t = rope_table(positions, rot, dtype=dtype, device=dev)
    assert t.shape == (positions, rot) and t.dtype == dtype
    check(t, list(range(positions)), rot)


@pytest.mark.parametrize("scaling", [
    None, {"rope_type": "default"}, {"type": "linear", "rope_type": "linear", "factor": 2.5}, LLAMA3,
    {**LLAMA3, "low_freq_factor": 2.0, "factor": 32}, YARN, {**YARN, "beta_fast": 16, "beta_slow": 2},
    {**YARN, "attention_factor": 0.75}, {**YARN, "original_max_position_embeddings": 64},
    {**YARN, "factor": 40, "mscale": 0.7, "mscale_all_dim": 1.2},
    {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 1000},
    {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 9000},
    {"rope_type": "longrope", "short_factor": [1.0] * 32, "long_factor": [1 + i / 3 for i in range(32)],
     "original_max_position_embeddings": 4096},
    {"rope_type": "longrope", "short_factor": [1.5] * 32, "long_factor": [9.0] * 32,
     "original_max_position_embeddings": 5000, "factor": 32.0},
    {"rope_type": "longrope", "short_factor": [0.01] * 32, "long_factor": [0.1] * 32,
     "original_max_position_embeddings": 9000, "attention_factor": 2.0}])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_scalings(dev, scaling, base):
    t = rope_table(5000, 64, base=base, scaling=scaling, device=dev)
    check(t, list(range(5000)), 64, base, scaling)


def test_far_positions(dev):
    """Two million of them, where an angle in 32 bits would be off by an eighth."""
    n = 2000003
    t = rope_table(n, 32, device=dev)
    rows = [0, 1, n // 3, 1 << 20, n - 2, n - 1]
    check(t, rows, 32)


def test_a_given_table(dev):
    """A strided out; the columns beside it stay."""
    hold = torch.full((300, 96), 5.0, dtype=torch.bfloat16, device=dev)
    out = rope_table(300, 64, out=hold[:, 16:80], scaling=YARN)
    assert out.data_ptr() == hold[:, 16:80].data_ptr()
    check(out, list(range(300)), 64, scaling=YARN)
    assert (hold[:, :16] == 5).all() and (hold[:, 80:] == 5).all()
    assert rope_table(0, 64, device=dev).shape == (0, 64)


def test_read_by_qk_norm_rope(dev):
    """A head rotated by the table and back is the head."""
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(70, 2, 64, generator=gen).to(torch.bfloat16).to(dev)
    pos = torch.arange(1000, 1070, device=dev)
    t = rope_table(2000, 64, scaling=LLAMA3, device=dev)
    back = t.clone()
    back[:, 32:] *= -1
    y, _ = qk_norm_rope(x, x, pos, t)
    z, _ = qk_norm_rope(y, y, pos, back)
    # two roundings to bf16 of values up to the pair's length
    pair = torch.hypot(x[..., :32].float(), x[..., 32:].float()).repeat(1, 1, 2)
    assert ((z.float() - x.float()).abs() <= 2 ** -8 * 2.5 * pair + 1e-6).all()
