"""GPU: float32 tables of ``rope_table``, near the rounding of the values in 64 bits."""

import math

import pytest
import torch

from hcp_vllm_plugin_amd import rope_table
from tests.test_gpu_rope_table import LLAMA3, YARN, frequencies

pytestmark = pytest.mark.gpu


def wanted(rows, rot, base, scaling, positions):
    """(values, angles) in 64 bits."""
    fs, a = frequencies(rot, base, scaling, positions)
    angle = torch.tensor(rows, dtype=torch.float64)[:, None] * torch.tensor(fs, dtype=torch.float64)
    return torch.cat([angle.cos(), angle.sin()], 1) * a, torch.cat([angle, angle], 1), a


@pytest.mark.parametrize("rot", [16, 48, 64, 128, 256])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("scaling", [
    None, LLAMA3, YARN, {**YARN, "attention_factor": 0.7}, {**YARN, "attention_factor": -1.3},
    {**YARN, "attention_factor": 1000.0}, {"rope_type": "linear", "factor": 3e-4}])
def test_values(dev, rot, base, scaling):
    """Before the last rounding a value of up to 1 is off by 7e-8.  The angle, a quarter turn's
    +-0.79 and a remainder of up to 2^-23, is exact to 2^-47.  Sine, p + (p^3 U + rest): three
    roundings of p^3 U, 0.08 at most, 1.5e-8; U 2^-29; the remainder times 1 - cos p, 0.29 of
    it, 3.4e-8; the bracket's rounding 4e-9.  Cosine, 1 + y: p^2 and y twice rounded, each 2^-26,
    4.5e-8, and 2^-29 for the rest.  Either times a factor in two terms: three roundings of a
    term up to 0.3 of it, 1e-8.  The angles here are off by 2^-52 of themselves (and
    those of the frequencies as much)."""
    n = 20011
    table = rope_table(n, rot, base=base, scaling=scaling, device=dev).cpu().double()
    want, angle, a = wanted(list(range(n)), rot, base, scaling, n)
    tol = abs(a) * (7e-8 + 2.0 ** -50 * angle) + 2.0 ** -24 * want.abs()
    off = (table - want).abs()
    assert (off <= tol).all(), ((off / tol).max(), off.max())


@pytest.mark.parametrize("scaling", [None, LLAMA3, YARN])
def test_far_positions(dev, scaling):
    n = 1 << 20
    table = rope_table(n, 128, base=500000.0, scaling=scaling, device=dev)
    rows = list(range(n - 5000, n)) + list(range(0, n, 1009))
    want, angle, a = wanted(rows, 128, 500000.0, scaling, n)
    tol = a * (7e-8 + 2.0 ** -50 * angle) + 2.0 ** -24 * want.abs()
    got = table[torch.tensor(rows, device=dev)].cpu().double()
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("scaling", [None, LLAMA3, YARN])
def test_small_angles(dev, scaling):
    """Sines of the slowest frequencies at the first positions, relative: two roundings of 32
    bits and, each position further, a frequency's 2^-64 turns."""
    n = 300
    table = rope_table(n, 128, base=1e6, scaling=scaling, device=dev).cpu().double()
    want, angle, a = wanted(list(range(n)), 128, 1e6, scaling, n)
    small = angle[:, 64:] < 2.0 ** -10
    assert small.sum() > 1000
    off = (table[:, 64:] - want[:, 64:]).abs()
    tol = 2.0 ** -22 * want[:, 64:].abs() + a * 2.0 ** -56 + 2.0 ** -60 * torch.arange(n)[:, None]
    assert (off <= tol)[small].all(), (off / tol)[small].max()


@pytest.mark.parametrize("base", [10000.0, 1e6])
def test_angles_next_to_the_borders(dev, base):
    """Position 1's angles at every eighth of a turn and within 2^-33 to 2^-20 turns of it, where
    quarters are told apart; the positions after it, and float32, fp16 and bf16 alike."""
    near = [0.0] + [s * 2.0 ** -e for e in range(20, 34) for s in (-1, 1)]
    fractions = [m / 8 + d for m in range(1, 17) for d in near]
    for at in range(0, len(fractions), 128):
        some = (fractions[at:at + 128] + [0.1] * 128)[:128]
        longer = {"rope_type": "longrope", "original_max_position_embeddings": 4096,
                  "attention_factor": 1.0, "long_factor": [1.0] * 128,
                  "short_factor": [base ** (-2 * i / 256) / (2 * math.pi * f) for i, f in enumerate(some)]}
        want, angle, _ = wanted(list(range(9)), 256, base, longer, 9)
        for dtype in (torch.float32, torch.bfloat16, torch.float16):
            table = rope_table(9, 256, base=base, scaling=longer, dtype=dtype, device=dev).cpu().double()
            own = 7e-8 if dtype == torch.float32 else 2.0 ** -22
            tol = own + 2.0 ** -50 * angle + torch.finfo(dtype).eps / 2 * want.abs() + \
                (2.0 ** -25 if dtype == torch.float16 else 0)
            off = (table - want).abs()
            assert (off <= tol).all(), (dtype, (off / tol).max(), (off > tol).nonzero()[:5])
