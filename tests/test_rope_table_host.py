"""CPU: scalings that ``rope_table`` refuses, for what they would make of the frequencies."""

import ctypes
import math

import pytest

from hcp_vllm_plugin_amd import _lib
from hcp_vllm_plugin_amd.qk_rope import _scaling_fields


def args(positions, **kw):
    a = _lib.RopeTableArgs()
    a.out, a.stride, a.num_positions, a.base, a.attention_factor = 0x10000, 64, positions, 1e4, 1.0
    a.rot, a.dtype = 64, _lib.DTYPE_F32
    a.factor, a.original, a.low_freq, a.high_freq = 4.0, 8192.0, 1.0, 4.0
    a.beta_fast, a.beta_slow = 32.0, 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("positions,least", [(100, 1e-308), (100, 1e-300), (100, 1e-15), (100, 3e-7),
                                             (1 << 20, 3e-3), (1 << 28, 0.99)])
def test_frequencies_past_what_64_bits_hold(positions, least):
    """An angle of more than 2^28 is off by more than 2^-25 in 64 bits; an infinite one is none."""
    L = _lib.lib()
    for scaling in (1, 2, 3):
        # (a context so short that llama3 and yarn divide the first frequencies too; yarn leaves
        # frequency 0, 1, and divides the next, 0.75)
        a = args(positions, scaling=scaling, factor=0.74 * least, original=1e-3)
        assert L.hcp_rope_table(ctypes.addressof(a), None) == _lib.HCP_EINVAL, scaling
    for at in (0, 5, 31):
        f = 1e4 ** (-2 * at / 64)
        d = (ctypes.c_double * 32)(*[1.0] * 32)
        d[at] = least * f
        a = args(positions, scaling=4, divisors=ctypes.addressof(d))
        assert L.hcp_rope_table(ctypes.addressof(a), None) == _lib.HCP_EINVAL, at


@pytest.mark.parametrize("positions", [1, 4095, 4096])
def test_longrope_needs_the_models_factor(positions):
    """A table no longer than the trained context says nothing of the model's own."""
    s = {"rope_type": "longrope", "short_factor": [1.0] * 32, "long_factor": [2.0] * 32,
         "original_max_position_embeddings": 4096}
    for more in ({}, {"factor": None}, {"attention_factor": None}):
        with pytest.raises(ValueError, match="factor"):
            _scaling_fields({**s, **more}, 64, 1e4, positions)
    for more, a in (({"factor": 32.0}, math.sqrt(1 + 5 / 12)), ({"factor": 1.0}, 1.0),
                    ({"attention_factor": 1.25}, 1.25), ({"factor": 8.0, "attention_factor": 1.0}, 1.0)):
        assert _scaling_fields({**s, **more}, 64, 1e4, positions)[8] == pytest.approx(a, rel=1e-15)
    # a longer one is taken for the model's context
    assert _scaling_fields(s, 64, 1e4, 16384)[8] == pytest.approx(math.sqrt(1 + 2 / 12), rel=1e-15)


def test_a_factor_past_32_bits():
    for x in (1e39, -1e300, float("inf"), float("nan")):
        a = args(100, attention_factor=x)
        assert _lib.lib().hcp_rope_table(ctypes.addressof(a), None) == _lib.HCP_EINVAL, x
