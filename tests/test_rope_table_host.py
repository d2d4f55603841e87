"""CPU: scalings that ``rope_table`` refuses, for what they would make of the frequencies."""

import ctypes

import pytest

from hcp_vllm_plugin_amd import _lib


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
