"""Rotary frequencies stretched by parts where an end of the ramp lies behind the last pair; no device needed."""
import ctypes as C
import math

import numpy as np
import pytest

from gufo_npu_b200 import _capi, backend, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _capi.load()


def frequencies(lib, rope_dim, theta, factor, original, fast, slow):
    params = backend.rope_params(rope_dim, theta, "halves", "by_parts", factor, original, fast, slow, 0.0)
    out, magnitude = (C.c_double * 256)(), C.c_double()
    assert lib.gufo_cuda_rope_frequencies(C.byref(params), out, C.byref(magnitude)) == 0
    return np.array(out[:rope_dim // 2])


@pytest.mark.parametrize("fast, slow", [(32.0, 1.0), (8.0, 0.5), (1e4, 0.01)])
@pytest.mark.parametrize("rope_dim, theta, factor, original", [
    (64, 1e7, 8.0, 32768.0), (64, 1e4, 8.0, 131072.0), (128, 1e4, 4.0, 131072.0), (64, 1e5, 8.0, 1048576.0),
    (64, 1e4, 8.0, 1e9), (10, 1e4, 40.0, 60000.0), (2, 1e4, 8.0, 1000.0), (512, 5e5, 16.0, 8192.0)])
def test_ramp_keeps_its_slope(lib, rope_dim, theta, factor, original, fast, slow):
    """The ends are held inside 0 .. rope_dim - 1, of which the pairs are the first half: a ramp that ends behind the last pair
    is not made steeper, and leaves pairs that still turn often short of the whole factor."""
    got = frequencies(lib, rope_dim, theta, factor, original, fast, slow)
    pair_of = lambda turns: rope_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
    low = min(max(math.floor(pair_of(fast)), 0), rope_dim - 1)
    high = min(max(math.ceil(pair_of(slow)), 0), rope_dim - 1)
    for i in range(rope_dim // 2):
        plain = theta ** (-2.0 * i / rope_dim)
        part = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
        want = plain * (1 - part) + plain / factor * part
        # (as in test_frequencies: a power and a handful of operations in 64 bits)
        assert abs(got[i] - want) <= 64 * 2.0 ** -53 * want, i
        if pair_of(fast) <= rope_dim - 1 and i < pair_of(slow):      # turns more than `slow` times
            assert got[i] > plain / factor * (1 + 1e-9), i
