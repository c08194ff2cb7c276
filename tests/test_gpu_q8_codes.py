"""Codes of 8-bit matrices next to the borders between two of them, under scales that
are no powers of two: 2^22 values, bit for bit.

v and s have 24 bits and a border h (of 8 bits) times s has 32, so v / s is off a
border by 2^-33 of itself at least or not at all, which a quotient in 64 bits shows.
"""
import numpy as np
import pytest

from op_tools import NAMES, Bench, rounded
from picograd_amd.capi import BF16, F16, F32
from test_gpu_q8 import keep, quantized

pytestmark = pytest.mark.gpu


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("r,k", [(1024, 4096), (400, 10240)])
def test_codes_next_to_borders(bench, dtype, axis, r, k):
    g = np.random.default_rng(r + k + dtype)
    power = g.integers(-9, 10, (r, 1)) if dtype == F16 else g.integers(-122, 120, (r, 1))
    top = rounded(np.ldexp(1 + g.random((r, 1)), power), dtype)
    s = (top / 127).astype(np.float32).astype(np.float64)
    # the borders, then the values of the type around each
    v = s * (g.integers(0, 127, (r, k)) + 0.5)
    v = rounded(v * (1 + g.integers(-2, 3, (r, k)) * 2.0 ** -23), dtype) * g.choice([-1, 1], (r, k))
    v = np.clip(v, -top, top)
    v[:, :1] = top
    a = v.T if axis == 0 else v
    got = keep(bench, bench.tensor(a, dtype), axis, a.shape)
    assert np.array_equal(got.T if axis == 0 else got, quantized(v))
