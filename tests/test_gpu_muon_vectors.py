"""Factors of a few values: their errors are those of f32 products.

A step of one row is x' = a x + (b s + c s s) x, s = x . x.  Near s = 1 its roundings in
f32 are (each relative to what it rounds, in halves of the last place, u): a x 3.44,
b s 4.78, c s s twice 2.03, their sum 2.74 and its product with x 2.74, x' 0.7; in
squares 58, of x' = 0.7.  The library's, which keeps S, B and X whole here and adds what
cancels first: b s 4.78, the sums 2.74 twice, x' 0.7 twice; in squares 39.  With the
three in two pieces instead: X's 2.74 (of a unit, not of half), B's another 5.5, S's twice
4.1, and the sums of three products each; some 150.  So over many inputs the
library's errors are 0.8 times those in f32, where two pieces have 1.6; 64 samples of a
root mean square are good for 9 %, and 1.4 is more than five of those off.
"""
import numpy as np
import pytest

from op_tools import Bench, rounded
from picograd_amd.capi import F32
from test_gpu_muon import factor, orth

pytestmark = pytest.mark.gpu


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


@pytest.mark.parametrize("steps", [3, 5])
@pytest.mark.parametrize("k,n", [(1, 7), (1, 50), (50, 1), (1, 200), (2, 10), (10, 2), (4, 60)])
def test_errors_of_a_few_values(bench, k, n, steps):
    r = np.random.default_rng(1000 * k + n)
    own, f32 = [], []
    for _ in range(64):
        g = rounded(r.standard_normal((k, n)), F32)
        want = factor(g, steps)
        own.append(np.linalg.norm(orth(bench, g, steps=steps) - want) / np.linalg.norm(want))
        f32.append(np.linalg.norm(factor(g, steps, np.float32) - want) / np.linalg.norm(want))
    own, f32 = (np.sqrt(np.mean(np.square(v))) for v in (own, f32))
    assert own <= 1.4 * f32, (own, f32)

