"""Products of few rows with 4-bit matrices whose reductions end inside a wave's run of
four steps of 128: the steps behind the end add nothing, whatever the weights
beside them hold."""
import numpy as np
import pytest

from op_tools import NAMES, Bench, rounded, within
from picograd_amd.capi import BF16, F32

pytestmark = pytest.mark.gpu


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


# one to six steps, ends in the first, the last and the second round of the eight waves
KS = [100, 256, 300, 520, 700, 768, 1400, 3900, 4096, 4100, 4400, 4700, 8300]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m", [1, 5, 16])
@pytest.mark.parametrize("k", KS)
def test_steps_behind_the_end(bench, dtype, m, k):
    """Values that 4 bits hold, so that every sum is exact; a NaN in each column of three spoils that column only."""
    L = bench.L
    g = np.random.default_rng(k + m)
    n = 50
    levels = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    draw = lambda *s: levels[g.integers(0, 8, s)] * g.choice([-1, 1], s)  # noqa: E731
    x, w = draw(m, k), draw(k, n)
    x[:, ::32], w[::32] = 6, -6  # each block's largest: its power is 1
    for at, col in ((0, 3), (k // 2, 17), (k - 1, 49)):
        w[at, col] = np.nan
    q = L.pg_amd_mx4_quantize(bench.tensor(w), 0)
    assert q, L.pg_autograd_last_error().decode()
    y = bench.unset((m, n))
    bench.ok(L.pg_amd_mx4_matmul(bench.tensor(rounded(x, dtype), dtype), q, y))
    L.pg_amd_mx4_free(q)
    within(bench.read(y), x @ w, 0, "y")
