"""Layer norm of rows that lie far from zero beside what they differ by: the mean
is as good as f32 holds it, and a row of equal values has its value as mean and
no variance.

With u = 2^-24: a first mean, 80 roundings deep at most (64 terms a thread, the
threads' sums, the factor 1 / d), is off by 80 u |x|; the mean of the differences
from it is exact but for as many roundings of itself, 6400 u^2 |x|, so the mean is
off by the half unit of its own rounding, u |x|, and nothing else that counts.  A
row of equal values has a mean that f32 holds: that rounding is exact, all
differences are 0, and so are their squares' sum and y before the bias.
"""
import numpy as np
import pytest

from op_tools import NAMES, TINY, UNIT, Bench, rounded, within
from picograd_amd.capi import BF16, F16, F32

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-5


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


# no whole number of steps for any type; past the square root of f32's range; subnormal
VALUES = [0.1, -0.1, 12345.67, 100000.3, 1e35, -7.7e34, -3e-30, 1e-17, 1e-42, 3.0, 0.0]
# every number of threads per row, rows in a block of 1024 threads (from 256 of them on) and rows in slices
SHAPES = [(1, 1), (1, 2), (1, 5), (1, 33), (1, 257), (1, 777), (1, 1023), (1, 2050), (1, 4095), (1, 8200), (33, 9001),
          (33, 17000), (33, 33001), (1, 50001)]


def rows_of(dtype, times):
    v = rounded([a for a in VALUES if abs(a) < 6e4 or dtype != F16], dtype)
    return np.tile(v, times)[:, None]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("times,d", SHAPES)
def test_rows_of_equal_values(bench, dtype, times, d):
    L = bench.L
    v = rows_of(dtype, times)
    m = len(v)
    x = np.broadcast_to(v, (m, d))
    g = np.random.default_rng(d)
    w, b = rounded(1 + 0.2 * g.standard_normal(d), F32), rounded(g.standard_normal(d), F32)
    dy = rounded(g.standard_normal((m, d)), dtype)
    tx, tw = bench.tensor(x, dtype), bench.tensor(w)
    for out in {dtype, F32}:
        y, stats = bench.unset((m, d), out), bench.unset((m, 2))
        bench.ok(L.pg_amd_layernorm(tx, tw, bench.tensor(b), EPS, y, stats))
        assert np.array_equal(bench.read(y), np.broadcast_to(rounded(b, out), (m, d)))
        bench.ok(L.pg_amd_layernorm(tx, None, None, EPS, y, stats))
        assert (bench.read(y) == 0).all()
    got, rstd = bench.read(stats), np.float64(np.float32(EPS)) ** -0.5
    assert np.array_equal(got[:, :1], v)
    assert (np.abs(got[:, 1] - rstd) <= 4 * U * rstd).all()  # a root and a quotient
    # eps 0: such a row has no norm
    bench.ok(L.pg_amd_layernorm(tx, None, None, 0.0, y, None))
    assert np.isnan(bench.read(y)).all()
    # n is 0: dx = rstd (h - mean h), dw = 0
    dx, dw, db = bench.unset((m, d), dtype), bench.unset((d,)), bench.unset((d,))
    bench.ok(L.pg_amd_layernorm_backward(tx, tw, stats, bench.tensor(dy, dtype), dx, dw, db))
    h = dy * w
    c = h.mean(1, keepdims=True)
    want = rstd * (h - c)
    bound = rstd * (10 * U * (np.abs(h) + np.abs(c)) + 64 * U * np.abs(h).mean(1, keepdims=True)) + TINY[F32]
    within(bench.read(dx), want, bound if dtype == F32 else bound + UNIT[dtype] * (np.abs(want) + bound) + TINY[dtype], "dx")
    assert (bench.read(dw) == 0).all()
    within(bench.read(db), dy.sum(0), 128 * U * np.abs(dy).sum(0), "db")


@pytest.mark.parametrize("rows,d", [(8, 33), (8, 777), (8, 4095), (300, 9001), (8, 50001)])
def test_rows_that_differ_by_their_last_places(bench, rows, d):
    """Three places up and down, one element alone, two values; eps 0."""
    L = bench.L
    g = np.random.default_rng(d)
    kinds = [lambda: g.integers(-3, 4, d), lambda: np.arange(d) == d // 2, lambda: np.where(np.arange(d) % 3 == 0, 5, -8)]
    x = []
    for i in range(rows):
        base = np.float32([12345.67, 100000.3, -0.1, 1e20][i % 4])
        x.append(np.float64(base) + np.float64(np.spacing(base)) * kinds[i % 3]())
    x = np.stack(x)
    assert np.array_equal(x, rounded(x, F32))
    y, stats = bench.unset((rows, d)), bench.unset((rows, 2))
    bench.ok(L.pg_amd_layernorm(bench.tensor(x), None, None, 0.0, y, stats))
    mean = x.mean(1, keepdims=True)
    c = x - mean
    rstd = (c * c).mean(1, keepdims=True) ** -0.5
    slices = d > 32768  # and then each slice's mean is rounded, and each joining of two
    em = (10 if slices else 1.001) * U * np.abs(mean)
    # the squares, 80 roundings deep, are about the mean before its last rounding; those of slices about theirs
    er = 80 * U + (em * rstd + (em * rstd) ** 2 if slices else 0)
    n = c * rstd
    within(bench.read(stats), np.concatenate([mean, rstd], 1), np.concatenate([em, rstd * er], 1) + TINY[F32], "stats")
    within(bench.read(y), n, np.abs(n) * (er + 2 * U) + em * rstd * (1 + er), "y")


@pytest.mark.parametrize("times,d", [(1, 40), (1, 5000), (33, 9001), (1, 40000)])
def test_the_same_bits_alone_and_among_others(bench, times, d):
    """Rows whose sums are taken twice stand beside others that are done."""
    L = bench.L
    g = np.random.default_rng(3)
    v = rows_of(F32, times)
    x = np.where(np.arange(len(v))[:, None] % 2 == 0, v, rounded(g.standard_normal((len(v), d)), F32))
    y, stats = bench.unset(x.shape), bench.unset((len(v), 2))
    first = None
    for _ in range(3):
        bench.ok(L.pg_amd_layernorm(bench.tensor(x), None, None, EPS, y, stats))
        got = [L.read(y), L.read(stats)]
        assert first is None or all(np.array_equal(a, b) for a, b in zip(got, first))
        first = got
    assert (first[0][::2] == 0).all() and np.array_equal(first[1][::2, :1], v[::2])
    c = x[1::2] - x[1::2].mean(1, keepdims=True)
    want = c / np.sqrt((c * c).mean(1, keepdims=True) + np.float64(np.float32(EPS)))
    assert (np.abs(first[0][1::2] - want) <= 100 * U * (np.abs(want) + 1)).all()
