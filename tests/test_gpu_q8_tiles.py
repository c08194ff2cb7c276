"""Products with 8-bit matrices on each of the tiles that take more than 16 rows: 64 x 64
(up to 128 tiles of 128 x 128), 128 x 128 one to a CU (up to 256 of them), 256 x 128 (up
to 256), and past that 256 x 256 or two of 128 x 128 to a CU, by their rounds over the
chip.  Bounds as the sums' exactness gives them: y's three f32 factors and its output's
rounding.
"""
import numpy as np
import pytest

from op_tools import NAMES, TINY, UNIT, Bench, rounded, to_bits, within
from picograd_amd.capi import BF16, F16, F32, shape_arg

pytestmark = pytest.mark.gpu


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


def parts(v):
    """v [R, K] as whole numbers and a scale per row."""
    top = np.abs(v).max(1)
    s = (top / 127).astype(np.float32).astype(np.float64)
    return np.clip(np.rint(v / s[:, None]), -127, 127), s


def kind(m, n):
    """The library's choice."""
    tiles = lambda a, b: -(-m // a) * -(-n // b)  # noqa: E731
    if tiles(128, 128) <= 128:
        return "64"
    if tiles(128, 128) <= 256:
        return "128"
    if tiles(256, 128) <= 256:
        return "256 x 128"
    return "256" if -(-tiles(256, 256) // 256) <= 0.34 * -(-tiles(128, 128) // 256) else "two of 128"


# the reduction in one stage, in some that are no whole round of them, in many
SIZES = [("64", 1007, 700, 1301), ("128", 1601, 300, 1503), ("128", 1000, 1030, 2050), ("256 x 128", 1401, 300, 3701),
         ("256 x 128", 2050, 130, 3470), ("256 x 128", 1409, 1000, 3603), ("256 x 128", 3001, 64, 1701),
         ("two of 128", 4500, 260, 3701), ("two of 128", 2901, 900, 5703), ("two of 128", 4353, 100, 4103),
         ("256", 3999, 290, 3503), ("256", 4001, 1030, 3506)]


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, F16)], ids=lambda d: NAMES[d])
@pytest.mark.parametrize("tile,m,k,n", SIZES)
def test_product(bench, tile, m, k, n, dtype, out):
    assert kind(m, n) == tile
    L = bench.L
    g = np.random.default_rng(m + 7 * k + 31 * n)
    x = rounded(g.standard_normal((m, k)) * np.exp(0.5 * g.standard_normal(k)), dtype)
    w = rounded(g.uniform(-1, 1, (k, n)) * k ** -0.5, F32)
    q = L.pg_amd_q8_quantize(bench.tensor(w), 0)
    assert q, L.pg_autograd_last_error().decode()
    # a row of y and 9 values behind it stay as they were
    store = bench.unset((m * n + n + 9,), out)
    y = L.pg_tensor_view(store)
    bench.frees.append((L.pg_tensor_free, y))
    i = L.tinfo(y)
    i.ndim, i.numel = 2, m * n
    i.shape[0], i.shape[1], i.stride[0], i.stride[1] = m, n, n, 1
    bench.ok(L.pg_amd_q8_matmul(bench.tensor(x, dtype), q, y))
    L.pg_amd_q8_free(q)
    whole = bench.read(store)
    assert (whole[m * n:] == rounded(777.0, out)).all()
    (qx, sx), (qw, sw) = parts(x), parts(w.T)
    want = (qx.astype(np.float32) @ qw.T.astype(np.float32)).astype(np.float64)  # whole numbers
    assert k * 127 * 127 < 2 ** 24  # so f32 holds every partial sum
    want *= sx[:, None] * sw
    bound = 3.01 * 2.0 ** -24 * np.abs(want) + TINY[F32]
    if out != F32:
        bound = bound + UNIT[out] * (np.abs(want) + bound) + TINY[out]
    within(whole[:m * n].reshape(m, n), want, bound, "y")


def test_the_most_columns_of_some_rows(bench):
    """193 rows by 2^28 columns and some: more tiles of 64 x 64 than a launch has threads for, of those that run a
    sixteenth.  W's values are 0 to 4, so that bf16 holds y."""
    L = bench.L
    m, n = 193, 2 ** 28 + 40
    w = np.resize(to_bits(np.arange(5), BF16), (1, n))
    t = L.tensor(w, BF16)
    q = L.pg_amd_q8_quantize(t, 0)
    L.pg_tensor_free(t)
    assert q, L.pg_autograd_last_error().decode()
    x = np.ones((m, 1))
    x[100], x[192] = 2, 0.5
    nd, sh = shape_arg((m, n))
    y = L.pg_tensor_empty_dtype(BF16, nd, sh)
    assert y, L.pg_amd_last_error().decode()
    try:
        bench.ok(L.pg_amd_q8_matmul(bench.tensor(x), q, y))
        for row in (0, 99, 100, 127, 128, 192):
            for at in (0, 2 ** 27 - 512, 2 ** 28 - 1024, n - 1024):
                v = L.pg_tensor_view(y)
                i = L.tinfo(v)
                i.dev += (row * n + at) * 2
                i.ndim, i.numel, i.shape[0], i.stride[0] = 1, 1024, 1024, 1
                got = bench.read(v)
                L.pg_tensor_free(v)
                assert np.array_equal(got, x[row] * ((at + np.arange(1024)) % 5)), (row, at)
    finally:
        L.pg_tensor_free(y)
        L.pg_amd_q8_free(q)

