"""4-bit matrices (pg_amd_mx4_*) against the definition: the rounding bit for
bit, the product within the f32 accumulation's (K + 2) 2^-24 of the sum of its
terms' magnitudes plus the output's own rounding.
"""
import numpy as np
import pytest

from op_tools import NAMES, TINY, UNIT, Bench, rounded, within
from picograd_amd.capi import BF16, F16, F32, shape_arg

pytestmark = pytest.mark.gpu

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


def quantized(v):
    """v [R, K] (f32 values in 64 bits) rounded along its rows."""
    v = np.asarray(v, np.float64)
    out = np.empty_like(v)
    for b in range(0, v.shape[1], 32):
        blk = v[:, b:b + 32]
        top = np.abs(blk).max(1)
        with np.errstate(invalid="ignore"):
            e = np.where(top > 0, np.frexp(np.where(np.isfinite(top), top, 1.0))[1] - 3, -127)
        unit = np.ldexp(1.0, np.maximum(e, -127))[:, None]
        a = np.abs(blk) / unit
        near = np.abs(np.where(np.isfinite(a), a, 0)[..., None] - GRID)
        code = near.argmin(-1)  # the lower of two at the same distance
        tie = (code < 7) & (near.min(-1) == np.take_along_axis(near, np.minimum(code + 1, 7)[..., None], -1)[..., 0])
        code = np.where(tie & (code % 2 == 1), code + 1, code)
        out[:, b:b + 32] = np.where(np.isfinite(top)[:, None], np.copysign(GRID[code], blk) * unit, np.nan)
    return out


def keep(bench, t, axis, shape, dtype=F32):
    L = bench.L
    q = L.pg_amd_mx4_quantize(t, axis)
    assert q, L.pg_autograd_last_error().decode()
    out = bench.unset(shape, dtype)
    bench.ok(L.pg_amd_mx4_dequantize(q, out))
    got = bench.read(out)
    L.pg_amd_mx4_free(q)
    return got


SHAPES = [(1, 1), (1, 32), (3, 31), (2, 33), (5, 64), (33, 100), (64, 256), (17, 257), (100, 500), (257, 1000)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("r,k", SHAPES)
def test_rounding(bench, dtype, axis, r, k):
    g = np.random.default_rng(r * k)
    v = rounded(g.standard_normal((r, k)) * np.exp(g.standard_normal((r, k)) * 2), dtype)
    a = v.T if axis == 0 else v
    want = quantized(v)
    want = want.T if axis == 0 else want
    got = keep(bench, bench.tensor(a, dtype), axis, a.shape)
    assert np.array_equal(got, want)
    assert np.array_equal(keep(bench, bench.transposed(a, dtype), axis, a.shape), want)
    for out in (F16, BF16):
        within(keep(bench, bench.tensor(a, dtype), axis, a.shape, out), rounded(want, out), 0, "rounded output")


@pytest.mark.parametrize("axis", [0, 1])
def test_ties_ends_and_what_is_no_number(bench, axis):
    rows = []
    exact = np.concatenate([GRID, -GRID, (GRID[1:] + GRID[:-1]) / 2, -(GRID[1:] + GRID[:-1]) / 2, [6.9, -7.9]])[:32]
    for scale in (1.0, 2.0 ** -20, 2.0 ** 100, 2.0 ** -126, 2.0 ** -140, 2.0 ** 124):
        rows.append(np.resize(exact, 32) * scale)
    rows.append(np.zeros(32))
    rows.append(np.full(32, -0.0))
    rows.append(np.full(32, np.finfo(np.float32).max))
    rows.append(np.resize([2.0 ** -149, -2.0 ** -149, 0, 2.0 ** -127], 32))
    rows.append(np.where(np.arange(32) == 5, np.nan, 1.0))
    rows.append(np.where(np.arange(32) == 31, np.inf, 1.0))
    rows.append(np.where(np.arange(32) == 0, -np.inf, 1.0))
    rows.append(np.resize([1.0, 1e-30], 32))
    v = np.asarray(rows, np.float32).astype(np.float64)
    v = np.concatenate([v, np.ones_like(v)], 1)  # the next block is its own
    a = v.T if axis == 0 else v
    want = quantized(v)
    got = keep(bench, bench.tensor(a), axis, a.shape)
    got = got.T if axis == 0 else got
    assert np.array_equal(got, want, equal_nan=True)
    assert np.isnan(got[10:13, :32]).all() and (got[10:13, 32:] == 1).all()
    assert np.array_equal(np.signbit(got[7, :32]), np.ones(32, bool))


def product(bench, x, w, dtype, out):
    """y, and what it should be, from f32 values."""
    L = bench.L
    q = L.pg_amd_mx4_quantize(bench.tensor(w), 0)
    assert q, L.pg_autograd_last_error().decode()
    y = bench.unset((x.shape[0], w.shape[1]), out)
    bench.ok(L.pg_amd_mx4_matmul(bench.tensor(x, dtype), q, y))
    got = bench.read(y)
    L.pg_amd_mx4_free(q)
    return got


PRODUCTS = [(1, 1, 1), (1, 32, 16), (1, 4096, 64), (2, 100, 33), (3, 257, 130), (8, 1000, 48), (15, 640, 100), (16, 512, 272),
            (17, 96, 65), (31, 300, 31), (33, 64, 64), (64, 2048, 40), (100, 130, 300), (128, 256, 128), (129, 288, 257),
            (257, 31, 129), (300, 1025, 520), (513, 544, 260)]


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16)],
                         ids=lambda d: NAMES[d])
@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_product(bench, dtype, out, m, k, n):
    g = np.random.default_rng(m + k + n)
    x = rounded(g.standard_normal((m, k)) * np.exp(g.standard_normal(k)), dtype)
    w = rounded(g.uniform(-1, 1, (k, n)) * k ** -0.5, F32)
    qx, qw = quantized(x), quantized(w.T).T
    want, size = qx @ qw, np.abs(qx) @ np.abs(qw)
    bound = (k + 2) * 2.0 ** -24 * size + TINY[F32]
    if out != F32:
        bound = bound + UNIT[out] * (np.abs(want) + bound) + TINY[out]
    within(product(bench, x, w, dtype, out), want, bound, "y")


# Sizes of every tile: 64 x 32 and 64 x 64 split eight ways, 64 x 64 split four
# ways, 128 x 128 in stages (one, two and several steps of 256 along the reduction).
TILES = [(640, 300, 640), (900, 260, 901), (1100, 900, 1210), (1100, 40, 1185), (1500, 100, 1600), (1601, 300, 1503),
         (1500, 700, 1601), (2000, 1025, 1300), (5000, 31, 600)]


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F32, F16)], ids=lambda d: NAMES[d])
@pytest.mark.parametrize("m,k,n", TILES)
def test_product_of_many_tiles(bench, dtype, out, m, k, n):
    g = np.random.default_rng(m + k + n)
    x = rounded(g.standard_normal((m, k)) * np.exp(g.standard_normal(k)), dtype)
    w = rounded(g.uniform(-1, 1, (k, n)) * k ** -0.5, F32)
    qx, qw = quantized(x), quantized(w.T).T
    want, size = qx @ qw, np.abs(qx) @ np.abs(qw)
    bound = (k + 2) * 2.0 ** -24 * size + TINY[F32]
    if out != F32:
        bound = bound + UNIT[out] * (np.abs(want) + bound) + TINY[out]
    within(product(bench, x, w, dtype, out), want, bound, "y")


@pytest.mark.parametrize("m", [1, 40, 300])
def test_a_block_that_is_nan_spoils_its_row_or_column_only(bench, m):
    g = np.random.default_rng(1)
    k, n = 200, 100
    x, w = rounded(g.standard_normal((m, k)), F32), rounded(g.standard_normal((k, n)), F32)
    w[150, 7] = np.nan
    w[3, n - 1] = np.inf
    if m > 1:
        x[m - 1, 199] = np.inf
    got = product(bench, x, w, F32, F32)
    bad = np.zeros((m, n), bool)
    bad[:, [7, n - 1]] = True
    if m > 1:
        bad[m - 1] = True
    assert np.array_equal(np.isnan(got), bad)


@pytest.mark.parametrize("m", [3, 200])
def test_wide_ranges_and_strides(bench, m):
    """Blocks of very different powers, and an x that is a transposed view."""
    L = bench.L
    g = np.random.default_rng(5)
    k, n = 320, 70
    x = rounded(g.standard_normal((m, k)) * 2.0 ** np.repeat(g.integers(-30, 30, k // 32), 32), F32)
    w = rounded(g.standard_normal((k, n)) * 2.0 ** np.repeat(g.integers(-30, 30, k // 32), 32)[:, None], F32)
    qx, qw = quantized(x), quantized(w.T).T
    q = L.pg_amd_mx4_quantize(bench.transposed(w), 0)
    y = bench.unset((m, n))
    bench.ok(L.pg_amd_mx4_matmul(bench.transposed(x), q, y))
    within(bench.read(y), qx @ qw, (k + 2) * 2.0 ** -24 * (np.abs(qx) @ np.abs(qw)), "y")
    L.pg_amd_mx4_free(q)


def test_the_same_call_gives_the_same_bits(bench):
    g = np.random.default_rng(3)
    for m, k, n in ((1, 2048, 512), (70, 999, 333)):
        x, w = rounded(g.standard_normal((m, k)), F32), rounded(g.standard_normal((k, n)), F32)
        first = product(bench, x, w, F32, F32)
        for _ in range(3):
            assert np.array_equal(product(bench, x, w, F32, F32), first)


def test_bytes(bench):
    L = bench.L
    q = L.pg_amd_mx4_quantize(bench.tensor(np.ones((256, 64))), 0)
    assert L.pg_amd_mx4_bytes(q) == 256 * 64 * 17 // 32
    L.pg_amd_mx4_free(q)
    L.pg_amd_mx4_free(None)
    assert L.pg_amd_mx4_bytes(None) == 0


def test_refusals(bench):
    L = bench.L
    t = bench.tensor(np.ones((64, 48)))
    for bad in ((None, 0), (t, 2), (t, -1), (bench.tensor(np.ones(64)), 0)):
        assert not L.pg_amd_mx4_quantize(*bad)
        assert "matrix" in L.pg_autograd_last_error().decode()
    q, other = L.pg_amd_mx4_quantize(t, 0), L.pg_amd_mx4_quantize(t, 1)
    bench.refused(L.pg_amd_mx4_dequantize(None, bench.unset((64, 48))), "shape")
    bench.refused(L.pg_amd_mx4_dequantize(q, None), "shape")
    bench.refused(L.pg_amd_mx4_dequantize(q, bench.unset((48, 64))), "shape")
    bench.refused(L.pg_amd_mx4_dequantize(q, bench.transposed(np.ones((64, 48)))), "contiguous")
    x, y = bench.tensor(np.ones((5, 64)), BF16), bench.unset((5, 48))
    bench.ok(L.pg_amd_mx4_matmul(x, q, y))
    bench.refused(L.pg_amd_mx4_matmul(None, q, y), "needs")
    bench.refused(L.pg_amd_mx4_matmul(x, None, y), "needs")
    bench.refused(L.pg_amd_mx4_matmul(x, q, None), "needs")
    bench.refused(L.pg_amd_mx4_matmul(x, other, y), "needs")  # its blocks do not run along the reduction
    bench.refused(L.pg_amd_mx4_matmul(bench.tensor(np.ones((5, 63)), BF16), q, y), "needs")
    bench.refused(L.pg_amd_mx4_matmul(x, q, bench.unset((4, 48))), "needs")
    bench.refused(L.pg_amd_mx4_matmul(x, q, bench.transposed(np.ones((5, 48)))), "contiguous")
    wide = bench.tensor(np.ones((64, 64)))
    q64 = L.pg_amd_mx4_quantize(wide, 0)
    bench.refused(L.pg_amd_mx4_matmul(wide, q64, wide), "overlaps")
    for p in (q, other, q64):
        L.pg_amd_mx4_free(p)


@pytest.mark.parametrize("k", [2 ** 24, 2 ** 24 - 33, 65535 * 256 + 1])
@pytest.mark.parametrize("axis", [0, 1])
def test_the_longest_blocked_dimension(bench, axis, k):
    """Up to 2^24 along the blocks, down a column as along a row: a pattern of 32 blocks, each times its own power."""
    g = np.random.default_rng(k)
    some = rounded(g.standard_normal((1, 1024)), F32)
    blocks = (k + 31) // 32
    power = np.repeat(2.0 ** (np.arange(blocks) % 61 - 30), 32)[:k]
    v = np.resize(some[0], k) * power
    want = np.resize(quantized(some)[0], k) * power
    if k % 32:
        want[blocks * 32 - 32:] = quantized(v[None, blocks * 32 - 32:])[0]
    shape = (k, 1) if axis == 0 else (1, k)
    assert np.array_equal(keep(bench, bench.tensor(v.reshape(shape)), axis, shape), want.reshape(shape))


@pytest.mark.parametrize("m", [1, 17])
def test_the_longest_reduction(bench, m):
    """2^24 terms of 0 or 1: every partial sum is exact."""
    k = 2 ** 24
    w = (np.arange(k) % 3 == 0).astype(np.float32)[:, None]
    assert (product(bench, np.ones((m, k), np.float32), w, BF16, F32) == w.sum(dtype=np.float64)).all()


def test_more_columns_than_a_launch_has_threads_for(bench):
    """2^27 columns of one value, 16 of them a tile of 512 threads."""
    n = 2 ** 27 + 40
    w = (np.arange(n, dtype=np.uint32) % 5).astype(np.float32)[None]
    x = bench.tensor(np.ones((1, 1)), BF16)
    q = bench.L.pg_amd_mx4_quantize(bench.tensor(w), 0)
    assert q, bench.L.pg_autograd_last_error().decode()
    y = bench.unset((1, n))
    bench.ok(bench.L.pg_amd_mx4_matmul(x, q, y))
    bench.L.pg_amd_mx4_free(q)
    assert np.array_equal(bench.L.read(y), w)


def inside(bench, a, dtype, skip):
    """A tensor of a's values that starts `skip` elements into its storage."""
    L, size = bench.L, np.asarray(a).size
    store = bench.tensor(np.concatenate([np.full(skip, 5.0), np.ravel(a)]), dtype)
    t = L.pg_tensor_view(store)
    bench.frees.append((L.pg_tensor_free, t))
    i = L.tinfo(t)
    i.dev += skip * i.elem_size
    i.numel, i.ndim = size, np.ndim(a)
    stride = size
    for d, n in enumerate(np.shape(a)):
        stride //= n
        i.shape[d], i.stride[d] = n, stride
    return t


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F32)], ids=lambda d: NAMES[d])
@pytest.mark.parametrize("m,k,n", [(3, 256, 64), (100, 256, 64), (1100, 128, 1600)])
def test_tensors_that_start_inside_their_storage(bench, dtype, out, m, k, n):
    """Rows whose lengths keep 16 bytes, but not where they start."""
    L = bench.L
    g = np.random.default_rng(m)
    x, w = rounded(g.standard_normal((m, k)), dtype), rounded(g.standard_normal((k, n)), dtype)
    qx, qw = quantized(x), quantized(w.T).T
    q, back, y = L.pg_amd_mx4_quantize(inside(bench, w, dtype, 1), 0), inside(bench, np.full((k, n), 777.0), out, 3), inside(
        bench, np.full((m, n), 777.0), out, 1)
    bench.ok(L.pg_amd_mx4_dequantize(q, back))
    bench.ok(L.pg_amd_mx4_matmul(inside(bench, x, dtype, 3), q, y))
    L.pg_amd_mx4_free(q)
    within(bench.read(back), rounded(qw, out), 0, "read back")
    bound = (k + 2) * 2.0 ** -24 * (np.abs(qx) @ np.abs(qw)) + TINY[F32]
    if out != F32:
        bound = bound + UNIT[out] * (np.abs(qx @ qw) + bound) + TINY[out]
    within(bench.read(y), qx @ qw, bound, "y")
