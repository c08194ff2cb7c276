"""8-bit matrices (pg_amd_q8_*) against the definition: the rounding bit for
bit, the product within the roundings of its exact sum, of that times each scale
(three of 2^-24) and of the output.
"""
import numpy as np
import pytest

from op_tools import NAMES, TINY, UNIT, Bench, rounded, within
from picograd_amd.capi import BF16, F16, F32

pytestmark = pytest.mark.gpu


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


def parts(v):
    """v [R, K] (f32 values in 64 bits) as whole numbers and a scale per row."""
    v = np.asarray(v, np.float64)
    top = np.abs(v).max(1)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        # two roundings meet only where 64 bits already decide: the quotient by 127 is no tie of 24 bits
        s = np.where(np.isfinite(top), (top / 127).astype(np.float32).astype(np.float64), np.nan)
        q = np.where(s[:, None] > 0, np.clip(np.rint(v / s[:, None]), -127, 127), 0)
    return q, s


def quantized(v):
    q, s = parts(v)
    with np.errstate(over="ignore"):
        return (q * s[:, None]).astype(np.float32).astype(np.float64)


def keep(bench, t, axis, shape, dtype=F32):
    L = bench.L
    q = L.pg_amd_q8_quantize(t, axis)
    assert q, L.pg_autograd_last_error().decode()
    out = bench.unset(shape, dtype)
    bench.ok(L.pg_amd_q8_dequantize(q, out))
    got = bench.read(out)
    L.pg_amd_q8_free(q)
    return got


SHAPES = [(1, 1), (1, 15), (1, 16), (3, 17), (2, 127), (5, 128), (33, 129), (64, 256), (17, 257), (100, 500), (257, 1000),
          (3, 2048), (2, 2049), (65, 8192), (3, 8193), (2, 16384), (1, 40001)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("r,k", SHAPES)
def test_rounding(bench, dtype, axis, r, k):
    g = np.random.default_rng(r * k)
    v = rounded(g.standard_normal((r, k)) * np.exp(g.standard_normal((r, k))), dtype)
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
    """Scales that are powers of two make ties exact; every step between two codes, and its neighbours in f32."""
    rows = []
    half = np.arange(-127, 127) + 0.5
    near = np.float32(half)
    exact = np.concatenate([half, np.nextafter(near, np.float32(300)), np.nextafter(near, np.float32(-300)), [127.0, -127.0],
                            np.zeros(4)]).astype(np.float64)
    for power in (0, -20, 100, -100, -119, -120, -121, -126, -130, -140):
        with np.errstate(under="ignore"):
            rows.append(np.float32(np.ldexp(exact, power)).astype(np.float64))
    n = len(exact)
    top = np.float64(np.finfo(np.float32).max)
    rows += [np.zeros(n), np.full(n, -0.0), np.full(n, top), np.resize([2.0 ** -149, -2.0 ** -149, 0, 2.0 ** -142], n),
             np.resize([2.0 ** -149], n), np.where(np.arange(n) == 5, np.nan, 1.0), np.where(np.arange(n) == n - 1, np.inf, 1.0),
             np.where(np.arange(n) == 0, -np.inf, 1.0), np.resize([1.0, 1e-30], n), np.resize([top, -top / 254, top / 127 * 2.5], n)]
    v = rounded(np.stack(rows), F32)
    a = v.T if axis == 0 else v
    got = keep(bench, bench.tensor(a), axis, a.shape)
    got = got.T if axis == 0 else got
    assert np.array_equal(got, quantized(v), equal_nan=True)
    assert np.isnan(got[15:18]).all() and (got[14] == 0).all()


def product(bench, x, w, dtype, out):
    """y from f32 values."""
    L = bench.L
    q = L.pg_amd_q8_quantize(bench.tensor(w), 0)
    assert q, L.pg_autograd_last_error().decode()
    y = bench.unset((x.shape[0], w.shape[1]), out)
    bench.ok(L.pg_amd_q8_matmul(bench.tensor(x, dtype), q, y))
    got = bench.read(y)
    L.pg_amd_q8_free(q)
    return got


def wanted(x, w, out):
    (qx, sx), (qw, sw) = parts(x), parts(w.T)
    y = (qx @ qw.T) * sx[:, None] * sw
    bound = 3.01 * 2.0 ** -24 * np.abs(y) + TINY[F32]
    return y, bound if out == F32 else bound + UNIT[out] * (np.abs(y) + bound) + TINY[out]


def case(m, k, n, dtype):
    g = np.random.default_rng(m + 7 * k + 31 * n)
    x = rounded(g.standard_normal((m, k)) * np.exp(0.5 * g.standard_normal(k)), dtype)
    return x, rounded(g.uniform(-1, 1, (k, n)) * k ** -0.5, F32)


PRODUCTS = [(1, 1, 1), (1, 16, 16), (1, 4096, 64), (2, 100, 33), (3, 257, 130), (8, 1000, 48), (15, 640, 100), (16, 512, 272),
            (16, 3001, 40), (1, 20000, 20), (17, 96, 65), (31, 300, 31), (33, 64, 64), (64, 2048, 40), (100, 130, 300),
            (128, 256, 128), (129, 288, 257), (257, 31, 129), (300, 1025, 520), (513, 544, 260)]


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16)],
                         ids=lambda d: NAMES[d])
@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_product(bench, dtype, out, m, k, n):
    x, w = case(m, k, n, dtype)
    within(product(bench, x, w, dtype, out), *wanted(x, w, out), "y")


# Sizes of every tile: 64 x 32 and 64 x 64 split eight ways, 64 x 64 split four
# ways, 128 x 128 and 256 x 256 in stages (one, two and several of 128 along the reduction).
TILES = [(640, 300, 640), (900, 260, 901), (1100, 900, 1210), (1100, 40, 1185), (1500, 100, 1600), (1601, 300, 1503),
         (1500, 700, 1601), (2000, 1025, 1300), (5000, 31, 600), (3500, 128, 3601), (3585, 129, 3600), (4000, 600, 3500),
         (50000, 20, 260)]


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F32, F16)], ids=lambda d: NAMES[d])
@pytest.mark.parametrize("m,k,n", TILES)
def test_product_of_many_tiles(bench, dtype, out, m, k, n):
    x, w = case(m, k, n, dtype)
    within(product(bench, x, w, dtype, out), *wanted(x, w, out), "y")


@pytest.mark.parametrize("m", [1, 40, 300, 4000])
def test_a_line_that_is_nan_spoils_its_row_or_column_only(bench, m):
    k, n = 200, 100 if m < 4000 else 4000
    x, w = case(m, k, n, F32)
    w[150, 7], w[3, n - 1] = np.nan, np.inf
    if m > 1:
        x[m - 1, 199] = np.inf
    got = product(bench, x, w, F32, F32)
    bad = np.zeros((m, n), bool)
    bad[:, [7, n - 1]] = True
    if m > 1:
        bad[m - 1] = True
    assert np.array_equal(np.isnan(got), bad)


@pytest.mark.parametrize("m", [3, 16, 200])
def test_wide_ranges_zero_rows_and_strides(bench, m):
    """Rows and columns of very different scales, empty ones, and an x that is a transposed view."""
    L = bench.L
    g = np.random.default_rng(5)
    k, n = 320, 70
    x = rounded(g.standard_normal((m, k)) * 2.0 ** g.integers(-30, 30, m)[:, None], F32)
    w = rounded(g.standard_normal((k, n)) * 2.0 ** g.integers(-30, 30, n), F32)
    x[1], w[:, 5] = 0, 0
    q = L.pg_amd_q8_quantize(bench.transposed(w), 0)
    y = bench.unset((m, n))
    bench.ok(L.pg_amd_q8_matmul(bench.transposed(x), q, y))
    within(bench.read(y), *wanted(x, w, F32), "y")
    assert (bench.read(y)[1] == 0).all() and (bench.read(y)[:, 5] == 0).all()
    L.pg_amd_q8_free(q)


@pytest.mark.parametrize("m", [3, 16, 200, 4000])
@pytest.mark.parametrize("up", [True, False])
def test_ranges_that_meet_in_the_middle(bench, m, up):
    """A sum times x's scale leaves f32 before the weights' scale brings it back."""
    g = np.random.default_rng(6)
    k, n = 1000, 70
    x, w = rounded(np.abs(g.standard_normal((m, k))), F32), rounded(np.abs(g.standard_normal((k, n))), F32)
    p = 2.0 ** (119 if up else -110)
    within(product(bench, x * p, w / p, F32, F32), *wanted(x * p, w / p, F32), "y")


@pytest.mark.parametrize("m", [1, 17, 300])
def test_the_longest_reduction_is_exact(bench, m):
    """2^17 products of 127 and 127 or -127: sums of up to 2^17 127^2, next to the ends of 32 bits."""
    k = 2 ** 17
    w = np.stack([np.full(k, 127.0), np.full(k, -127.0), np.where(np.arange(k) % 3 == 0, -127.0, 127.0)], 1)
    got = product(bench, np.full((m, k), 127.0), w, BF16, F32)
    want = 127.0 * w.sum(0)
    assert (np.abs(got - want) <= 2.0 ** -24 * np.abs(want)).all()  # the one rounding: the scales are 1


def test_the_same_call_gives_the_same_bits(bench):
    for m, k, n in ((1, 2048, 512), (70, 999, 333), (4000, 300, 3800)):
        x, w = case(m, k, n, F32)
        first = product(bench, x, w, F32, F32)
        for _ in range(2):
            assert np.array_equal(product(bench, x, w, F32, F32), first)


def test_rows_do_not_depend_on_their_batch(bench):
    """The sums are exact, so a row alone has the bits that it has in any batch."""
    x, w = case(4500, 700, 3700, BF16)
    L = bench.L
    q = L.pg_amd_q8_quantize(bench.tensor(w), 0)
    got = {}
    for m in (1, 16, 17, 300, 1400, 4500):
        y = bench.unset((m, 3700))
        bench.ok(L.pg_amd_q8_matmul(bench.tensor(x[:m], BF16), q, y))
        got[m] = L.read(y)
    L.pg_amd_q8_free(q)
    for m, y in got.items():
        assert np.array_equal(y, got[4500][:m]), m


def inside(bench, a, dtype, skip):
    """A tensor of a's values that starts `skip` elements into its storage, and the storage."""
    L, size = bench.L, np.asarray(a).size
    store = bench.tensor(np.concatenate([np.full(skip, 5.0), np.ravel(a), np.full(9, 6.0)]), dtype)
    t = L.pg_tensor_view(store)
    bench.frees.append((L.pg_tensor_free, t))
    i = L.tinfo(t)
    i.dev += skip * i.elem_size
    i.numel, i.ndim = size, np.ndim(a)
    stride = size
    for d, n in enumerate(np.shape(a)):
        stride //= n
        i.shape[d], i.stride[d] = n, stride
    return t, store


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F32)], ids=lambda d: NAMES[d])
@pytest.mark.parametrize("m,k,n", [(3, 256, 64), (100, 256, 64), (1100, 128, 1600), (1500, 130, 1601)])
def test_tensors_that_start_inside_their_storage(bench, dtype, out, m, k, n):
    """Rows whose lengths keep 16 bytes, but not where they start; what lies around the outputs stays."""
    L = bench.L
    x, w = case(m, k, n, dtype)
    w = rounded(w, dtype)
    q = L.pg_amd_q8_quantize(inside(bench, w, dtype, 1)[0], 0)
    (back, sb), (y, sy) = inside(bench, np.full((k, n), 777.0), out, 3), inside(bench, np.full((m, n), 777.0), out, 1)
    bench.ok(L.pg_amd_q8_dequantize(q, back))
    bench.ok(L.pg_amd_q8_matmul(inside(bench, x, dtype, 3)[0], q, y))
    L.pg_amd_q8_free(q)
    for store, skip in ((sb, 3), (sy, 1)):
        v = bench.read(store)
        assert (v[:skip] == 5).all() and (v[-9:] == 6).all()
    within(bench.read(back), rounded(quantized(w.T).T, out), 0, "read back")
    within(bench.read(y), *wanted(x, w, out), "y")


def test_bytes_and_empty_batches(bench):
    L = bench.L
    q = L.pg_amd_q8_quantize(bench.tensor(np.ones((256, 64))), 0)
    assert L.pg_amd_q8_bytes(q) == 256 * 64 + 64 * 4
    bench.ok(L.pg_amd_q8_matmul(bench.unset((0, 256)), q, bench.unset((0, 64))))
    L.pg_amd_q8_free(q)
    L.pg_amd_q8_free(None)
    assert L.pg_amd_q8_bytes(None) == 0


def test_refusals(bench):
    L = bench.L
    t = bench.tensor(np.ones((64, 48)))
    for bad in ((None, 0), (t, 2), (t, -1), (bench.tensor(np.ones(64)), 0), (bench.unset((0, 4)), 0),
                (bench.tensor(np.ones((2 ** 17 + 1, 2)), BF16), 0), (bench.tensor(np.ones((2, 2 ** 17 + 1)), BF16), 1)):
        assert not L.pg_amd_q8_quantize(*bad)
        assert "matrix" in L.pg_autograd_last_error().decode()
    q, other = L.pg_amd_q8_quantize(t, 0), L.pg_amd_q8_quantize(t, 1)
    bench.refused(L.pg_amd_q8_dequantize(None, bench.unset((64, 48))), "shape")
    bench.refused(L.pg_amd_q8_dequantize(q, None), "shape")
    bench.refused(L.pg_amd_q8_dequantize(q, bench.unset((48, 64))), "shape")
    bench.refused(L.pg_amd_q8_dequantize(q, bench.transposed(np.ones((64, 48)))), "contiguous")
    x, y = bench.tensor(np.ones((5, 64)), BF16), bench.unset((5, 48))
    bench.ok(L.pg_amd_q8_matmul(x, q, y))
    bench.refused(L.pg_amd_q8_matmul(None, q, y), "needs")
    bench.refused(L.pg_amd_q8_matmul(x, None, y), "needs")
    bench.refused(L.pg_amd_q8_matmul(x, q, None), "needs")
    bench.refused(L.pg_amd_q8_matmul(x, other, y), "needs")  # its lines do not run along the reduction
    bench.refused(L.pg_amd_q8_matmul(bench.tensor(np.ones((5, 63)), BF16), q, y), "needs")
    bench.refused(L.pg_amd_q8_matmul(x, q, bench.unset((4, 48))), "needs")
    bench.refused(L.pg_amd_q8_matmul(x, q, bench.transposed(np.ones((5, 48)))), "contiguous")
    wide = bench.tensor(np.ones((64, 64)))
    q64 = L.pg_amd_q8_quantize(wide, 0)
    bench.refused(L.pg_amd_q8_matmul(wide, q64, wide), "overlaps")
    for p in (q, other, q64):
        L.pg_amd_q8_free(p)
