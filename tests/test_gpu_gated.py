"""The gated layer (pg_amd_gated, pg_amd_gated_backward, pg_amd_ag_gated16)
against the formula in 64 bits on the same 16-bit operands, and its grads
against differences.

Bounds: a dot product of n terms in f32 is off by at most (n + 4) 2^-24 times
the sum of its terms' magnitudes; act and act' are within 2^-20 of their
argument's scale (a few units of f32 over an exponential); every rounding to
16 bits adds half a unit in the last place of what it rounds.
"""
import ctypes as C

import numpy as np
import pytest
from scipy.special import ndtr

from op_tools import NAMES, TINY, UNIT, Bench, rounded, within
from picograd_amd.capi import BF16, F16, F32, shape_arg

pytestmark = pytest.mark.gpu

ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}
F = 2.0 ** -24
MATH = 2.0 ** -20


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


def act64(g, act):
    """act(g) and act'(g)."""
    if act == "none":
        return g, np.ones_like(g)
    if act == "relu":
        return np.maximum(g, 0), (g > 0) * 1.0
    if act == "gelu":
        return g * ndtr(g), ndtr(g) + g * np.exp(-g * g / 2) / np.sqrt(2 * np.pi)
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-g))
    return (s, s * (1 - s)) if act == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def data(m, k, f, dtype, bias, seed=0):
    r = np.random.default_rng(seed)
    x = rounded(r.standard_normal((m, k)), dtype)
    w = rounded(r.uniform(-1, 1, (k, 2 * f)) * max(k, 1) ** -0.5, dtype)
    b = rounded(r.standard_normal(2 * f) * 0.1, F32) if bias else None
    dh = rounded(r.standard_normal((m, f)) * 0.5, dtype)
    return x, w, b, dh


def model(x, w, b, dh, act, dtype):
    """Values and bounds: name -> (value, f32 bound)."""
    f = w.shape[1] // 2
    z = x @ w + (0 if b is None else b)
    ez = (x.shape[1] + 4) * F * (np.abs(x) @ np.abs(w) + (0 if b is None else np.abs(b))) + TINY[F32]
    g, u, eg, eu = z[:, :f], z[:, f:], ez[:, :f], ez[:, f:]
    a, da = act64(g, act)
    ea = 1.2 * eg + MATH * (np.abs(a) + np.abs(g) * 2.0 ** -2)
    eda = 1.2 * eg + MATH * (1 + np.abs(g) * 2.0 ** -2)
    if act == "relu":
        eda = np.where(np.abs(g) <= eg, 1.0, 0.0)
    out = {"z": (z, ez), "h": (a * u, np.abs(a) * eu + np.abs(u) * ea + ea * eu + 2 * F * np.abs(a * u))}
    if dh is None:
        return out
    dz = np.concatenate([dh * u * da, dh * a], 1)
    e32 = np.concatenate([np.abs(dh) * (np.abs(u) * eda + np.abs(da) * eu + eda * eu), np.abs(dh) * ea], 1)
    e32 = e32 + 3 * F * np.abs(dz) + TINY[F32]
    e16 = e32 + UNIT[dtype] * (np.abs(dz) + e32) + TINY[dtype]
    m = x.shape[0]
    out["db"] = (dz.sum(0), e32.sum(0) + (m + 4) * F * np.abs(dz).sum(0))
    out["dx"] = (dz @ w.T, e16 @ np.abs(w).T + (2 * f + 4) * F * ((np.abs(dz) + e16) @ np.abs(w).T))
    out["dw"] = (x.T @ dz, np.abs(x).T @ e16 + (m + 4) * F * (np.abs(x).T @ (np.abs(dz) + e16)))
    return out


def check(got, pair, dtype, what):
    want, bound = pair
    within(got, want, bound + (0 if dtype == F32 else UNIT[dtype] * (np.abs(want) + bound) + TINY[dtype]), what)


SHAPES = [(1, 8, 8), (1, 1024, 512), (1, 7, 3), (2, 64, 32), (5, 33, 40), (16, 256, 136), (17, 100, 64), (33, 1000, 9),
          (64, 64, 64), (100, 72, 200), (130, 520, 129), (257, 40, 264), (300, 136, 1000)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m,k,f", SHAPES)
def test_forward_and_backward(bench, dtype, m, k, f):
    L = bench.L
    act = sorted(ACTS)[(m + k + f) % 5]
    x, w, b, dh = data(m, k, f, dtype, bias=(m + f) % 2 == 0)
    ref = model(x, w, b, dh, act, dtype)
    tx, tw, tb, th = bench.tensor(x, dtype), bench.tensor(w, dtype), None if b is None else bench.tensor(b), bench.tensor(dh, dtype)
    for hd in (dtype, F32):
        h, z = bench.unset((m, f), hd), bench.unset((m, 2 * f))
        bench.ok(L.pg_amd_gated(tx, tw, tb, ACTS[act], h, z))
        check(bench.read(h), ref["h"], hd, "h")
        check(bench.read(z), ref["z"], F32, "z")
        alone = bench.unset((m, f), hd)  # without z: the same values
        bench.ok(L.pg_amd_gated(tx, tw, tb, ACTS[act], alone, None))
        check(bench.read(alone), ref["h"], hd, "h alone")
    for gd in (dtype, F32):
        dx, dw, db = bench.unset((m, k), gd), bench.unset((k, 2 * f), gd), bench.unset((2 * f,))
        bench.ok(L.pg_amd_gated_backward(tx, tw, z, th, ACTS[act], dx, dw, db))
        check(bench.read(dx), ref["dx"], gd, "dx")
        check(bench.read(dw), ref["dw"], gd, "dw")
        check(bench.read(db), ref["db"], F32, "db")


# Large enough for every tile of the forward (few outputs of one row beside many;
# 128 x 128, 128 x 256 and 256 x 256 tiles at whole and odd widths), and for
# several strips of rows in the backward.
LARGE = [(1, 40, 4100), (3, 64, 5000), (16, 37, 4501), (300, 80, 1500), (512, 104, 4096), (500, 72, 4001), (1024, 64, 2048),
         (1023, 50, 2049), (1024, 72, 8192), (1001, 33, 8001), (2100, 48, 130)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m,k,f", LARGE)
def test_every_tile(bench, dtype, m, k, f):
    L, act = bench.L, sorted(ACTS)[(m + f) % 5]
    x, w, b, dh = data(m, k, f, dtype, bias=f % 3 != 0, seed=7)
    ref = model(x, w, b, dh, act, dtype)
    tx, tw, tb, th = bench.tensor(x, dtype), bench.tensor(w, dtype), None if b is None else bench.tensor(b), bench.tensor(dh, dtype)
    h, z = bench.unset((m, f), dtype), bench.unset((m, 2 * f))
    bench.ok(L.pg_amd_gated(tx, tw, tb, ACTS[act], h, z))
    check(bench.read(h), ref["h"], dtype, "h")
    check(bench.read(z), ref["z"], F32, "z")
    for gd in (dtype, F32):
        dx, dw, db = bench.unset((m, k), gd), bench.unset((k, 2 * f), gd), bench.unset((2 * f,))
        bench.ok(L.pg_amd_gated_backward(tx, tw, z, th, ACTS[act], dx, dw, db))
        check(bench.read(dx), ref["dx"], gd, "dx")
        check(bench.read(dw), ref["dw"], gd, "dw")
        check(bench.read(db), ref["db"], F32, "db")


# Sizes at which both products of the backward are one launch: in one to eight
# slices of the dgrad's reduction, at whole and odd widths.
BOTH = [(300, 1000, 1031), (257, 1030, 2048), (1000, 520, 2060), (1600, 2050, 600), (20, 1024, 2048), (129, 777, 1501),
        (520, 512, 1000)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m,k,f", BOTH)
def test_both_grads(bench, dtype, m, k, f):
    L = bench.L
    x, w, _, dh = data(m, k, f, dtype, False, seed=9)
    ref = model(x, w, None, dh, "silu", dtype)
    tx, tw, th, z = bench.tensor(x, dtype), bench.tensor(w, dtype), bench.tensor(dh, dtype), bench.tensor(ref["z"][0])
    for xd, wd in ((dtype, dtype), (F32, F32), (dtype, F32), (F32, dtype)):
        dx, dw = bench.unset((m, k), xd), bench.unset((k, 2 * f), wd)
        bench.ok(L.pg_amd_gated_backward(tx, tw, z, th, ACTS["silu"], dx, dw, None))
        check(bench.read(dx), ref["dx"], xd, "dx")
        check(bench.read(dw), ref["dw"], wd, "dw")


@pytest.mark.parametrize("dtype", [F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m,k,f", [(1, 64, 64), (3, 30, 68), (4, 700, 2000), (9, 129, 333), (16, 1024, 1030)])
def test_few_rows_round_once(bench, dtype, m, k, f):
    """Up to 16 rows [dg | du] is not rounded on the way to dx and dW: the bounds are those of f32."""
    L = bench.L
    x, w, _, dh = data(m, k, f, dtype, False, seed=13)
    z = rounded(x @ w, F32)
    a, da = act64(z[:, :f], "silu")
    u = z[:, f:]
    dz = np.concatenate([dh * u * da, dh * a], 1)
    e = np.abs(dh) * MATH * (1 + np.abs(z[:, :f]) * 2.0 ** -2)
    e = np.concatenate([np.abs(u) * e, e], 1) + 3 * F * np.abs(dz) + TINY[F32]
    dx, dw = bench.unset((m, k)), bench.unset((k, 2 * f))
    bench.ok(L.pg_amd_gated_backward(bench.tensor(x, dtype), bench.tensor(w, dtype), bench.tensor(z), bench.tensor(dh, dtype), 3,
                                     dx, dw, None))
    within(bench.read(dx), dz @ w.T, e @ np.abs(w).T + (2 * f + 4) * F * ((np.abs(dz) + e) @ np.abs(w).T), "dx")
    within(bench.read(dw), x.T @ dz, np.abs(x).T @ e + (m + 4) * F * (np.abs(x).T @ (np.abs(dz) + e)), "dw")


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m,f", [(3, 24), (40, 24), (200, 130)])
def test_every_activation(bench, act, m, f):
    L, dtype, k = bench.L, BF16, 48
    x, w, b, dh = data(m, k, f, dtype, True, seed=3)
    w = rounded(w * 6, dtype)  # gates into their flat ends
    ref = model(x, w, b, dh, act, dtype)
    t = [bench.tensor(x, dtype), bench.tensor(w, dtype), bench.tensor(b)]
    h, z = bench.unset((m, f), F32), bench.unset((m, 2 * f))
    bench.ok(L.pg_amd_gated(*t, ACTS[act], h, z))
    check(bench.read(h), ref["h"], F32, "h")
    dx, dw = bench.unset((m, k), F32), bench.unset((k, 2 * f), F32)
    dh32 = bench.tensor(dh)  # an f32 upstream grad
    bench.ok(L.pg_amd_gated_backward(t[0], t[1], z, dh32, ACTS[act], dx, dw, None))
    check(bench.read(dx), ref["dx"], F32, "dx")
    check(bench.read(dw), ref["dw"], F32, "dw")


def test_each_grad_alone_and_strided_inputs(bench):
    L, dtype, m, k, f = bench.L, F16, 37, 56, 48
    x, w, b, dh = data(m, k, f, dtype, True, seed=5)
    ref = model(x, w, b, dh, "silu", dtype)
    tx, tw, th = (bench.transposed(v, dtype) for v in (x, w, dh))
    h, z = bench.unset((m, f), dtype), bench.unset((m, 2 * f))
    bench.ok(L.pg_amd_gated(tx, tw, bench.tensor(b), 3, h, z))
    check(bench.read(h), ref["h"], dtype, "h")
    for name, shape, gd in (("dx", (m, k), dtype), ("dw", (k, 2 * f), F32), ("db", (2 * f,), F32)):
        g = bench.unset(shape, gd)
        args = {"dx": None, "dw": None, "db": None, name: g}
        bench.ok(L.pg_amd_gated_backward(tx, tw, z, th, 3, args["dx"], args["dw"], args["db"]))
        check(bench.read(g), ref[name], gd, name)


def test_a_nan_stays_in_its_row(bench):
    L, m, k, f = bench.L, 20, 40, 16
    x, w, b, dh = data(m, k, f, BF16, False)
    x[7, 3] = np.nan
    x[9, 0] = np.inf
    h = bench.unset((m, f), F32)
    bench.ok(L.pg_amd_gated(bench.tensor(x, BF16), bench.tensor(w, BF16), None, 3, h, None))
    got = bench.read(h)
    assert np.isnan(got[7]).all()
    rows = [i for i in range(m) if i not in (7, 9)]
    assert np.isfinite(got[rows]).all()


def test_empty_batches(bench):
    L, k, f = bench.L, 16, 24
    w = bench.tensor(np.ones((k, 2 * f)), BF16)
    nd, sh = shape_arg((0, k))
    x0 = L.pg_tensor_empty_dtype(BF16, nd, sh)
    h0 = L.pg_tensor_empty_dtype(BF16, 2, shape_arg((0, f))[1])
    z0 = L.pg_tensor_empty_dtype(F32, 2, shape_arg((0, 2 * f))[1])
    if not (x0 and h0 and z0):
        pytest.skip("no tensors without elements")
    bench.ok(L.pg_amd_gated(x0, w, None, 3, h0, z0))
    dw = bench.unset((k, 2 * f), F32)
    bench.ok(L.pg_amd_gated_backward(x0, w, z0, h0, 3, None, dw, None))
    assert (bench.read(dw) == 0).all()
    for t in (x0, h0, z0):
        L.pg_tensor_free(t)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m,k,f,bias", [(4, 16, 8, True), (64, 128, 256, False), (33, 50, 21, True), (128, 64, 72, True)])
def test_node(bench, dtype, m, k, f, bias):
    """f32 nodes, rounded to the 16-bit type; the grads add up over two nodes."""
    L = bench.L
    r = np.random.default_rng(11)
    x, w = r.standard_normal((m, k)).astype(np.float32), (r.uniform(-1, 1, (k, 2 * f)) * k ** -0.5).astype(np.float32)
    b = (r.standard_normal(2 * f) * 0.1).astype(np.float32) if bias else None
    dh = (r.standard_normal((m, f)) * 0.5).astype(np.float32)
    nx, nw, nb = bench.var(x), bench.var(w), bench.var(b) if bias else None
    ref = model(rounded(x, dtype), rounded(w, dtype), None if b is None else b.astype(np.float64), dh.astype(np.float64),
                "silu", dtype)
    seed = bench.tensor(dh)
    for times in (1, 2):
        h = bench.node(L.pg_amd_ag_gated16(nx, nw, nb, 3, dtype))
        check(L.value(h).astype(np.float64), ref["h"], F32, "h")
        if times == 2:  # two nodes over the same leaves
            h = bench.node(L.pg_ag_add(h, bench.node(L.pg_amd_ag_gated16(nx, nw, nb, 3, dtype))))
        L.pg_amd_backward_from(h, seed)
        for n, name in ((nx, "dx"), (nw, "dw")) + (((nb, "db"),) if bias else ()):
            want, bound = ref[name]
            within(L.grad(n), times * want, times * bound + 2 * F * np.abs(want), name)


def test_node_feeds_a_linear_layer(bench):
    """gated16 then linear16, their grads against differences of the f32 formula."""
    L, m, k, f, n = bench.L, 24, 32, 40, 16
    r = np.random.default_rng(2)
    x, wg, wd = r.standard_normal((m, k)), r.standard_normal((k, 2 * f)) * 0.3, r.standard_normal((f, n)) * 0.3
    x, wg, wd = (rounded(v, F16) for v in (x, wg, wd))  # nothing lost by the operands' rounding

    def loss(x, wg, wd):
        z = x @ wg
        g, u = z[:, :f], z[:, f:]
        return ((g / (1 + np.exp(-g)) * u) @ wd).sum()

    nodes = [bench.var(v) for v in (x, wg, wd)]
    h = bench.node(L.pg_amd_ag_gated16(nodes[0], nodes[1], None, 3, F16))
    y = bench.node(L.pg_amd_ag_linear16(h, nodes[2], None, 0, F16))
    total = bench.node(L.pg_ag_sum_all(y))
    L.pg_backward(total)
    for which, v in enumerate((x, wg, wd)):
        got = L.grad(nodes[which]).astype(np.float64)
        scale = np.abs(got).max()
        for _ in range(12):
            at = tuple(r.integers(0, s) for s in v.shape)
            args = [[a.copy() for a in (x, wg, wd)] for _ in range(2)]
            args[0][which][at] += 1e-5
            args[1][which][at] -= 1e-5
            slope = (loss(*args[0]) - loss(*args[1])) / 2e-5
            # three roundings to f16 (h, dz, the upstream grad) of values under the largest grad's scale
            assert abs(got[at] - slope) <= 8 * UNIT[F16] * scale, (which, at)


def test_node_without_grads_keeps_nothing(bench):
    L = bench.L
    x, w = bench.var(np.ones((4, 8)), False), bench.var(np.ones((8, 16)), False)
    n = bench.node(L.pg_amd_ag_gated16(x, w, None, 3, BF16))
    assert not L.node(n).ctx and not L.node(n).requires_grad


def test_one_tensor_as_both_operands(bench):
    """x and W in one storage: each of their grads lands in it."""
    L, k = bench.L, 32
    r = np.random.default_rng(4)
    v = rounded(r.standard_normal((k, k)) * 0.2, F16)
    dh = rounded(r.standard_normal((k, k // 2)), F16)
    n = bench.var(v)
    h = bench.node(L.pg_amd_ag_gated16(n, n, None, 3, F16))
    ref = model(v, v, None, dh, "silu", F16)
    check(L.value(h), ref["h"], F32, "h")
    L.pg_amd_backward_from(h, bench.tensor(dh))
    within(L.grad(n), ref["dx"][0] + ref["dw"][0], ref["dx"][1] + ref["dw"][1] + 2 * F * np.abs(ref["dx"][0] + ref["dw"][0]),
           "grad")


def test_refusals(bench):
    L = bench.L
    x, w, b = bench.tensor(np.ones((4, 8)), BF16), bench.tensor(np.ones((8, 12)), BF16), bench.tensor(np.ones(12))
    h, z = bench.unset((4, 6), BF16), bench.unset((4, 12))
    good = (x, w, b, 3, h, z)
    bench.ok(L.pg_amd_gated(*good))
    bench.refused(L.pg_amd_gated(None, *good[1:]), "null")
    bench.refused(L.pg_amd_gated(x, w, b, 5, h, z), "act")
    bench.refused(L.pg_amd_gated(x, w, b, -1, h, z), "act")
    bench.refused(L.pg_amd_gated(bench.tensor(np.ones((4, 8)), F16), *good[1:]), "dtype")
    bench.refused(L.pg_amd_gated(bench.tensor(np.ones((4, 8))), *good[1:]), "dtype")
    bench.refused(L.pg_amd_gated(bench.tensor(np.ones((4, 7)), BF16), *good[1:]), "x [M, K]")
    bench.refused(L.pg_amd_gated(x, bench.tensor(np.ones((8, 11)), BF16), None, 3, h, z), "x [M, K]")
    bench.refused(L.pg_amd_gated(x, w, bench.tensor(np.ones(6)), 3, h, z), "x [M, K]")
    bench.refused(L.pg_amd_gated(x, w, b, 3, bench.unset((4, 12), BF16), z), "h must be")
    bench.refused(L.pg_amd_gated(x, w, b, 3, bench.unset((4, 6), F16), z), "h must be")
    bench.refused(L.pg_amd_gated(x, w, b, 3, None, z), "h must be")
    bench.refused(L.pg_amd_gated(x, w, b, 3, h, bench.unset((4, 6))), "h must be")
    square = bench.tensor(np.ones((8, 16)), BF16)
    xs = bench.tensor(np.ones((8, 8)), BF16)
    bench.refused(L.pg_amd_gated(xs, square, None, 3, xs, None), "overlaps")
    dh, dx, dw, db = (bench.unset(s, BF16) for s in ((4, 6), (4, 8), (8, 12), (12,)))
    db = bench.unset((12,))
    bench.ok(L.pg_amd_gated_backward(x, w, z, dh, 3, dx, dw, db))
    bench.refused(L.pg_amd_gated_backward(x, w, None, dh, 3, dx, dw, db), "z f32")
    bench.refused(L.pg_amd_gated_backward(x, w, z, None, 3, dx, dw, db), "dh")
    bench.refused(L.pg_amd_gated_backward(x, w, z, bench.unset((4, 6), F16), 3, dx, dw, db), "dh")
    bench.refused(L.pg_amd_gated_backward(x, w, z, dh, 3, bench.unset((4, 6), BF16), dw, db), "dx must be")
    bench.refused(L.pg_amd_gated_backward(x, w, z, dh, 3, dx, bench.unset((8, 12), F16), db), "dx must be")
    bench.refused(L.pg_amd_gated_backward(x, w, z, dh, 3, dx, dw, bench.unset((6,))), "dx must be")
    bench.refused(L.pg_amd_gated_backward(x, w, z, dh, 3, x, dw, db), "overlaps")
    nx, nw = bench.var(np.ones((4, 8))), bench.var(np.ones((8, 12)))
    for bad, word in (((None, nw, None, 3, BF16), "null"), ((nx, nw, None, 3, F32), "dtype"),
                      ((nx, nw, None, 9, BF16), "act"), ((nx, nx, None, 3, BF16), "x [M, K]")):
        assert not L.pg_amd_ag_gated16(*bad)
        assert word in L.pg_autograd_last_error().decode()


@pytest.mark.parametrize("m,k2", [(40, 24), (512, 64), (3000, 40)])
def test_a_gated_row_as_the_bias_of_a_linear_layer(bench, m, k2):
    """The bias grad, whose last sums may wait for a later pass, is the gated node's upstream one."""
    L, k, f = bench.L, 24, 64
    r = np.random.default_rng(m)
    x, w, _, _ = data(1, k, f, BF16, False, seed=15)
    dy = r.integers(-8, 9, (m, f)) / 16.0  # its column sums are exact
    nodes = [bench.var(v) for v in (x, w, r.standard_normal((m, k2)), r.standard_normal((k2, f)))]
    h = bench.node(L.pg_amd_ag_gated16(nodes[0], nodes[1], None, 3, BF16))
    y = bench.node(L.pg_amd_ag_linear16(nodes[2], nodes[3], h, 0, BF16))
    L.pg_amd_backward_from(y, bench.tensor(dy))
    ref = model(x, w, None, dy.sum(0)[None], "silu", BF16)
    within(L.grad(h), dy.sum(0)[None], 0, "the bias grad")
    within(L.grad(nodes[0]), *ref["dx"], "dx")
    within(L.grad(nodes[1]), *ref["dw"], "dw")


@pytest.mark.parametrize("m,f", [(1, 1), (17, 8)])
def test_more_inputs_than_a_launch_has_threads_for(bench, m, f):
    """K past 2^27: 2^32 threads at 512 for 16 rows of W.  Operands of one value each, so that every sum is exact."""
    L, k = bench.L, 2 ** 27 + 40
    made = {}
    for name, shape, dtype, value in (("x", (m, k), F16, 0.5), ("w", (k, 2 * f), F16, 0.25), ("z", (m, 2 * f), F32, 2.0),
                                      ("dh", (m, f), F16, 1.0), ("dx", (m, k), F16, 777.0), ("dw", (k, 2 * f), F16, 777.0)):
        nd, sh = shape_arg(shape)
        made[name] = L.pg_tensor_full_dtype(dtype, nd, sh, value)
        assert made[name], L.pg_amd_last_error().decode()
    done = L.pg_amd_gated_backward(*(made[n] for n in ("x", "w", "z", "dh")), 0, made["dx"], made["dw"], None)
    get = L.lib.pg_tensor_get
    get.restype, get.argtypes = C.c_float, [C.c_void_p, C.POINTER(C.c_size_t)]
    at = [0, 5, 2 ** 26 - 1, 2 ** 26, 2 ** 27 - 17, 2 ** 27, k - 1]
    dx = [get(made["dx"], (C.c_size_t * 2)(m - 1, i)) for i in at] if done else []
    dw = [get(made["dw"], (C.c_size_t * 2)(i, 2 * f - 1)) for i in at] if done else []
    L.sync()
    for t in made.values():
        L.pg_tensor_free(t)
    L.lib.pg_tensor_pool_clear()
    bench.ok(done)
    # act NONE: [dg | du] = dh [u | g] = 2
    assert dx == [2 * 0.25 * 2 * f] * len(at) and dw == [0.5 * 2 * m] * len(at)


def test_more_rows_than_a_launch_has_threads_for_are_refused(bench):
    L = bench.L
    made = [L.pg_tensor_empty_dtype(F16, *shape_arg(s)) for s in ((2 ** 31 - 1, 1), (1, 2), (2 ** 31 - 1, 1))]
    assert all(made), L.pg_amd_last_error().decode()
    done = L.pg_amd_gated(made[0], made[1], None, 3, made[2], None)
    for t in made:
        L.pg_tensor_free(t)
    L.lib.pg_tensor_pool_clear()
    bench.refused(done, "x [M, K]")


@pytest.mark.parametrize("k", [4, 8, 16])
def test_one_tensor_as_both_operands_of_few_rows(bench, k):
    """Up to 16 rows, where both grads could be one launch: x's is added to W's in the one storage."""
    L = bench.L
    r = np.random.default_rng(k)
    v = rounded(r.standard_normal((k, k)) * 0.4, F16)
    dh = rounded(r.standard_normal((k, k // 2)), F16)
    n = bench.var(v)
    h = bench.node(L.pg_amd_ag_gated16(n, n, None, 3, F16))
    ref = model(v, v, None, dh, "silu", F16)
    check(L.value(h), ref["h"], F32, "h")
    L.pg_amd_backward_from(h, bench.tensor(dh))
    within(L.grad(n), ref["dx"][0] + ref["dw"][0], ref["dx"][1] + ref["dw"][1] + 2 * F * np.abs(ref["dx"][0] + ref["dw"][0]),
           "grad")


@pytest.mark.parametrize("m,f", [(3, 24), (40, 24), (40, 129)])
def test_an_empty_reduction(bench, m, f):
    """x [m, 0]: z is the bias, db what it is for any other layer."""
    L = bench.L
    _, _, b, dh = data(m, 1, f, BF16, True, seed=16)
    nd, sh = shape_arg((m, 0))
    x, w, dx, dw = (L.pg_tensor_empty_dtype(BF16, *shape_arg(s)) for s in ((m, 0), (0, 2 * f), (m, 0), (0, 2 * f)))
    if not (x and w and dx and dw):
        pytest.skip("no tensors without elements")
    ref = model(np.zeros((m, 0)), np.zeros((0, 2 * f)), b, dh, "gelu", BF16)
    h, z, db = bench.unset((m, f)), bench.unset((m, 2 * f)), bench.unset((2 * f,))
    bench.ok(L.pg_amd_gated(x, w, bench.tensor(b), 2, h, z))
    check(bench.read(z), (np.tile(b, (m, 1)), 0 * ref["z"][1]), F32, "z")
    check(bench.read(h), ref["h"], F32, "h")
    bench.ok(L.pg_amd_gated_backward(x, w, z, bench.tensor(dh, BF16), 2, dx, dw, db))
    check(bench.read(db), ref["db"], F32, "db")
    for t in (x, w, dx, dw):
        L.pg_tensor_free(t)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("f", [1, 4, 8])
def test_narrow_layers_of_many_inputs(bench, dtype, f):
    """dW of at most 16 columns and 1100 rows, in 16 bits and in f32."""
    L, m, k = bench.L, 40, 1100
    x, w, b, dh = data(m, k, f, dtype, True, seed=17)
    ref = model(x, w, b, dh, "silu", dtype)
    tx, tw, th = bench.tensor(x, dtype), bench.tensor(w, dtype), bench.tensor(dh, dtype)
    h, z = bench.unset((m, f), dtype), bench.unset((m, 2 * f))
    bench.ok(L.pg_amd_gated(tx, tw, bench.tensor(b), 3, h, z))
    check(bench.read(h), ref["h"], dtype, "h")
    for gd in (dtype, F32):
        dx, dw, db = bench.unset((m, k), gd), bench.unset((k, 2 * f), gd), bench.unset((2 * f,))
        bench.ok(L.pg_amd_gated_backward(tx, tw, z, th, 3, dx, dw, db))
        check(bench.read(dx), ref["dx"], gd, "dx")
        check(bench.read(dw), ref["dw"], gd, "dw")
        check(bench.read(db), ref["db"], F32, "db")


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


@pytest.mark.parametrize("dtype", [F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m,k,f", [(3, 64, 40), (40, 64, 40), (300, 136, 520), (512, 1024, 2048)])
def test_tensors_that_start_inside_their_storage(bench, dtype, m, k, f):
    """Operands and outputs none of which starts on 16 bytes."""
    L = bench.L
    x, w, b, dh = data(m, k, f, dtype, True, seed=18)
    ref = model(x, w, b, dh, "silu", dtype)
    tx, tw, th = (inside(bench, v, dtype, s) for v, s in ((x, 1), (w, 3), (dh, 5)))
    h, z = inside(bench, np.full((m, f), 777.0), dtype, 7), inside(bench, np.full((m, 2 * f), 777.0), F32, 1)
    bench.ok(L.pg_amd_gated(tx, tw, inside(bench, b, F32, 1), 3, h, z))
    check(bench.read(h), ref["h"], dtype, "h")
    check(bench.read(z), ref["z"], F32, "z")
    for gd in (dtype, F32):
        dx, dw, db = (inside(bench, np.full(s, 777.0), d, n) for s, d, n in (((m, k), gd, 3), ((k, 2 * f), gd, 1), (2 * f, F32, 1)))
        bench.ok(L.pg_amd_gated_backward(tx, tw, z, th, 3, dx, dw, db))
        check(bench.read(dx), ref["dx"], gd, "dx")
        check(bench.read(dw), ref["dw"], gd, "dw")
        check(bench.read(db), ref["db"], F32, "db")
