"""Layer norm (pg_amd_layernorm, pg_amd_layernorm_backward, pg_ag_layernorm)
against the formulas in 64 bits, and those against differences.

Bounds, with u = 2^-24 and A the mean of |x| over a row: a thread adds at most
32 terms and ten more levels join the threads (twenty with slices), so a mean
is off by em = 64 u A, a difference from it by em + u |c|, the variance by
(64 + 3) u of itself plus 2 em sigma + em^2, and rstd, half of that and its own
roundings, by er = 40 u + em rstd + (em rstd)^2 relative.  So n is off by
en = |n| (er + 2 u) + em rstd.  What follows adds its own roundings, and each
output the rounding to its type.
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


def out_bound(want, bound, dtype):
    return bound if dtype == F32 else bound + UNIT[dtype] * (np.abs(want) + bound) + TINY[dtype]


class Model:
    """y and the grads, each with the bound of its f32 value."""

    def __init__(self, x, w, b, dy=None, eps=EPS):
        d = x.shape[1]
        mean = x.mean(1, keepdims=True)
        c = x - mean
        rstd = 1 / np.sqrt((c * c).mean(1, keepdims=True) + eps)
        n = c * rstd
        em = 64 * U * np.abs(x).mean(1, keepdims=True)
        er = 40 * U + em * rstd + (em * rstd) ** 2
        en = np.abs(n) * (er + 2 * U) + em * rstd
        one = np.ones(d) if w is None else w
        self.stats, self.estats = np.concatenate([mean, rstd], 1), np.concatenate([em, rstd * er], 1)
        self.y = n * one + (0 if b is None else b)
        self.ey = np.abs(one) * en + U * np.abs(n * one) + U * np.abs(self.y) + TINY[F32]
        if dy is None:
            return
        h = dy * one
        c1, c2 = h.mean(1, keepdims=True), (h * n).mean(1, keepdims=True)
        e1 = 64 * U * np.abs(h).mean(1, keepdims=True)
        e2 = 64 * U * np.abs(h * n).mean(1, keepdims=True) + (np.abs(h) * en).mean(1, keepdims=True)
        self.dx = rstd * (h - c1 - n * c2)
        self.edx = rstd * ((np.abs(h) + np.abs(c1) + np.abs(n * c2)) * (er + 6 * U) + e1 + np.abs(n) * e2
                           + en * np.abs(c2)) + TINY[F32]
        # rows per block, the groups of a block, the blocks: at most 128 additions deep
        self.dw, self.db = (dy * n).sum(0), dy.sum(0)
        self.edw = (np.abs(dy) * en).sum(0) + 128 * U * np.abs(dy * n).sum(0) + TINY[F32]
        self.edb = 128 * U * np.abs(dy).sum(0) + TINY[F32]


def data(m, d, dtype, seed=0):
    g = np.random.default_rng(seed + 1000 * m + d)
    x = rounded(g.standard_normal((m, d)) * np.exp(0.5 * g.standard_normal(d)) + 0.5 * g.standard_normal(d), dtype)
    return (x, rounded(1 + 0.2 * g.standard_normal(d), F32), rounded(0.1 * g.standard_normal(d), F32),
            rounded(0.1 * g.standard_normal((m, d)), dtype))


def forward(bench, x, w, b, y, stats=None, eps=EPS):
    bench.ok(bench.L.pg_amd_layernorm(x, w, b, eps, y, stats))


# one chunk of a row and less, every number of threads per row and its ends, rows
# that start anywhere, one row and more rows than blocks, rows in slices
SHAPES = [(1, 1), (3, 1), (5, 2), (1, 3), (7, 8), (33, 10), (1000, 31), (300, 32), (257, 33), (4, 64), (40, 255), (65, 256),
          (9, 257), (3, 1000), (1030, 1023), (2, 1024), (5, 1025), (17, 2048), (6, 2049), (1, 4096), (2, 4097), (3, 8192),
          (2, 8200), (1, 16384), (2, 16391), (3, 32768), (2, 32775), (1, 65537), (5, 50001), (256, 9001), (257, 17000),
          (300, 33001)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m,d", SHAPES)
def test_forward_and_backward(bench, dtype, m, d):
    x, w, b, dy = data(m, d, dtype)
    eps = EPS if d > 1 else 0.25
    tx, tw, tb, tdy = bench.tensor(x, dtype), bench.tensor(w), bench.tensor(b), bench.tensor(dy, dtype)
    full = Model(x, w, b, dy, eps)
    for out in {dtype, F32}:
        y, stats = bench.unset((m, d), out), bench.unset((m, 2))
        forward(bench, tx, tw, tb, y, stats, eps)
        within(bench.read(y), full.y, out_bound(full.y, full.ey, out), "y")
        within(bench.read(stats), full.stats, full.estats + TINY[F32], "stats")
        dx, dw, db = bench.unset((m, d), out), bench.unset((d,)), bench.unset((d,))
        bench.ok(bench.L.pg_amd_layernorm_backward(tx, tw, stats, tdy, dx, dw, db))
        within(bench.read(dx), full.dx, out_bound(full.dx, full.edx, out), "dx")
        within(bench.read(dw), full.dw, full.edw, "dw")
        within(bench.read(db), full.db, full.edb, "db")
    # no weights, no stats
    bare = Model(x, None, None, dy, eps)
    y = bench.unset((m, d), dtype)
    forward(bench, tx, None, None, y, None, eps)
    within(bench.read(y), bare.y, out_bound(bare.y, bare.ey, dtype), "y without weights")
    dx = bench.unset((m, d), dtype)
    bench.ok(bench.L.pg_amd_layernorm_backward(tx, None, stats, tdy, dx, None, None))
    within(bench.read(dx), bare.dx, out_bound(bare.dx, bare.edx, dtype), "dx without weights")


def test_the_formulas_against_differences():
    g = np.random.default_rng(4)
    x, w, b, dy = (g.standard_normal(s) for s in ((3, 7), (7,), (7,), (3, 7)))
    m, step = Model(x, w, b, dy), 1e-5
    for v, got in ((x, m.dx), (w, m.dw), (b, m.db)):
        for i in range(v.size):
            keep = v.flat[i]
            v.flat[i] = keep + step
            up = (Model(x, w, b).y * dy).sum()
            v.flat[i] = keep - step
            down = (Model(x, w, b).y * dy).sum()
            v.flat[i] = keep
            # (f(x + s) - f(x - s)) / 2 s: s^2 f''' / 6 and 2^-52 |f| / s, each under 1e-8 here
            assert abs((up - down) / (2 * step) - got.flat[i]) < 1e-7


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m,d", [(5, 48), (3, 2049), (2, 40000)])
def test_each_output_alone_and_mixed_types(bench, dtype, m, d):
    L = bench.L
    x, w, b, dy = data(m, d, dtype, 1)
    tx, tw = bench.tensor(x, dtype), bench.tensor(w)
    stats = bench.unset((m, 2))
    forward(bench, tx, tw, None, bench.unset((m, d), dtype), stats)
    for gd in {dtype, F32}:
        want = Model(x, w, b, dy)
        tdy = bench.tensor(dy, gd)
        for out in {dtype, F32}:
            dx, dw, db = bench.unset((m, d), out), bench.unset((d,)), bench.unset((d,))
            bench.ok(L.pg_amd_layernorm_backward(tx, tw, stats, tdy, dx, None, None))
            bench.ok(L.pg_amd_layernorm_backward(tx, tw, stats, tdy, None, dw, None))
            bench.ok(L.pg_amd_layernorm_backward(tx, tw, stats, tdy, None, None, db))
            within(bench.read(dx), want.dx, out_bound(want.dx, want.edx, out), "dx")
            within(bench.read(dw), want.dw, want.edw, "dw")
            within(bench.read(db), want.db, want.edb, "db")
    bench.ok(L.pg_amd_layernorm_backward(tx, tw, stats, tdy, None, None, None))


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("d", [40, 777, 9000, 40001])
def test_in_place_and_three_dimensions(bench, dtype, d):
    x, w, b, _ = data(6, d, dtype, 2)
    t = bench.tensor(x.reshape(2, 3, d), dtype)
    forward(bench, t, bench.tensor(w), bench.tensor(b), t)
    want = Model(x, w, b)
    within(bench.read(t).reshape(6, d), want.y, out_bound(want.y, want.ey, dtype), "y in x's place")


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
def test_strided_inputs(bench, dtype):
    m, d = 21, 34
    x, w, b, dy = data(m, d, dtype, 3)
    stats, y = bench.unset((m, 2)), bench.unset((m, d), dtype)
    forward(bench, bench.transposed(x, dtype), bench.tensor(w), bench.tensor(b), y, stats)
    want = Model(x, w, b, dy)
    within(bench.read(y), want.y, out_bound(want.y, want.ey, dtype), "y")
    dx, dw = bench.unset((m, d), dtype), bench.unset((d,))
    bench.ok(bench.L.pg_amd_layernorm_backward(bench.transposed(x, dtype), bench.tensor(w), stats,
                                               bench.transposed(dy, dtype), dx, dw, None))
    within(bench.read(dx), want.dx, out_bound(want.dx, want.edx, dtype), "dx")
    within(bench.read(dw), want.dw, want.edw, "dw")


def inside(bench, a, dtype, skip):
    """A tensor of a's values that starts `skip` elements into its storage."""
    L, size = bench.L, np.asarray(a).size
    store = bench.tensor(np.concatenate([np.full(skip, 5.0), np.ravel(a), np.full(9, 6.0)]), dtype)
    t = L.pg_tensor_view(store)
    bench.frees.append((L.pg_tensor_free, t))
    i = L.tinfo(t)
    i.dev += skip * i.elem_size
    i.numel, i.ndim = size, np.ndim(a)
    stride = size
    for n, s in enumerate(np.shape(a)):
        stride //= s
        i.shape[n], i.stride[n] = s, stride
    return t, store


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("m,d", [(3, 64), (2, 4100), (2, 40000)])
def test_tensors_that_start_inside_their_storage(bench, dtype, m, d):
    """And what lies around the outputs stays as it was."""
    x, w, b, dy = data(m, d, dtype, 5)
    want = Model(x, w, b, dy)
    (y, sy), (dx, sdx), (stats, _) = (inside(bench, np.zeros(s), t, k) for s, t, k in (((m, d), dtype, 1), ((m, d), dtype, 3),
                                                                                      ((m, 2), F32, 2)))
    (dw, sdw), (db, sdb) = (inside(bench, np.zeros(d), F32, k) for k in (1, 3))
    tx, tw, tdy = inside(bench, x, dtype, 3)[0], inside(bench, w, F32, 1)[0], inside(bench, dy, dtype, 1)[0]
    forward(bench, tx, tw, inside(bench, b, F32, 3)[0], y, stats)
    bench.ok(bench.L.pg_amd_layernorm_backward(tx, tw, stats, tdy, dx, dw, db))
    for t, store, v, e, skip, dt in ((y, sy, want.y, want.ey, 1, dtype), (dx, sdx, want.dx, want.edx, 3, dtype),
                                     (dw, sdw, want.dw, want.edw, 1, F32), (db, sdb, want.db, want.edb, 3, F32)):
        whole = bench.read(store)
        within(whole[skip:-9].reshape(v.shape), v, out_bound(v, e, dt), "inside")
        assert (whole[:skip] == 5).all() and (whole[-9:] == 6).all()


@pytest.mark.parametrize("d", [20, 3000, 40000])
def test_what_is_no_number_stays_in_its_row(bench, d):
    m = 5
    x, w, b, dy = data(m, d, F32, 6)
    x[1, d - 1], x[3, 0] = np.nan, np.inf
    y, stats, dx = bench.unset((m, d)), bench.unset((m, 2)), bench.unset((m, d))
    dw, db = bench.unset((d,)), bench.unset((d,))
    tx, tw = bench.tensor(x), bench.tensor(w)
    forward(bench, tx, tw, bench.tensor(b), y, stats)
    bench.ok(bench.L.pg_amd_layernorm_backward(tx, tw, stats, bench.tensor(dy), dx, dw, db))
    good = [0, 2, 4]
    want = Model(x[good], w, b, dy[good])
    got, gdx = bench.read(y), bench.read(dx)
    assert np.isnan(got[[1, 3]]).all() and np.isnan(gdx[[1, 3]]).all()
    within(got[good], want.y, want.ey, "y")
    within(gdx[good], want.dx, want.edx, "dx")
    assert np.isnan(bench.read(dw)).all()
    within(bench.read(db), dy.sum(0), 128 * U * np.abs(dy).sum(0), "db")


@pytest.mark.parametrize("d", [7, 5000, 40000])
def test_rows_far_from_zero_and_of_equal_values(bench, d):
    """The variance is of the differences: rows at 1e4 with a spread of 1, large and small ones, equal values."""
    g = np.random.default_rng(7)
    x = rounded(np.stack([1e4 + g.standard_normal(d), 1e15 * (5 + g.standard_normal(d)), np.full(d, 3.0), np.zeros(d),
                          1e-30 * g.standard_normal(d)]), F32)
    y = bench.unset(x.shape)
    forward(bench, bench.tensor(x), None, None, y)
    want = Model(x, None, None)
    within(bench.read(y), want.y, want.ey, "y")
    # eps 0: rows of equal values have no norm
    forward(bench, bench.tensor(x[2:4]), None, None, y2 := bench.unset((2, d)), None, 0.0)
    assert np.isnan(bench.read(y2)).all()


@pytest.mark.parametrize("m,d", [(40, 24), (3000, 100), (4, 40000)])
def test_the_same_call_gives_the_same_bits(bench, m, d):
    x, w, b, dy = data(m, d, F32, 8)
    tx, tw, tb, tdy = (bench.tensor(v) for v in (x, w, b, dy))
    first = None
    for _ in range(3):
        outs = [bench.unset(s) for s in ((m, d), (m, 2), (m, d), (d,), (d,))]
        forward(bench, tx, tw, tb, outs[0], outs[1])
        bench.ok(bench.L.pg_amd_layernorm_backward(tx, tw, outs[1], tdy, *outs[2:]))
        got = [bench.L.read(t) for t in outs]
        assert first is None or all(np.array_equal(a, c) for a, c in zip(got, first))
        first = got


def test_many_rows(bench):
    """More rows than a grid of the forward has blocks for 32 rows each, and sums over all of them."""
    m, d = (1 << 25) + 77, 2
    row = rounded([1.0, -2.0], F32)
    L = bench.L
    x = bench.tensor(np.tile(row, (m, 1)), F16)
    y, stats, dw, db = (bench.unset(s, t) for s, t in (((m, d), F16), ((m, 2), F32), ((d,), F32), ((d,), F32)))
    forward(bench, x, None, None, y, stats)
    want = Model(row[None], None, None)
    got = L.read(y)
    assert (got == got[0]).all()
    within(rounded(np.float32(got[0].view(np.float16)), F32), want.y[0], out_bound(want.y, want.ey, F16)[0], "y")
    bench.ok(L.pg_amd_layernorm_backward(x, None, stats, x, None, dw, db))
    # 2^25 equal terms, 2^11 of them added one after the other, then the tree
    n = 2.0 ** 12 * U
    within(bench.read(db), m * row, n * m * np.abs(row), "db")
    within(bench.read(dw), m * row * want.y[0], 2 * n * m * np.abs(row * want.y[0]), "dw")


# ---------------------------------------------------------------- the node

def loss_of(L, n, r):
    """sum(n r) as a node, and the nodes to free."""
    p = L.op("mul", n, r)
    return L.op("sum_all", p), p


@pytest.mark.parametrize("jit", [True, False])
@pytest.mark.parametrize("m,d", [(1, 5), (40, 24), (130, 1030), (2, 20000)])
@pytest.mark.parametrize("weights", [(True, True), (True, False), (False, True), (False, False)])
def test_node(bench, m, d, weights, jit):
    L = bench.L
    x, w, b, dy = data(m, d, F32, 9)
    want = Model(x, w if weights[0] else None, b if weights[1] else None, dy)
    nx, nr = bench.var(x), bench.var(dy, False)
    nw, nb = (bench.var(v) if on else None for v, on in zip((w, b), weights))
    L.pg_autograd_set_jit(jit)
    try:
        n = bench.node(L.pg_ag_layernorm(nx, nw, nb, EPS))
        within(L.value(n), want.y, want.ey, "y")
        loss, p = (bench.node(v) for v in loss_of(L, n, nr))
        L.pg_backward(loss)
        within(L.grad(nx), want.dx, want.edx, "dx")
        if nw:
            within(L.grad(nw), want.dw, want.edw, "dw")
        if nb:
            within(L.grad(nb), want.db, want.edb, "db")
    finally:
        L.pg_autograd_set_jit(True)


def test_a_grad_of_ones(bench):
    L = bench.L
    x, w, b, _ = data(33, 70, F32, 13)
    nx, nw, nb = (bench.var(v) for v in (x, w, b))
    L.pg_backward(bench.node(L.op("sum_all", bench.node(L.pg_ag_layernorm(nx, nw, nb, EPS)))))
    want = Model(x, w, b, np.ones((33, 70)))
    within(L.grad(nx), want.dx, want.edx, "dx")
    within(L.grad(nw), want.dw, want.edw, "dw")
    assert (L.grad(nb) == 33).all()


def test_grads_add_to_what_is_there(bench):
    """One x under two norms with one weight: the grads are the sums."""
    L = bench.L
    m, d = 30, 50
    x, w, b, dy = data(m, d, F32, 10)
    nx, nw, nb, nr = bench.var(x), bench.var(w), bench.var(b), bench.var(dy, False)
    one, two = (bench.node(L.pg_ag_layernorm(nx, nw, nb, e)) for e in (EPS, 0.5))
    loss, *rest = loss_of(L, s := L.op("add", one, two), nr)
    for n in (s, loss, *rest):
        bench.node(n)
    L.pg_backward(loss)
    a, c = Model(x, w, b, dy), Model(x, w, b, dy, 0.5)
    within(L.grad(nx), a.dx + c.dx, a.edx + c.edx + U * np.abs(a.dx + c.dx), "dx")
    within(L.grad(nw), a.dw + c.dw, a.edw + c.edw + U * np.abs(a.dw + c.dw), "dw")
    within(L.grad(nb), a.db + c.db, a.edb + c.edb + U * np.abs(a.db + c.db), "db")


@pytest.mark.parametrize("d", [40, 20000])
@pytest.mark.parametrize("same", ["xw", "xb", "wb", "xwb"])
def test_one_node_as_several_operands(bench, same, d):
    L = bench.L
    g = np.random.default_rng(11)
    v = {k: rounded(g.standard_normal(d), F32) for k in "xwb"}
    dy = rounded(g.standard_normal((1, d)), F32)
    for k in same[1:]:
        v[k] = v[same[0]]
    nodes = {}
    for k in "xwb":
        nodes[k] = nodes[same[0]] if k in same and same[0] in nodes else bench.var(v[k])
    n = bench.node(L.pg_ag_layernorm(nodes["x"], nodes["w"], nodes["b"], EPS))
    nr = bench.var(dy[0], False)
    loss, p = loss_of(L, n, nr)
    bench.node(p)
    bench.node(loss)
    L.pg_backward(loss)
    m = Model(v["x"][None], v["w"], v["b"], dy)
    part = {"x": (m.dx[0], m.edx[0]), "w": (m.dw, m.edw), "b": (m.db, m.edb)}
    for k in "xwb":
        of = same if k in same else k
        want, bound = sum(part[i][0] for i in of), sum(part[i][1] for i in of) + 2 * U * sum(np.abs(part[i][0]) for i in of)
        within(L.grad(nodes[k]), want, bound, k)


def test_a_norm_between_layers(bench):
    """x W1 + b1, gelu, norm, W2 in bf16: the norm takes a deferred activation and feeds a 16-bit layer."""
    L = bench.L
    g = np.random.default_rng(12)
    m, k, d, n = 64, 48, 96, 33
    x, w1, b1, w2 = (rounded(g.standard_normal(s) * f, BF16) for s, f in (((m, k), 1), ((k, d), 0.2), ((d,), 0.1), ((d, n), 0.2)))
    lw, lb = rounded(1 + 0.1 * g.standard_normal(d), F32), rounded(0.1 * g.standard_normal(d), F32)
    nx, n1, nb1, nlw, nlb, n2 = (bench.var(v) for v in (x, w1, b1, lw, lb, w2))
    h = bench.node(L.pg_amd_ag_linear16(nx, n1, nb1, 2, BF16))
    y = bench.node(L.pg_ag_layernorm(h, nlw, nlb, EPS))
    z = bench.node(L.pg_amd_ag_linear16(y, n2, None, 0, BF16))
    hv = L.value(h).astype(np.float64)
    want = Model(hv, lw, lb)
    within(L.value(y), want.y, want.ey, "y")
    yq = rounded(L.value(y), BF16)
    within(L.value(z), yq @ w2, (d + 2) * U * (np.abs(yq) @ np.abs(w2)), "z")
    loss = bench.node(L.op("sum_all", z))
    L.pg_backward(loss)
    dz = np.ones((m, n))
    dy = dz @ w2.T
    back = Model(hv, lw, lb, dy)
    # dy from the products of bf16 ones and weights: f32 sums
    ey = (n + 2) * U * np.abs(w2).sum(1)
    within(L.grad(nlb), back.db, back.edb + m * ey, "db")
    within(L.grad(nlw), back.dw, back.edw + (ey * np.abs(back.y)).sum(0) + ey * m * 4, "dw")
    assert L.grad(n1) is not None and np.isfinite(L.grad(n1)).all()


def test_without_grads_nothing_is_kept(bench):
    L = bench.L
    x, w, b, _ = data(50, 64, F32, 13)
    nx, nw, nb = (bench.var(v, False) for v in (x, w, b))
    L.sync()
    before = L.pg_amd_bytes_in_use()
    n = L.pg_ag_layernorm(nx, nw, nb, EPS)
    assert L.pg_amd_bytes_in_use() - before <= 50 * 64 * 4 + 4096 and not L.node(n).requires_grad
    L.pg_node_free(n)
    L.pg_no_grad_push()
    n = bench.node(L.pg_ag_layernorm(bench.var(x), None, None, EPS))
    L.pg_no_grad_pop()
    assert not L.node(n).requires_grad


def test_empty_batches(bench):
    L = bench.L
    x, y, stats, dw, db = (bench.unset(s) for s in ((0, 5), (0, 5), (0, 2), (5,), (5,)))
    bench.ok(L.pg_amd_layernorm(x, None, None, EPS, y, stats))
    bench.ok(L.pg_amd_layernorm_backward(x, None, stats, y, None, dw, db))
    assert (bench.read(dw) == 0).all() and (bench.read(db) == 0).all()


def test_refusals(bench):
    L = bench.L
    x, y, s, w = bench.tensor(np.ones((4, 6))), bench.unset((4, 6)), bench.unset((4, 2)), bench.tensor(np.ones(6))
    h = bench.tensor(np.ones((4, 6)), BF16)
    fwd = lambda *a: L.pg_amd_layernorm(*a)  # noqa: E731
    bench.refused(fwd(None, None, None, EPS, y, None), "needs")
    bench.refused(fwd(bench.unset((4, 0)), None, None, EPS, y, None), "needs")
    bench.refused(fwd(x, bench.tensor(np.ones(5)), None, EPS, y, None), "weight")
    bench.refused(fwd(x, None, bench.tensor(np.ones(6), BF16), EPS, y, None), "weight")
    for eps in (-1e-5, float("nan"), float("inf")):
        bench.refused(fwd(x, None, None, eps, y, None), "eps")
    bench.refused(fwd(x, None, None, EPS, None, None), "shape")
    bench.refused(fwd(x, None, None, EPS, bench.unset((6, 4)), None), "shape")
    bench.refused(fwd(x, None, None, EPS, bench.unset((4, 6), F16), None), "shape")
    bench.refused(fwd(h, None, None, EPS, bench.unset((4, 6), F16), None), "shape")
    bench.refused(fwd(x, None, None, EPS, y, bench.unset((4, 3))), "stats")
    bench.refused(fwd(x, None, None, EPS, bench.transposed(np.ones((4, 6))), None), "contiguous")
    bench.refused(fwd(x, w, w, EPS, inside(bench, np.ones((4, 6)), F32, 2)[0], bench.transposed(np.ones((4, 2)))), "contiguous")
    store = bench.unset((10, 6))
    half = L.pg_tensor_view(store)
    bench.frees.append((L.pg_tensor_free, half))
    i = L.tinfo(half)
    i.shape[0], i.numel = 4, 24
    over = L.pg_tensor_view(store)
    bench.frees.append((L.pg_tensor_free, over))
    j = L.tinfo(over)
    j.shape[0], j.numel, j.dev = 4, 24, j.dev + 24
    bench.refused(fwd(half, None, None, EPS, over, None), "overlaps")
    bwd = lambda *a: L.pg_amd_layernorm_backward(*a)  # noqa: E731
    bench.refused(bwd(x, w, None, y, y, None, None), "stats")
    bench.refused(bwd(x, w, s, None, y, None, None), "dy")
    bench.refused(bwd(h, w, s, bench.unset((4, 6), F16), None, None, None), "dy")
    bench.refused(bwd(x, w, s, y, bench.unset((4, 6), BF16), None, None), "dx")
    bench.refused(bwd(x, w, s, y, None, bench.unset((5,)), None), "dw")
    bench.refused(bwd(x, w, s, y, y, None, None), "overlaps")
    d = bench.unset((6,))
    bench.refused(bwd(x, w, s, y, None, d, d), "overlaps")
    n, n16 = bench.var(np.ones((4, 6))), bench.node(L.var(np.zeros((4, 6), np.uint16), True, BF16))
    for bad in ((None, None, None, EPS), (n16, None, None, EPS), (n, bench.var(np.ones(5)), None, EPS), (n, None, n, EPS),
                (n, None, None, -1.0)):
        assert not L.pg_ag_layernorm(*bad)
        assert "layernorm" in L.pg_autograd_last_error().decode()
