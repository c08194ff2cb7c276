"""Distillation from a teacher's top logits (pg_amd_distill,
pg_amd_ag_distill) against the definition in 64 bits, and the grad against
differences.

Bounds: the f32 logits, maxima and indices are exact inputs.  An exponential
of d = (s - max) / T is off by (|d| + 4) 2^-23 relative, of which |d| e^d is at
most 0.4; a sum of V terms by V / 256 + 32 units more (every thread adds at
most V / 256 of them, the rest is a tree); a logarithm by 4 units of its value
or of 1.  So q, p and r carry eps = (V / 256 + 64) 2^-24 of each element's size
plus (|d| + 4) 2^-23 of the element itself.
"""
import ctypes as C

import numpy as np
import pytest

from op_tools import NAMES, TINY, UNIT, Bench, rounded, within
from picograd_amd.capi import BF16, F16, F32, DistillCfg, shape_arg

pytestmark = pytest.mark.gpu


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


def softmax(v):
    with np.errstate(invalid="ignore"):
        e = np.exp(v - v.max())
        return e / e.sum()


def model(s, t, idx, label, T, alpha, scale):
    """loss, its bound, ds, its bound."""
    n, v = s.shape
    loss, eloss, ds, eds = np.zeros(n), np.zeros(n), np.zeros((n, v)), np.zeros((n, v))
    eps = (v / 256 + 64) * 2.0 ** -24
    for i in range(n):
        there = (idx[i] >= 0) & (idx[i] < v) & ~np.isneginf(t[i])
        lab = -1 if label is None or not 0 <= label[i] < v or alpha == 1 else int(label[i])
        y = s[i] / T
        if there.any() and alpha > 0:
            p = softmax(t[i][there] / T)
            at = idx[i][there].astype(int)
            with np.errstate(divide="ignore", invalid="ignore"):
                d = y - y.max()
                logq = d - np.log(np.exp(d).sum())
                q = softmax(y)
                loss[i] += alpha * T * T * (p * (np.log(p) - logq[at])).sum()
                size = (p * (np.abs(np.log(p)) + np.abs(logq[at]) + 4)).sum()
            eloss[i] += alpha * T * T * (eps + 2.0 ** -20) * size
            g = q.copy()
            np.subtract.at(g, at, p)
            both = q.copy()
            np.add.at(both, at, p)
            ds[i] += alpha * T * g
            eds[i] += alpha * T * (eps + 2.0 ** -20 + np.where(np.isfinite(d), np.abs(d), 0) * 2.0 ** -22) * both
        if lab >= 0:
            with np.errstate(divide="ignore", invalid="ignore"):
                d = s[i] - s[i].max()
                logr = d - np.log(np.exp(d).sum())
                r = softmax(s[i])
            loss[i] -= (1 - alpha) * logr[lab]
            eloss[i] += (1 - alpha) * (eps + 2.0 ** -20) * (np.abs(logr[lab]) + 4)
            g = r.copy()
            g[lab] -= 1
            ds[i] += (1 - alpha) * g
            r[lab] += 1
            eds[i] += (1 - alpha) * (eps + 2.0 ** -20 + np.where(np.isfinite(d), np.abs(d), 0) * 2.0 ** -22) * r
    return scale * loss, abs(scale) * eloss + TINY[F32], scale * ds, abs(scale) * eds + TINY[F32]


def data(n, v, top, dtype, labels, seed=0):
    r = np.random.default_rng(seed)
    s = rounded(r.standard_normal((n, v)) * 2, dtype)
    t = rounded(r.standard_normal((n, top)) * 2 + 4, F32)
    idx = np.stack([r.choice(v, top, replace=top > v) for _ in range(n)]).astype(np.float64)
    idx[r.random((n, top)) < 0.15] = -1
    lab = r.integers(0, v, n).astype(np.float64) if labels else None
    if labels:
        lab[r.random(n) < 0.2] = -1
    if n > 2:
        idx[1] = -1  # a row that the teacher says nothing about
        if labels:
            lab[1] = -1
    return s, t, idx, lab


def go(bench, s, t, idx, lab, T, alpha, scale, dtype, out=None, inplace=False, top_dtype=F32):
    """loss and grad as the library gives them."""
    L = bench.L
    n, v = s.shape
    ts = bench.tensor(s, dtype)
    args = [ts, bench.tensor(t, top_dtype), bench.tensor(idx), None if lab is None else bench.tensor(lab)]
    cfg = DistillCfg(T, alpha, scale)
    loss = bench.unset((n,))
    ds = ts if inplace else bench.unset((n, v), dtype if out is None else out)
    alone = bench.unset((n,))
    bench.ok(L.pg_amd_distill(*args, C.byref(cfg), alone, None))
    bench.ok(L.pg_amd_distill(*args, C.byref(cfg), loss, ds))
    a, b = bench.read(alone), bench.read(loss)
    # the loss alone may add its sums in another order
    assert np.array_equal(np.isnan(a), np.isnan(b)), "the loss alone"
    return a, b, bench.read(ds)


def check(bench, s, t, idx, lab, T, alpha, scale, dtype, **kw):
    alone, loss, ds = go(bench, s, t, idx, lab, T, alpha, scale, dtype, **kw)
    wl, el, wd, ed = model(s, rounded(t, kw.get("top_dtype", F32)), idx, lab, np.float64(np.float32(T)),
                           np.float64(np.float32(alpha)), np.float64(np.float32(scale)))
    within(loss, wl, el, "loss")
    within(alone, wl, el, "loss alone")
    out = kw.get("out")
    out = dtype if out is None else out
    within(ds, wd, ed + (0 if out == F32 else UNIT[out] * (np.abs(wd) + ed) + TINY[out]), "grad")


SHAPES = [(1, 1, 1), (1, 2, 1), (3, 10, 4), (7, 63, 5), (64, 10, 10), (300, 17, 3), (5, 64, 64), (4, 65, 9), (2, 1000, 100),
          (9, 1023, 16), (3, 4096, 256), (2, 5001, 33), (1, 20000, 64)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("labels", [False, True])
@pytest.mark.parametrize("n,v,top", SHAPES)
def test_loss_and_grad(bench, dtype, labels, n, v, top):
    T, alpha = (1.0, 1.0) if (n + v) % 3 == 0 else (2.0, 0.7) if (n + v) % 3 == 1 else (1.7, 0.25)
    s, t, idx, lab = data(n, v, top, dtype, labels)
    check(bench, s, t, idx, lab, T, alpha, 1.0 / n, dtype)
    if dtype != F32:
        check(bench, s, t, idx, lab, T, alpha, 1.0, dtype, out=F32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("n,v", [(1, 70001), (2, 140000), (3, 65537), (1, 262144), (2, 300001), (40, 33000)])
def test_long_rows(bench, dtype, n, v):
    """Rows past what a block holds, and few of them."""
    s, t, idx, lab = data(n, v, 20, dtype, True)
    if n > 2:
        idx[2, :3] = [0, v - 1, v // 2]
    check(bench, s, t, idx, lab, 2.0, 0.5, 1.0, dtype)


@pytest.mark.parametrize("dtype,n,v", [(BF16, 300, 66001), (F32, 300, 33001), (F16, 600, 33003), (F32, 600, 16500),
                                       (BF16, 1100, 8300), (F32, 1100, 4200), (F16, 1700, 2100), (F32, 1900, 300)])
def test_many_rows(bench, dtype, n, v):
    """Blocks that take several rows each, rows of every alignment among them."""
    s, t, idx, lab = data(n, v, 5, dtype, True)
    check(bench, s, t, idx, lab, 1.7, 0.5, 1.0 / n if dtype != F16 else 1.0, dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("n,v", [(200, 600), (700, 64), (50, 256), (33, 65), (9, 257)])
def test_short_rows(bench, dtype, n, v):
    for top in (1, 16, 17, 64, 65):
        if top <= v:
            s, t, idx, lab = data(n, v, top, dtype, True, seed=top)
            check(bench, s, t, idx, lab, 2.0, 0.5, 1.0, dtype)
            check(bench, s, t, idx, None, 1.0, 1.0, 1.0, dtype, out=F32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("v", [40, 3001, 70001])
def test_in_place(bench, dtype, v):
    s, t, idx, lab = data(6, v, 8, dtype, True)
    check(bench, s, t, idx, lab, 1.7, 0.5, 1.0, dtype, inplace=True)


@pytest.mark.parametrize("alpha", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("T", [0.5, 1.0, 4.0])
def test_weights_and_temperatures(bench, alpha, T):
    s, t, idx, lab = data(12, 333, 12, F32, True, seed=3)
    check(bench, s, t, idx, lab, T, alpha, 0.25, F32)


@pytest.mark.parametrize("top_dtype", [F16, BF16], ids=NAMES.get)
def test_sixteen_bit_teacher(bench, top_dtype):
    s, t, idx, lab = data(8, 100, 6, BF16, True)
    check(bench, s, t, idx, lab, 2.0, 0.5, 1.0, BF16, top_dtype=top_dtype)


@pytest.mark.parametrize("v", [50, 2050, 66000])
def test_repeated_and_outside_indices(bench, v):
    """An index that occurs twice counts twice, the label may be one of them; outside the row is padding."""
    s, t, idx, lab = data(5, v, 6, F32, True, seed=8)
    idx[0] = [7, 7, 7, 3, -1, 7]
    lab[0] = 7
    idx[2] = [v, v + 5, 1e6, 2, -3, 1]
    lab[2] = v
    idx[3] = [0, v - 1, 0, v - 1, 0, 0]
    lab[3] = v - 1
    lab[4] = 4
    check(bench, s, t, idx, lab, 1.5, 0.6, 1.0, F32)
    check(bench, rounded(s, BF16), t, idx, lab, 1.5, 0.6, 1.0, BF16)


@pytest.mark.parametrize("v", [24, 1500, 70000])
def test_rows_without_targets_are_zero_whatever_they_hold(bench, v):
    s, t, idx, lab = data(6, v, 4, F32, True, seed=1)
    idx[:] = -1
    lab[:] = -1
    s[0, :] = np.nan
    s[1, 5] = np.inf
    s[2, :] = -np.inf
    idx[3] = 2
    t[3] = -np.inf  # a teacher whose every entry is masked
    alone, loss, ds = go(bench, s, t, idx, lab, 2.0, 0.5, 1.0, F32)
    assert (alone == 0).all() and (loss == 0).all() and (ds == 0).all()


@pytest.mark.parametrize("v", [24, 1500, 70000])
def test_masked_logits(bench, v):
    """Masks of the type's lowest value and -inf, a masked teacher entry, and rows that have no softmax."""
    r = np.random.default_rng(9)
    s, t, idx, lab = data(6, v, 4, F32, True, seed=2)
    low = -np.finfo(np.float32).max
    idx[:] = np.stack([r.permutation(v)[:4] for _ in range(6)])
    lab[:] = 3
    s[0, 6:] = low
    idx[0] = [0, 1, 2, 3]
    s[1, 6:] = -np.inf
    idx[1] = [0, 1, 2, 3]
    t[2, 1] = -np.inf
    s[3, :] = 0.25  # all alike
    s[4, :] = -np.inf
    s[5, 2] = np.nan
    idx[5] = [4, 5, 6, 7]
    _, loss, ds = go(bench, s, t, idx, lab, 2.0, 0.5, 1.0, F32)
    wl, el, wd, ed = model(s[:4], t[:4], idx[:4], lab[:4], 2.0, 0.5, 1.0)
    within(loss[:4], wl, el, "loss")
    within(ds[:4], wd, ed, "grad")
    assert np.isnan(loss[4:]).all() and np.isnan(ds[4:]).all()


def test_a_logit_at_minus_infinity_that_the_teacher_wants(bench):
    s, t, idx, _ = data(2, 30, 3, F32, False)
    idx[:] = [[0, 1, 2], [3, 4, 5]]
    s[0, 1] = -np.inf
    _, loss, ds = go(bench, s, t, idx, None, 1.0, 1.0, 1.0, F32)
    wl, el, wd, ed = model(s, t, idx, None, 1.0, 1.0, 1.0)
    assert np.isposinf(loss[0]) and np.isfinite(loss[1])
    within(ds, wd, ed, "grad")


def test_strided_inputs(bench):
    L = bench.L
    s, t, idx, lab = data(9, 40, 5, F16, True, seed=6)
    cfg = DistillCfg(1.3, 0.5, 1.0)
    loss, ds = bench.unset((9,)), bench.unset((9, 40), F16)
    bench.ok(L.pg_amd_distill(bench.transposed(s, F16), bench.transposed(t), bench.transposed(idx), bench.tensor(lab),
                              C.byref(cfg), loss, ds))
    wl, el, wd, ed = model(s, t, idx, lab, np.float64(np.float32(1.3)), 0.5, 1.0)
    within(bench.read(loss), wl, el, "loss")
    within(bench.read(ds), wd, ed + UNIT[F16] * (np.abs(wd) + ed) + TINY[F16], "grad")


@pytest.mark.parametrize("n,v,top,labels", [(6, 10, 4, True), (33, 257, 20, False), (3, 5000, 16, True)])
def test_node(bench, n, v, top, labels):
    """The loss node; its backward adds to the grad and scales it by the upstream one."""
    L = bench.L
    s, t, idx, lab = data(n, v, top, F32, labels, seed=4)
    T, alpha = 2.0, 0.75
    wl, el, wd, ed = model(s, t, idx, lab, T, alpha, np.float64(np.float32(1 / n)))
    x = bench.var(s)
    args = (bench.tensor(t), bench.tensor(idx), None if lab is None else bench.tensor(lab))
    cfg = DistillCfg(T, alpha, 1 / n)
    for times in (1, 2):
        loss = bench.node(L.pg_amd_ag_distill(x, *args, C.byref(cfg)))
        within(L.value(loss), [wl.sum()], el.sum() + n * 2.0 ** -24 * np.abs(wl).sum(), "loss")
        if times == 2:  # two nodes over the same logits
            loss = bench.node(L.pg_ag_add(loss, bench.node(L.pg_amd_ag_distill(x, *args, C.byref(cfg)))))
        L.pg_backward(loss)
        within(L.grad(x), times * wd, times * (ed + 4 * 2.0 ** -24 * np.abs(wd)), "grad")
    y = bench.var(s)
    half = bench.node(L.pg_amd_ag_distill(y, *args, C.byref(cfg)))
    L.pg_amd_backward_from(half, bench.tensor([0.5]))
    within(L.grad(y), 0.5 * wd, 0.5 * ed + 2.0 ** -24 * np.abs(wd), "upstream")


def test_node_outlives_the_callers_tensors(bench):
    L = bench.L
    s, t, idx, _ = data(4, 50, 6, F32, False, seed=5)
    _, _, wd, ed = model(s, t, idx, None, 1.0, 1.0, 1.0)
    x = bench.var(s)
    tt, ti = L.tensor(t.astype(np.float32)), L.tensor(idx.astype(np.float32))
    cfg = DistillCfg(1.0, 1.0, 1.0)
    loss = bench.node(L.pg_amd_ag_distill(x, tt, ti, None, C.byref(cfg)))
    L.pg_tensor_free(tt)
    L.pg_tensor_free(ti)
    other = bench.tensor(np.full((4, 6), 3.0))  # takes the freed memory, if it was freed
    L.pg_backward(loss)
    within(L.grad(x), wd, ed, "grad")
    assert (bench.read(other) == 3).all()


def test_grad_against_differences(bench):
    s, t, idx, lab = data(3, 40, 5, F32, True, seed=7)
    lab[:] = [1, 2, 3]
    T, alpha = 1.5, 0.5
    _, _, ds = go(bench, s, t, idx, lab, T, alpha, 1.0, F32)
    r = np.random.default_rng(0)
    for _ in range(30):
        i, j = r.integers(0, 3), r.integers(0, 40)
        up, down = s.copy(), s.copy()
        up[i, j] += 1e-5
        down[i, j] -= 1e-5
        slope = (model(up, t, idx, lab, T, alpha, 1.0)[0][i] - model(down, t, idx, lab, T, alpha, 1.0)[0][i]) / 2e-5
        assert abs(ds[i, j] - slope) <= 1e-5


def test_no_rows(bench):
    L = bench.L
    made = [L.pg_tensor_empty_dtype(F32, *shape_arg(sh)) for sh in ((0, 8), (0, 2), (0, 2), (0,), (0, 8))]
    if not all(made):
        pytest.skip("no tensors without elements")
    cfg = DistillCfg(1.0, 1.0, 1.0)
    bench.ok(L.pg_amd_distill(made[0], made[1], made[2], None, C.byref(cfg), made[3], made[4]))
    for t in made:
        L.pg_tensor_free(t)


def test_refusals(bench):
    L = bench.L
    s, t, idx, lab = (bench.tensor(np.zeros(sh)) for sh in ((4, 9), (4, 3), (4, 3), (4,)))
    loss, ds = bench.unset((4,)), bench.unset((4, 9))

    def call(s=s, t=t, idx=idx, lab=lab, cfg=(1.0, 0.5, 1.0), loss=loss, ds=ds):
        return L.pg_amd_distill(s, t, idx, lab, C.byref(DistillCfg(*cfg)) if cfg else None, loss, ds)

    bench.ok(call())
    bench.refused(call(s=None), "null")
    bench.refused(call(t=None), "null")
    bench.refused(call(idx=None), "null")
    bench.refused(call(cfg=None), "null")
    bench.refused(call(t=bench.tensor(np.zeros((3, 3)))), "logits [N, V]")
    bench.refused(call(idx=bench.tensor(np.zeros((4, 2)))), "logits [N, V]")
    bench.refused(call(lab=bench.tensor(np.zeros(3))), "logits [N, V]")
    bench.refused(call(s=bench.tensor(np.zeros(36))), "logits [N, V]")
    wide = bench.tensor(np.zeros((4, 257)))
    bench.refused(call(t=wide, idx=wide), "256")
    bench.refused(call(idx=bench.tensor(np.zeros((4, 3)), F16)), "f32")
    bench.refused(call(lab=bench.tensor(np.zeros(4), BF16)), "f32")
    for cfg in ((0.0, 0.5, 1.0), (-1.0, 0.5, 1.0), (np.inf, 0.5, 1.0), (np.nan, 0.5, 1.0), (1.0, 1.5, 1.0), (1.0, -0.1, 1.0),
                (1.0, np.nan, 1.0), (1.0, 0.5, np.inf)):
        bench.refused(call(cfg=cfg), "temperature")
    bench.refused(call(loss=None), "loss")
    bench.refused(call(loss=bench.unset((5,))), "loss")
    bench.refused(call(loss=bench.unset((4,), F16)), "loss")
    bench.refused(call(ds=bench.unset((4, 8))), "dlogits")
    bench.refused(call(ds=bench.unset((4, 9), F16)), "dlogits")
    bench.refused(call(ds=bench.transposed(np.zeros((4, 9)))), "contiguous")
    bench.refused(call(loss=lab), "overlaps")
    assert not L.pg_amd_ag_distill(None, t, idx, lab, C.byref(DistillCfg(1.0, 0.5, 1.0)))
    assert not L.pg_amd_ag_distill(bench.var(np.zeros((4, 9))), t, idx, bench.tensor(np.zeros(5)),
                                   C.byref(DistillCfg(1.0, 0.5, 1.0)))


def test_more_rows_than_a_launch_has_threads_for(bench):
    """Past 2^32 threads at 16, 64 and 1024 a row.  One entry and equal logits: the loss is log V, the grad 1 / V,
    less 1 at the entry."""
    L = bench.L
    cfg = DistillCfg(1.0, 1.0, 1.0)

    def full(shape, dtype, value):
        nd, sh = shape_arg(shape)
        t = L.pg_tensor_full_dtype(dtype, nd, sh, value)
        assert t, L.pg_amd_last_error().decode()
        return t

    def at(t, *i):
        return bench.get(t, (C.c_size_t * len(i))(*i))

    bench.get = L.lib.pg_tensor_get
    bench.get.restype, bench.get.argtypes = C.c_float, [C.c_void_p, C.POINTER(C.c_size_t)]
    for n, v, dtype in ((2 ** 28 + 17, 2, BF16), (2 ** 26 + 5, 65, BF16)):
        made = [full((n, v), dtype, 0.5), full((n, 1), BF16, 3.0), full((n, 1), F32, 1.0), full((n,), F32, 777.0)]
        done = L.pg_amd_distill(*made[:3], None, C.byref(cfg), made[3], None)
        got = [at(made[3], i) for i in (0, 1, n // 2, n - 17, n - 1)] if done else []
        L.sync()
        for t in made:
            L.pg_tensor_free(t)
        bench.ok(done)
        within(got, np.full(5, np.log(v)), (v / 256 + 64 + 16) * 2.0 ** -24 * (np.log(v) + 4), (n, v))
        L.lib.pg_tensor_pool_clear()
    # two losses over one node: the second adds to the grad
    n, v = 2 ** 22 + 3, 257
    top, idx = full((n, 1), BF16, 3.0), full((n, 1), F32, 2.0)
    nd, sh = shape_arg((n, v))
    x = L._check(L.pg_var_full(nd, sh, 0.5, True))
    parts = [L._check(L.pg_amd_ag_distill(x, top, idx, None, C.byref(cfg))) for _ in range(2)]
    total = L._check(L.pg_ag_add(*parts))
    L.pg_backward(total)
    g = L.node(x).grad
    got = [at(g, i, j) for i in (0, 2 ** 22 - 1, 2 ** 22, n - 1) for j in (0, 2, 256)]
    L.sync()
    for node in (total, *parts, x):
        L.pg_node_free(node)
    for t in (top, idx):
        L.pg_tensor_free(t)
    L.lib.pg_tensor_pool_clear()
    want = np.array([2 / v, 2 / v - 2, 2 / v] * 4)
    within(got, want, 2 * (v / 256 + 64 + 16) * 2.0 ** -24 * np.array([1 / v, 1 + 1 / v, 1 / v] * 4), "two losses")


# Each block of k_distill_rows at rows of an odd length, more of them than blocks:
# 1024 x 16, 512 x 16, 256 x 16, 256 x 4 and 256 x 1 pieces of 16 bytes.
ROWS = [(BF16, 300, 66001), (F16, 600, 33003), (BF16, 1100, 8301), (F16, 1700, 2101), (BF16, 1900, 601)]


@pytest.mark.parametrize("dtype,n,v", ROWS)
def test_many_rows_in_place(bench, dtype, n, v):
    """The grad of a row is stored while the next row's logits are fetched."""
    s, t, idx, lab = data(n, v, 5, dtype, True, seed=10)
    check(bench, s, t, idx, lab, 1.7, 0.5, 1.0 / n if dtype != F16 else 1.0, dtype, inplace=True)


@pytest.mark.parametrize("dtype,n,v", ROWS)
def test_many_rows_without_labels(bench, dtype, n, v):
    """One exponential a value, in place too; entries enough that several waves correct the row before."""
    s, t, idx, _ = data(n, v, 130, dtype, False, seed=11)
    idx[:, 1] = 0
    idx[:, 2] = v - 1
    check(bench, s, t, idx, None, 1.0, 1.0, 1.0 / n if dtype != F16 else 1.0, dtype, inplace=n in (600, 1900))


@pytest.mark.parametrize("dtype,n,v", ROWS)
@pytest.mark.parametrize("labels", [False, True])
def test_many_rows_with_f32_grads(bench, dtype, n, v, labels):
    """Two stored pieces for each one loaded, with one exponential and with two."""
    s, t, idx, lab = data(n, v, 7, dtype, labels, seed=12)
    check(bench, s, t, idx, lab, 1.7 if labels else 1.0, 0.5 if labels else 1.0, 1.0, dtype, out=F32)


@pytest.mark.parametrize("n,v", [(300, 33001), (600, 16501), (1100, 4203), (1700, 1030), (1900, 301)])
def test_many_f32_rows_in_place_and_without_labels(bench, n, v):
    s, t, idx, lab = data(n, v, 9, F32, True, seed=13)
    check(bench, s, t, idx, lab, 1.7, 0.5, 1.0, F32, inplace=True)
    check(bench, s, t, idx, None, 1.0, 1.0, 1.0, F32)


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


@pytest.mark.parametrize("dtype,out", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32)], ids=lambda d: NAMES[d])
@pytest.mark.parametrize("n,v", [(5, 30), (40, 3001), (3, 70001)])
@pytest.mark.parametrize("skip", [(1, 1), (3, 0), (0, 5)])
def test_tensors_that_start_inside_their_storage(bench, dtype, out, n, v, skip):
    """Logits and grad whose 16-byte pieces fall together, and not."""
    L, T, alpha = bench.L, 2.0, 0.5
    s, t, idx, lab = data(n, v, 6, dtype, True, seed=14)
    cfg = DistillCfg(T, alpha, 1.0)
    loss, ds = inside(bench, np.full(n, 777.0), F32, 3), inside(bench, np.full((n, v), 777.0), out, skip[1])
    bench.ok(L.pg_amd_distill(inside(bench, s, dtype, skip[0]), inside(bench, t, F32, 1), inside(bench, idx, F32, 3),
                              inside(bench, lab, F32, 1), C.byref(cfg), loss, ds))
    wl, el, wd, ed = model(s, t, idx, lab, T, alpha, 1.0)
    within(bench.read(loss), wl, el, "loss")
    within(bench.read(ds), wd, ed + (0 if out == F32 else UNIT[out] * (np.abs(wd) + ed) + TINY[out]), "grad")
