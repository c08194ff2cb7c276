"""Orthogonal factors (pg_amd_orthogonalise) and the optimiser made of them
(pg_amd_muon_*) against the formulas in 64 bits.

Bounds, in the norm of the whole difference over that of the result.  The library
keeps f32's exactness from pieces of 22 bits where f32 has 24, so its roundings
are four times as large and the product of the low pieces that it leaves out
is two more: six times the error that the same steps in f32 have.  Where that
happens to be next to nothing (a few values), three roundings of 2^-22 a step
remain, which grow by at most 3.4445 a step while a value is small and less after that:
3 2^-22 (1 + 3.4445 + .. + 3.4445^4) = 1.5e-4, more for more steps.
"""
import ctypes as C

import numpy as np
import pytest

from op_tools import NAMES, UNIT, Bench, rounded
from picograd_amd.capi import BF16, F16, F32, MuonCfg

pytestmark = pytest.mark.gpu
A, B_, C_ = 3.4445, -4.7750, 2.0315


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


def factor(g, steps=5, dtype=np.float64):
    """The same in 64 bits, or in f32."""
    size = np.linalg.norm(g.astype(np.float64))
    x = (g / (size if size > 0 else 1.0)).astype(dtype)
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.T.copy()
    a, b, c = (dtype(v) for v in (A, B_, C_))
    for _ in range(steps):
        s = x @ x.T
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.T if tall else x


def tolerance(g, want, steps=5):
    with np.errstate(all="ignore"):
        f32 = np.linalg.norm(factor(g, steps, np.float32) - want) / np.linalg.norm(want)
    return 6 * f32 + 3 * 2.0 ** -22 * sum(A ** k for k in range(min(steps, 5)))


def near(got, want, tol, what=""):
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= tol, (what, off, tol)


def grads(k, n, seed=0, decay=4.0):
    """Some directions carry most of it."""
    r = np.random.default_rng(seed + 1000 * k + n)
    d = min(k, n)
    return (r.standard_normal((k, d)) * np.exp(-decay * np.arange(d) / d)) @ r.standard_normal((d, n)) * 1e-3


def orth(bench, g, dtype=F32, out=F32, steps=5):
    o = bench.unset(g.shape, out)
    bench.ok(bench.L.pg_amd_orthogonalise(bench.tensor(g, dtype), steps, o))
    return bench.read(o)


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (1, 1000), (3, 64), (64, 3), (10, 10), (31, 33), (64, 64), (65, 63), (64, 65),
          (100, 257), (257, 100), (128, 128), (129, 129), (192, 200), (300, 1000), (1000, 300), (513, 512), (40, 5000),
          (5000, 40)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("k,n", SHAPES)
def test_factor(bench, dtype, k, n):
    g = rounded(grads(k, n) * (100 if dtype == F16 else 1), dtype)
    want = factor(g)
    tol = tolerance(g, want)
    for out in {dtype, F32}:
        near(orth(bench, g, dtype, out), want, tol + (UNIT[out] if out != F32 else 0), NAMES[out])


# either side of what a block holds in registers
THIN = [(16, 16), (16, 17), (1, 4096), (16, 1024), (1025, 15), (4096, 16), (16, 4097), (17, 31), (32, 512), (513, 30),
        (2047, 32), (18, 2048), (17, 2049)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=NAMES.get)
@pytest.mark.parametrize("k,n", THIN)
def test_thin_factors(bench, dtype, k, n):
    test_factor(bench, dtype, k, n)


# enough tiles for the larger ones, square, wide and tall
@pytest.mark.parametrize("k,n", [(2000, 2100), (2950, 2901), (700, 6100), (4500, 1500)])
def test_large_factors(bench, k, n):
    g = rounded(grads(k, n), F32)
    want = factor(g)
    near(orth(bench, g), want, tolerance(g, want))


@pytest.mark.parametrize("steps", [1, 2, 3, 7, 12])
def test_other_numbers_of_steps(bench, steps):
    g = rounded(grads(70, 90, 1), F32)
    want = factor(g, steps)
    near(orth(bench, g, steps=steps), want, tolerance(g, want, steps))


def test_the_values_come_near_one(bench):
    r = np.random.default_rng(2)
    g = r.standard_normal((200, 300))
    s = np.linalg.svd(orth(bench, g), compute_uv=False)
    assert 0.6 < s.min() and s.max() < 1.21
    u, _, vt = np.linalg.svd(g, full_matrices=False)
    o = orth(bench, g)
    # the directions are g's: u^T O v is diagonal, but for rounding
    d = u.T @ o @ vt.T
    assert np.abs(d - np.diag(np.diag(d))).max() < 1e-4 and np.diag(d).min() > 0.6


@pytest.mark.parametrize("k,n", [(50, 80), (80, 50), (300, 300)])
def test_the_norm_does_not_matter(bench, k, n):
    """A power of two times g has the same bits; the squares of 1e30 and 1e-30 fit 64 bits."""
    g = rounded(grads(k, n, 3), F32)
    first = orth(bench, g)
    for p in (-90, -10, 10, 100):
        assert np.array_equal(orth(bench, g * 2.0 ** p), first)


def test_ranks_zeros_and_what_is_no_number(bench):
    r = np.random.default_rng(4)
    assert (orth(bench, np.zeros((40, 70))) == 0).all()
    for g in (np.outer(r.standard_normal(60), r.standard_normal(90)), np.ones((70, 70)), np.eye(65),
              np.diag(np.r_[np.ones(30), np.zeros(40)]), np.where(np.arange(6400).reshape(80, 80) == 1234, 1.0, 0.0)):
        g = rounded(g, F32)
        want = factor(g)
        # values of zero stay next to it: what rounding puts there grows as the small ones do
        near(orth(bench, g), want, tolerance(g, want))
    for bad in (np.nan, np.inf, -np.inf):
        for k, n in ((30, 100), (100, 30)):
            g = grads(k, n, 5)
            g[3, 7] = bad
            assert np.isnan(orth(bench, g)).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("k,n", [(5, 90), (33, 70), (70, 33), (30, 700), (200, 200)])
def test_in_place_strided_and_inside_a_storage(bench, dtype, k, n):
    L = bench.L
    g = rounded(grads(k, n, 6), dtype)
    want = orth(bench, g, dtype, dtype)
    t = bench.tensor(g, dtype)
    bench.ok(L.pg_amd_orthogonalise(t, 5, t))
    assert np.array_equal(bench.read(t), want)
    o = bench.unset((k, n), dtype)
    bench.ok(L.pg_amd_orthogonalise(bench.transposed(g, dtype), 5, o))
    assert np.array_equal(bench.read(o), want)
    stores = []
    for values, skip in ((g, 1), (np.zeros((k, n)), 3)):
        store = bench.tensor(np.concatenate([np.full(skip, 5.0), values.ravel(), np.full(9, 6.0)]), dtype)
        v = L.pg_tensor_view(store)
        bench.frees.append((L.pg_tensor_free, v))
        i = L.tinfo(v)
        i.dev, i.ndim, i.numel = i.dev + skip * i.elem_size, 2, k * n
        i.shape[0], i.shape[1], i.stride[0], i.stride[1] = k, n, n, 1
        stores.append((v, store))
    bench.ok(L.pg_amd_orthogonalise(stores[0][0], 5, stores[1][0]))
    whole = bench.read(stores[1][1])
    assert np.array_equal(whole[3:-9].reshape(k, n), want) and (whole[:3] == 5).all() and (whole[-9:] == 6).all()


@pytest.mark.parametrize("k,n", [(64, 64), (16, 3000), (31, 1500), (130, 700), (2000, 2100)])
def test_the_same_call_gives_the_same_bits(bench, k, n):
    g = grads(k, n, 7)
    first = orth(bench, g)
    assert np.array_equal(orth(bench, g), first) and np.array_equal(orth(bench, g), first)


# ---------------------------------------------------------------- the optimiser

def optimiser(bench, lr=0.02, momentum=0.95, wd=0.0, rms=0.0, steps=5, nesterov=True):
    o = bench.L.pg_amd_muon_new(C.byref(MuonCfg(lr, momentum, wd, rms, steps, nesterov)))
    assert o, bench.L.pg_autograd_last_error().decode()
    bench.frees.append((bench.L.pg_amd_muon_free, o))
    return o


def set_grad(bench, n, g):
    """A leaf's grad, by a backward from its sum with 0."""
    L = bench.L
    node = L.node(n)
    if node.grad:
        L.pg_tensor_free(node.grad)
        node.grad = None
    root = bench.node(L.op("add", n, bench.node(L.pg_var_scalar(0.0, False))))
    L.pg_amd_backward_from(root, bench.tensor(g))
    assert np.array_equal(L.grad(n), np.float32(g))


class Model:
    """The steps in 64 bits, with the bound of W's error in the norm."""

    def __init__(self, w, lr=0.02, momentum=0.95, wd=0.0, rms=0.0, steps=5, nesterov=True):
        self.w, self.m, self.off = w.copy(), np.zeros_like(w), 0.0
        self.lr, self.mu, self.wd, self.steps, self.nesterov = lr, momentum, wd, steps, nesterov
        k, n = w.shape
        self.size = rms * max(k, n) ** 0.5 if rms else max(1.0, n / k) ** 0.5

    def step(self, g):
        self.m = self.mu * self.m + g
        u = g + self.mu * self.m if self.nesterov else self.m
        o = factor(u, self.steps)
        # u itself is f32: three roundings, that grow as the rest does
        self.off += self.lr * self.size * np.linalg.norm(o) * 2 * tolerance(u, o, self.steps)
        self.w = (1 - self.lr * self.wd) * self.w - self.lr * self.size * o
        self.off += 4 * 2.0 ** -24 * (np.linalg.norm(self.w) + self.lr * self.size * np.linalg.norm(o))

    def check(self, w, m=None):
        assert np.linalg.norm(w - self.w) <= self.off, (np.linalg.norm(w - self.w), self.off)
        if m is not None:
            assert np.linalg.norm(m - self.m) <= 16 * 2.0 ** -24 * np.linalg.norm(np.abs(self.m)) + 1e-30


CFGS = [dict(), dict(nesterov=False), dict(momentum=0.0), dict(wd=0.1, lr=0.05), dict(rms=0.2, wd=0.01), dict(steps=3, lr=0.1)]


@pytest.mark.parametrize("cfg", CFGS, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()) or "default")
def test_steps(bench, cfg):
    """Matrices of very different shapes in one launch, over three steps."""
    L = bench.L
    r = np.random.default_rng(8)
    opt, nodes, models = optimiser(bench, **cfg), [], []
    for k, n in ((64, 64), (10, 300), (300, 10), (129, 200), (1, 5), (700, 650), (2000, 10), (30, 600)):
        w = rounded(r.uniform(-1, 1, (k, n)) * k ** -0.5, F32)
        nodes.append(bench.var(w))
        models.append(Model(w, **cfg))
        assert L.pg_amd_muon_add_param(opt, nodes[-1]) == 0
    assert L.pg_amd_muon_num_params(opt) == len(nodes)
    for step in range(3):
        L.pg_amd_muon_zero_grad(opt)
        for i, (n, m) in enumerate(zip(nodes, models)):
            if (i + step) % 4 == 3:
                continue  # no grad: the parameter and its momentum stay
            g = rounded(grads(*m.w.shape, seed=step), F32)
            set_grad(bench, n, g)
            m.step(g)
        bench.ok(L.pg_amd_muon_step(opt))
        for i, (n, m) in enumerate(zip(nodes, models)):
            buf = L.pg_amd_muon_buffer(opt, i)
            assert bool(buf) == (m.mu > 0)
            m.check(L.value(n).astype(np.float64), L.read(buf) if buf else None)
    assert not L.pg_amd_muon_buffer(opt, len(nodes))


def test_more_matrices_than_a_launch_takes(bench):
    L = bench.L
    r = np.random.default_rng(9)
    opt, nodes, models = optimiser(bench), [], []
    for i in range(29):
        w = rounded(r.uniform(-1, 1, (5 + 3 * i, 90 - 3 * i)), F32)
        nodes.append(bench.var(w))
        models.append(Model(w))
        assert L.pg_amd_muon_add_param(opt, nodes[-1]) == 0
        g = rounded(grads(*w.shape), F32)
        set_grad(bench, nodes[-1], g)
        models[-1].step(g)
    bench.ok(L.pg_amd_muon_step(opt))
    for n, m in zip(nodes, models):
        m.check(L.value(n).astype(np.float64))
    # a matrix has the same bits in whatever company
    alone = optimiser(bench)
    w = rounded(np.random.default_rng(9).uniform(-1, 1, (5, 90)), F32)
    n = bench.var(w)
    assert L.pg_amd_muon_add_param(alone, n) == 0
    set_grad(bench, n, rounded(grads(5, 90), F32))
    bench.ok(L.pg_amd_muon_step(alone))
    assert np.array_equal(L.value(n), L.value(nodes[0]))


@pytest.mark.parametrize("k,n", [(48, 64), (50, 33), (16, 700), (301, 9), (24, 37), (1100, 20)])
def test_kept_copies_follow(bench, k, n):
    """A 16-bit layer before and after a step: its product uses the stepped weights."""
    L = bench.L
    r = np.random.default_rng(10)
    w, x = rounded(r.uniform(-1, 1, (k, n)), F32), rounded(r.standard_normal((20, k)), BF16)
    nw, nx = bench.var(w), bench.var(x, False)
    opt = optimiser(bench, lr=0.3)
    assert L.pg_amd_muon_add_param(opt, nw) == 0
    for dtype in (BF16, BF16, F16):
        y = bench.node(L.pg_amd_ag_linear16(nx, nw, None, 0, dtype))
        loss = bench.node(L.op("mean_all", y))
        L.pg_amd_muon_zero_grad(opt)
        L.pg_backward(loss)
        bench.ok(L.pg_amd_muon_step(opt))
        again = bench.node(L.pg_amd_ag_linear16(nx, nw, None, 0, dtype))
        fresh = bench.node(L.pg_amd_ag_linear16(nx, bench.var(L.value(nw)), None, 0, dtype))
        assert np.array_equal(L.value(again), L.value(fresh)) and not np.array_equal(L.value(again), L.value(y))


@pytest.mark.parametrize("shape", [(40, 60), (9, 130), (300, 30), (100, 110)])
def test_a_clipped_grad(bench, shape):
    """The direction does not change with the norm, the momentum does."""
    L = bench.L
    r = np.random.default_rng(11)
    w, g = rounded(r.uniform(-1, 1, shape), F32), rounded(r.standard_normal(shape), F32)
    n, model = bench.var(w), Model(w)
    opt = optimiser(bench)
    assert L.pg_amd_muon_add_param(opt, n) == 0
    set_grad(bench, n, g)
    norm = L.pg_clip_grad_norm((C.c_void_p * 1)(n), 1, 0.5, -1.0)
    clipped = g * (0.5 / (norm + 1e-6))
    model.step(clipped)
    bench.ok(L.pg_amd_muon_step(opt))
    model.check(L.value(n).astype(np.float64))
    m = L.read(L.pg_amd_muon_buffer(opt, 0))
    assert np.abs(m - clipped).max() <= 8 * 2.0 ** -24 * np.abs(clipped).max()
    assert np.abs(L.grad(n) - clipped).max() <= 8 * 2.0 ** -24 * np.abs(clipped).max()


def test_a_grad_from_a_graph_and_one_of_zeros(bench):
    L = bench.L
    r = np.random.default_rng(12)
    w, x = rounded(r.uniform(-1, 1, (30, 40)), F32), rounded(r.standard_normal((9, 30)), F32)
    nw, nx, other = bench.var(w), bench.var(x, False), bench.var(w[:5])
    opt = optimiser(bench)
    for n in (nw, other):
        assert L.pg_amd_muon_add_param(opt, n) == 0
    set_grad(bench, other, np.zeros((5, 40)))
    y = bench.node(L.op("matmul", nx, nw))
    L.pg_backward(bench.node(L.op("sum_all", bench.node(L.op("mul", y, y)))))
    model = Model(w)
    model.step(rounded(L.grad(nw), F32))
    bench.ok(L.pg_amd_muon_step(opt))
    model.check(L.value(nw).astype(np.float64))
    assert np.array_equal(L.value(other), np.float32(w[:5]))


def test_rates_and_decay_alone(bench):
    L = bench.L
    w = rounded(np.random.default_rng(13).uniform(-1, 1, (6, 9)), F32)
    n, opt = bench.var(w), optimiser(bench, lr=0.0, wd=0.5)
    assert L.pg_amd_muon_add_param(opt, n) == 0
    set_grad(bench, n, grads(6, 9))
    bench.ok(L.pg_amd_muon_step(opt))
    assert np.array_equal(L.value(n), np.float32(w)) and L.pg_amd_muon_get_lr(opt) == 0
    assert L.pg_amd_muon_set_lr(opt, 0.5) and L.pg_amd_muon_get_lr(opt) == 0.5
    L.pg_amd_muon_zero_grad(opt)
    assert L.grad(n) is None
    bench.ok(L.pg_amd_muon_step(opt))  # no grads: nothing moves
    assert np.array_equal(L.value(n), np.float32(w))


def test_saved_momenta(bench, tmp_path):
    L = bench.L
    path = str(tmp_path / "muon").encode()
    r = np.random.default_rng(14)
    ws = [rounded(r.uniform(-1, 1, s), F32) for s in ((20, 30), (30, 4))]

    def fresh(**kw):
        opt, nodes = optimiser(bench, **kw), [bench.var(w) for w in ws]
        for n in nodes:
            assert L.pg_amd_muon_add_param(opt, n) == 0
        return opt, nodes

    def step(opt, nodes, seed):
        for n, w in zip(nodes, ws):
            set_grad(bench, n, grads(*w.shape, seed=seed))
        bench.ok(L.pg_amd_muon_step(opt))

    opt, nodes = fresh()
    step(opt, nodes, 0)
    assert L.pg_amd_muon_save(opt, path)
    after = [L.value(n) for n in nodes]
    step(opt, nodes, 1)
    other, onodes = fresh()
    for n, v in zip(onodes, after):
        L.pg_tensor_copy_from(L.node(n).value, t := L.tensor(v))
        L.pg_tensor_free(t)
    assert L.pg_amd_muon_load_into(other, path)
    step(other, onodes, 1)
    for a, b in zip(nodes, onodes):
        assert np.array_equal(L.value(a), L.value(b))
    bare, _ = fresh(momentum=0.0)
    assert not L.pg_amd_muon_load_into(bare, path)  # nowhere to load it
    few = optimiser(bench)
    assert not L.pg_amd_muon_load_into(few, path) and not L.pg_amd_muon_load_into(other, b"/nonexistent")
    assert L.pg_amd_muon_save(bare, path) and L.pg_amd_muon_load_into(other, path)
    assert (L.read(L.pg_amd_muon_buffer(other, 0)) == 0).all()


def test_refusals(bench):
    L = bench.L
    g, o = bench.tensor(np.ones((4, 6))), bench.unset((4, 6))
    orthogonalise = L.pg_amd_orthogonalise
    for bad in ((None, 5, o), (g, 5, None), (g, 5, bench.unset((6, 4))), (bench.tensor(np.ones(6)), 5, bench.unset((6,))),
                (bench.unset((0, 6)), 5, bench.unset((0, 6))),
                (bench.unset((1, 2 ** 16 + 1), BF16), 5, bench.unset((1, 2 ** 16 + 1), BF16))):
        bench.refused(orthogonalise(*bad), "matrix")
    for steps in (0, -1, 101):
        bench.refused(orthogonalise(g, steps, o), "steps")
    bench.refused(orthogonalise(g, 5, bench.transposed(np.ones((4, 6)))), "contiguous")
    square = bench.transposed(np.ones((4, 4)))
    base = L.pg_tensor_view(square)
    bench.frees.append((L.pg_tensor_free, base))
    i = L.tinfo(base)
    i.stride[0], i.stride[1] = 4, 1
    bench.refused(orthogonalise(square, 5, base), "overlaps")
    nan = float("nan")
    for bad in ((-1, .9, 0, 0, 5), (nan, .9, 0, 0, 5), (1, -1, 0, 0, 5), (1, .9, -1, 0, 5), (1, .9, 0, -1, 5),
                (1, .9, 0, 0, 0), (1, .9, 0, 0, 101), (1, float("inf"), 0, 0, 5)):
        assert not L.pg_amd_muon_new(C.byref(MuonCfg(*bad, True)))
        assert "muon" in L.pg_autograd_last_error().decode()
    opt = L.pg_amd_muon_new(None)
    bench.frees.append((L.pg_amd_muon_free, opt))
    d = L.pg_amd_muon_cfg_default()
    assert abs(L.pg_amd_muon_get_lr(opt) - d.lr) == 0 and (d.steps, d.nesterov, d.rms) == (5, True, 0)
    n = bench.var(np.ones((4, 6)))
    for bad in ((None, n), (opt, None), (opt, bench.var(np.ones((4, 6)), False)), (opt, bench.var(np.ones(4))),
                (opt, bench.node(L.var(np.zeros((4, 6), np.uint16), True, BF16)))):
        assert L.pg_amd_muon_add_param(*bad) == -1
        assert "matrix" in L.pg_autograd_last_error().decode()
    assert L.pg_amd_muon_add_param(opt, n) == 0 and L.pg_amd_muon_add_param(opt, n) == -1
    assert "already" in L.pg_autograd_last_error().decode() and L.pg_amd_muon_num_params(opt) == 1
    for lr in (-1.0, nan, float("inf")):
        bench.refused(L.pg_amd_muon_set_lr(opt, lr), "rate")
    bench.refused(L.pg_amd_muon_step(None), "null")
    L.pg_amd_muon_free(None)
    L.pg_amd_muon_zero_grad(None)
    # a grad of another shape: nothing is stepped
    other = bench.var(np.ones((3, 3)))
    assert L.pg_amd_muon_add_param(opt, other) == 0
    set_grad(bench, other, np.ones((3, 3)))
    L.node(n).grad = t = L.tensor(np.ones((6, 4), np.float32))
    bench.refused(L.pg_amd_muon_step(opt), "shape")
    assert (L.value(other) == 1).all() and (L.read(L.pg_amd_muon_buffer(opt, 1)) == 0).all()
    assert t
