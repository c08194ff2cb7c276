"""Orthogonal factors and steps whose products run on the largest tiles (256 x 256, whole
and with a rest that is split along the reduction and joined), and what the other tests
of factors leave to the small kernels: numbers that are none, 16-bit copies, the
rounding of 16-bit outputs.

Bounds are those of test_gpu_muon.py.
"""
import numpy as np
import pytest

from op_tools import NAMES, Bench, rounded
from picograd_amd.capi import BF16, F16, F32
from test_gpu_muon import Model, factor, grads, near, optimiser, orth, set_grad, tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


# By the measured times these take their tiles so (S and B; X), `a + b / z` for a whole ones and b that are split into z
# slices: 128 x 128, 512 + 118 / 2; 256 x 256, 256 + 68 / 3.  64 x 64, 1536 + 4 / 16; 256 x 256, 196.
@pytest.mark.parametrize("k,n", [(4401, 4500), (4500, 4401), (3500, 3460), (3460, 3500)])
def test_one_large_matrix(bench, k, n):
    g = rounded(grads(k, n), F32)
    want = factor(g, 2)
    near(orth(bench, g, steps=2), want, tolerance(g, want, 2))


LISTS = {
    # 256 x 256: 256 + 32 / 5; 512 + 32 / 5
    "split": [(2000, 2100), (2100, 2000), (1950, 2040), (2040, 1990), (2048, 2048), (1990, 2111), (2111, 1985), (2000, 1999)],
    # S 128 x 128, B and X 256 x 256, all whole: ends inside a tile, matrices of 64 rows in one
    "whole": [(2000, 2100), (2100, 2000), (1950, 2040), (2040, 1990), (1900, 2000), (1800, 2150), (64, 3000), (2600, 50)],
    # 256 x 256: 256 + 27 / 7; 512 + 112 / 2, slices of 4096 and shorter reductions side by side
    "depths": [(4000, 4100), (4100, 4000), (1000, 4000), (4000, 10)],
}


@pytest.mark.parametrize("name", LISTS)
def test_steps_of_lists(bench, name):
    L = bench.L
    r = np.random.default_rng(20)
    steps = 2 if name == "depths" else 3
    cfg = dict(steps=steps, wd=0.1, lr=0.05)
    opt, nodes, models = optimiser(bench, **cfg), [], []
    for k, n in LISTS[name]:
        w = rounded(r.uniform(-1, 1, (k, n)) * k ** -0.5, F32)
        nodes.append(bench.var(w))
        models.append(Model(w, **cfg))
        assert L.pg_amd_muon_add_param(opt, nodes[-1]) == 0
        g = rounded(grads(k, n, seed=3), F32)
        set_grad(bench, nodes[-1], g)
        models[-1].step(g)
    bench.ok(L.pg_amd_muon_step(opt))
    for i, (n, m) in enumerate(zip(nodes, models)):
        m.check(L.value(n).astype(np.float64), L.read(L.pg_amd_muon_buffer(opt, i)))


def test_company_may_change_the_order_of_sums_only(bench):
    """A matrix alone and in two lists, that give its products other tiles, or (4096 x 10) another kernel."""
    L = bench.L
    r = np.random.default_rng(21)
    for k, n in ((700, 650), (4096, 10), (64, 64)):
        w, g = rounded(r.uniform(-1, 1, (k, n)) * k ** -0.5, F32), rounded(grads(k, n), F32)
        model = Model(w)
        model.step(g)
        for others in ([], [(300, 400)], [(1024, 1100)] * 3):
            opt = optimiser(bench)
            nodes = [bench.var(w)] + [bench.var(np.ones(s)) for s in others]
            for node, s in zip(nodes, [(k, n)] + others):
                assert L.pg_amd_muon_add_param(opt, node) == 0
                set_grad(bench, node, g if s == (k, n) else rounded(grads(*s), F32))
            bench.ok(L.pg_amd_muon_step(opt))
            model.check(L.value(nodes[0]).astype(np.float64))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=NAMES.get)
@pytest.mark.parametrize("k,n", [(64, 64), (16, 3000), (50, 200), (2049, 777), (300, 1000), (1024, 2000), (3500, 3460)])
def test_16_bit_outputs_round_the_f32_factor_once(bench, dtype, k, n):
    """From one grad the f32 output and the 16-bit one hold the same sums, every time."""
    g = rounded(grads(k, n, 22) * 100, dtype)
    wide = orth(bench, g, dtype, F32, steps=3)
    for _ in range(3):
        assert np.array_equal(orth(bench, g, dtype, dtype, steps=3), rounded(wide, dtype))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("k,n", [(64, 64), (50, 200), (250, 40), (33, 700), (129, 200), (300, 1000), (1000, 300), (3460, 3500)])
def test_what_is_no_number_spoils_the_whole_factor(bench, k, n, bad):
    """In LDS, on small and on large tiles, wherever it stands."""
    for at in ((0, 0), (k - 1, n - 1), (k // 2, n // 3)):
        g = rounded(grads(k, n, 23), F32)
        g[at] = bad
        assert np.isnan(orth(bench, g, steps=2)).all(), at


def test_what_is_no_number_stays_in_its_matrix(bench):
    """Of those that share launches."""
    L = bench.L
    r = np.random.default_rng(24)
    shapes = [(700, 650), (300, 1000), (64, 64), (2000, 10), (40, 3000), (129, 200)]
    for spoilt in range(len(shapes)):
        opt, nodes = optimiser(bench, steps=2), []
        for i, s in enumerate(shapes):
            nodes.append(bench.var(r.uniform(-1, 1, s)))
            assert L.pg_amd_muon_add_param(opt, nodes[-1]) == 0
            g = rounded(grads(*s), F32)
            if i == spoilt:
                g[s[0] - 1, 3] = np.nan
            L.node(nodes[-1]).grad = L.tensor(np.float32(g))
        bench.ok(L.pg_amd_muon_step(opt))
        for i, n in enumerate(nodes):
            v = L.value(n)
            assert np.isnan(v).all() if i == spoilt else np.isfinite(v).all(), (i, spoilt)


def layers(bench, shapes, dtype, lr=0.3):
    """16-bit layers before and after a step: their products use the stepped weights."""
    L = bench.L
    r = np.random.default_rng(25)
    opt = optimiser(bench, lr=lr, steps=2)
    ws = [rounded(r.uniform(-1, 1, s) * s[0] ** -0.5, F32) for s in shapes]
    nodes = [bench.var(w) for w in ws]
    xs = [bench.var(rounded(r.standard_normal((20, s[0])), BF16), False) for s in shapes]
    for n in nodes:
        assert L.pg_amd_muon_add_param(opt, n) == 0
    for _ in range(2):
        L.pg_amd_muon_zero_grad(opt)
        before = []
        for x, n in zip(xs, nodes):
            y = bench.node(L.pg_amd_ag_linear16(x, n, None, 0, dtype))
            before.append(L.value(y))
            L.pg_backward(bench.node(L.op("mean_all", bench.node(L.op("mul", y, y)))))
        bench.ok(L.pg_amd_muon_step(opt))
        for x, n, old in zip(xs, nodes, before):
            again = L.value(bench.node(L.pg_amd_ag_linear16(x, n, None, 0, dtype)))
            fresh = L.value(bench.node(L.pg_amd_ag_linear16(x, bench.var(L.value(n)), None, 0, dtype)))
            assert np.array_equal(again, fresh) and not np.array_equal(again, old)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=NAMES.get)
@pytest.mark.parametrize("k,n", [(130, 700), (700, 130), (129, 333), (1024, 4096), (4096, 1024), (2001, 770), (60, 1999)])
def test_kept_copies_follow_on_tiles(bench, k, n, dtype):
    layers(bench, [(k, n)], dtype)


@pytest.mark.parametrize("name", ["split", "whole"])
def test_kept_copies_follow_in_lists(bench, name):
    layers(bench, LISTS[name], BF16)
