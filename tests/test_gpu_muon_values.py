"""Steps over nodes whose value is replaced by another tensor behind their registration."""
import ctypes as C

import numpy as np
import pytest

from op_tools import Bench
from picograd_amd.capi import MuonCfg

pytestmark = pytest.mark.gpu


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


def optimiser(bench, momentum, *nodes):
    L = bench.L
    o = L.pg_amd_muon_new(C.byref(MuonCfg(0.02, momentum, 0.0, 0.0, 5, True)))
    assert o, L.pg_autograd_last_error().decode()
    bench.frees.append((L.pg_amd_muon_free, o))
    for n in nodes:
        assert L.pg_amd_muon_add_param(o, n) == 0
    return o


def set_grad(bench, n, g):
    node = bench.L.node(n)
    if node.grad:
        bench.L.pg_tensor_free(node.grad)
    node.grad = bench.L.tensor(np.asarray(g, np.float32))


def replace(bench, n, t):
    """t, which the node owns from here on, becomes its value."""
    node = bench.L.node(n)
    bench.frees.append((bench.L.pg_tensor_free, node.value))
    node.value = t


@pytest.mark.parametrize("shape", [(6, 4), (3, 4), (40, 60), (300, 500), (2, 12)])
def test_a_value_of_another_shape(bench, shape):
    L = bench.L
    first, other = bench.var(np.ones((4, 6))), bench.var(np.ones((5, 5)))
    opt = optimiser(bench, 0.95, other, first)
    set_grad(bench, other, np.eye(5))
    replace(bench, first, L.tensor(np.ones(shape, np.float32)))
    set_grad(bench, first, np.ones(shape))
    bench.refused(L.pg_amd_muon_step(opt), "momentum")
    assert (L.value(other) == 1).all() and (L.value(first) == 1).all()  # nothing is stepped
    for i in (0, 1):
        assert (L.read(L.pg_amd_muon_buffer(opt, i)) == 0).all()
    # its own shape again
    replace(bench, first, L.tensor(np.full((4, 6), 2.0, np.float32)))
    set_grad(bench, first, np.ones((4, 6)))
    bench.ok(L.pg_amd_muon_step(opt))
    assert (L.value(first) != 2).all() and (L.value(other)[0, 0] != 1)


def test_without_momentum_a_value_may_change_its_shape(bench):
    L = bench.L
    n = bench.var(np.ones((4, 6)))
    opt = optimiser(bench, 0.0, n)
    replace(bench, n, L.tensor(np.ones((70, 90), np.float32)))
    set_grad(bench, n, np.random.default_rng(0).standard_normal((70, 90)))
    bench.ok(L.pg_amd_muon_step(opt))
    assert np.isfinite(L.value(n)).all() and (L.value(n) != 1).any()


@pytest.mark.parametrize("momentum", [0.95, 0.0])
def test_values_that_share_memory(bench, momentum):
    L = bench.L
    a, b = bench.var(np.ones((4, 6))), bench.var(np.ones((4, 6)))
    opt = optimiser(bench, momentum, a, b)
    replace(bench, b, L.pg_tensor_view(L.node(a).value))
    for n in (a, b):
        set_grad(bench, n, np.ones((4, 6)))
    bench.refused(L.pg_amd_muon_step(opt), "overlap")
    assert (L.value(a) == 1).all()
    L.pg_tensor_free(L.node(b).grad)
    L.node(b).grad = None  # one of them alone may step
    bench.ok(L.pg_amd_muon_step(opt))
    assert (L.value(a) != 1).all() and np.array_equal(L.value(a), L.value(b))
