"""Tensors that enter a graph, as a leaf or as the upstream grad, whatever the
order of their elements in memory and whether these are written yet."""
import numpy as np
import pytest

from op_tools import Bench
from picograd_amd.capi import BF16, F16, F32

pytestmark = pytest.mark.gpu

M, K, N = 24, 16, 32


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


def node_of(bench, kind, x, w):
    """A node [M, N] over x, and x's node."""
    L = bench.L
    nx = bench.var(x)
    if kind == "gated16":
        return bench.node(L.pg_amd_ag_gated16(nx, bench.var(np.concatenate([w, w], 1)), None, 3, BF16)), nx
    if kind == "linear16":
        return bench.node(L.pg_amd_ag_linear16(nx, bench.var(w), None, 2, BF16)), nx
    if kind == "matmul16":
        return bench.node(L.pg_amd_ag_matmul16(nx, bench.var(w), F16)), nx
    if kind == "matmul":
        return bench.node(L.pg_ag_matmul(nx, bench.var(w))), nx
    nx = bench.var(x @ w)
    return bench.node(L.pg_ag_gelu(nx) if kind == "gelu" else L.pg_ag_mul(nx, bench.var(w[:1]))), nx


@pytest.mark.parametrize("kind", ["gated16", "linear16", "matmul16", "matmul", "gelu", "mul"])
def test_strided_seed(bench, kind):
    """An upstream grad that is a transposed view gives the bits of its row-major copy."""
    r = np.random.default_rng(1)
    x, w = r.standard_normal((M, K)).astype(np.float32), r.standard_normal((K, N)).astype(np.float32)
    seed = r.standard_normal((M, N)).astype(np.float32)
    grads = []
    for t in (bench.tensor(seed), bench.transposed(seed)):
        n, nx = node_of(bench, kind, x, w)
        bench.L.pg_amd_backward_from(n, t)
        grads.append(bench.L.grad(nx))
    assert np.array_equal(grads[0].view(np.uint32), grads[1].view(np.uint32))


@pytest.mark.parametrize("act", [1, 2])
def test_leaf_of_a_value_not_yet_written(bench, act):
    """A linear16 layer's output whose elements are pending until they are read."""
    L = bench.L
    r = np.random.default_rng(2)
    n = bench.node(L.pg_amd_ag_linear16(bench.var(r.standard_normal((M, K))), bench.var(r.standard_normal((K, N))), None, act,
                                        BF16))
    leaf = bench.node(L.pg_var_from_tensor(L.node(n).value, False))
    got = L.value(leaf)
    assert np.array_equal(got.view(np.uint32), L.value(n).view(np.uint32)) and np.abs(got).max() > 0


@pytest.mark.parametrize("dtype", [F32, F16])
def test_leaf_of_a_strided_tensor(bench, dtype):
    v = np.arange(M * N, dtype=np.float32).reshape(M, N)
    leaf = bench.node(bench.L.pg_var_from_tensor(bench.transposed(v, dtype), False))
    assert np.array_equal(bench.read(bench.L.node(leaf).value), v)


def test_leaf_of_a_grad(bench):
    L = bench.L
    x = bench.var(np.ones((M, N)))
    L.pg_backward(bench.node(L.pg_ag_sum_all(x)))
    leaf = bench.node(L.pg_var_from_tensor(L.node(x).grad, False))
    assert (L.value(leaf) == 1).all()
