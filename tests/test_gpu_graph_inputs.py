"""Tensors that enter a graph, as a leaf or as the upstream grad, whatever the
order of their elements in memory and whether these are written yet."""
import numpy as np
import pytest

from op_tools import Bench
from picograd_amd.capi import BF16, F16

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
