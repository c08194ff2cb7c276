"""picograd_amd/distill.py with a layer norm, orthogonalised updates and an output
layer in 8 bits: the run, a step's grads and update, and the served rows."""
import numpy as np
import pytest

import test_gpu_layernorm as norm
import test_gpu_muon as muon
from op_tools import BF16, F32, UNIT, Bench, rounded, within
from picograd_amd import distill
from picograd_amd.capi import DistillCfg

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture()
def bench(lib):
    b = Bench(lib)
    yield b
    b.close()


@pytest.mark.parametrize("opts", [dict(norm=True, muon=True, bits=8), dict(norm=True), dict(muon=True), dict(bits=8)],
                         ids=lambda o: "-".join(o))
def test_it_runs(lib, opts):
    said = []
    small = dict(steps=30, rows=1024, classes=100, k=32, hidden=64, f=64, top=8, batch=256, say=said.append)
    got = distill.train(lib, **small, **opts)
    assert np.isfinite(got["losses"]).all() and np.isfinite(got["one"]).all() and len(said) == len(got["losses"]) + 1
    again = distill.train(lib, **small, **opts)  # the same seed: the same bits
    assert again["losses"] == got["losses"] and np.array_equal(again["one"], got["one"])


def logsoft(a):
    a = a - a.max(1, keepdims=True)
    return a - np.log(np.exp(a).sum(1, keepdims=True))


def test_a_step(bench):
    """The grads behind the logits, from the values that the nodes hold, and what the two optimisers make of them."""
    L = bench.L
    r = np.random.default_rng(1)
    m, k, f, v, top = 48, 24, 40, 90, 6
    s = distill.Student(L, k, f, v, r, norm=True, muon=True)
    bench.frees.append((lambda st: st.free(), s))
    x = bench.var(r.standard_normal((m, k)), False)
    idx = np.argsort(r.standard_normal((m, v)), axis=1)[:, :top]
    t = rounded(r.standard_normal((m, top)) * 2, F32)
    made = s.forward(x)
    assert len(made) == 3
    h, y, z = (L.value(n).astype(np.float64) for n in made)
    for n in reversed(made):
        L.pg_node_free(n)
    w, _, wo, _, lw, lb = (L.value(p).astype(np.float64) for p in s.params)
    within(y, norm.Model(h, lw, lb).y, norm.Model(h, lw, lb).ey, "the norm")
    T = 2.0
    loss = s.step(x, bench.tensor(t), bench.tensor(idx), None, DistillCfg(T, 1.0, 1.0 / m))
    bench.node(loss)
    p, q = np.exp(logsoft(t / T)), np.exp(logsoft(z / T))
    g = q.copy()
    np.subtract.at(g, (np.arange(m)[:, None], idx), p)
    g *= T / m
    # exponentials and sums in f32: 2^-18 of each part
    eg = 2.0 ** -18 * (q + np.abs(g) * m / T) * T / m
    # the products round their operands to bf16: g's rounding may go either way where eg moves it
    wq, yq = rounded(wo, BF16), rounded(y, BF16)
    gq, egq = rounded(g, BF16), UNIT[BF16] * 2 * np.abs(g) + eg
    dwo, edwo = yq.T @ gq, np.abs(yq).T @ egq + 2.0 ** -20 * np.abs(yq).T @ np.abs(gq)
    within(L.grad(s.params[2]), dwo, edwo, "output layer")
    dy, edy = gq @ wq.T, egq @ np.abs(wq).T + 2.0 ** -20 * np.abs(gq) @ np.abs(wq).T
    back = norm.Model(h, lw, lb, dy)
    n = (h - h.mean(1, keepdims=True)) / np.sqrt(h.var(1, keepdims=True) + distill.NORM_EPS)
    within(L.grad(s.params[5]), back.db, back.edb + edy.sum(0), "norm's bias")
    within(L.grad(s.params[4]), back.dw, back.edw + (edy * np.abs(n)).sum(0), "norm's weight")
    # the matrices' update follows their grads, AdamW's moves the others
    for i, before in ((0, w), (2, wo)):
        model = muon.Model(before, lr=0.02, wd=1e-2)
        model.step(L.grad(s.params[i]).astype(np.float64))
        model.check(L.value(s.params[i]).astype(np.float64))
    for i, before in ((4, lw), (5, lb)):
        step = np.abs(L.value(s.params[i]) - before)
        assert step.max() <= 2.1e-3 and step.min() > 0  # the first step is lr for every value


@pytest.mark.parametrize("rows", [1, 16, 17, 300])
def test_served_rows(bench, rows):
    """Against the layers in 64 bits.  h and y are off by their bf16 rounding (a half
    step of h moves n by rstd times that), q8's rows and columns by 1 / 254 of
    their largest value each."""
    L = bench.L
    r = np.random.default_rng(rows)
    s = distill.Student(L, 64, 96, 50, r, norm=True)
    served = s.freeze(8)
    x = r.standard_normal((rows, 64)).astype(np.float32)
    got = served.logits(x)
    w, b, wo, bo, lw, lb = (L.value(p).astype(np.float64) for p in s.params)
    z = rounded(x, BF16) @ rounded(w, BF16) + b
    h = z[:, :96] / (1 + np.exp(-z[:, :96])) * z[:, 96:]
    rstd = 1 / np.sqrt(h.var(1, keepdims=True) + distill.NORM_EPS)
    n = (h - h.mean(1, keepdims=True)) * rstd
    eh = UNIT[BF16] * np.abs(h) + 2.0 ** -18 * np.abs(h).max(1, keepdims=True)
    en = rstd * (eh + eh.mean(1, keepdims=True)) + np.abs(n) * rstd * np.sqrt((eh ** 2).mean(1, keepdims=True)) * 1.1
    y = n * lw + lb
    ey = np.abs(lw) * en + UNIT[BF16] * (np.abs(y) + en)
    ymax, wmax = np.abs(y).max(1, keepdims=True) + ey.max(1, keepdims=True), np.abs(wo).max(0)
    bound = (ey + ymax / 254) @ (np.abs(wo) + wmax / 254) + np.abs(y) @ np.broadcast_to(wmax / 254, wo.shape) + 1e-5
    within(got, y @ wo + bo, bound, "logits")
    one = served.logits(x[rows - 1:])
    # the sums of whole numbers are exact; the gated layer's may round h the other way in another batch
    assert np.abs(one[0] - got[rows - 1]).max() <= bound[rows - 1].max()
    served.free()
    s.free()
