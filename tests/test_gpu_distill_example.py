"""picograd_amd/distill.py: a 4-bit teacher, its top logits, a gated student
trained on them and served."""
import numpy as np
import pytest

import test_gpu_gated as gated
import test_gpu_mx4 as mx4
from op_tools import F32, rounded, within
from picograd_amd import distill
from picograd_amd.capi import BF16, DistillCfg

pytestmark = pytest.mark.gpu


def test_the_student_learns(lib):
    said = []
    small = dict(steps=200, rows=2048, classes=100, k=32, hidden=64, f=64, top=8, batch=256, say=said.append)
    got = distill.train(lib, **small)
    assert got["losses"][-1] < got["losses"][0] / 2 and np.isfinite(got["losses"]).all()
    assert got["after"] > got["before"] + 0.2
    assert len(said) == len(got["losses"]) + 1
    again = distill.train(lib, **small)  # the same seed: the same bits
    assert again["losses"] == got["losses"] and np.array_equal(again["one"], got["one"])


def test_a_step_against_64_bits(lib):
    """The loss of a step from the values of its own logits, and the update's direction."""
    r = np.random.default_rng(1)
    m, k, f, v, top = 48, 24, 40, 90, 6
    s = distill.Student(lib, k, f, v, r)
    x = lib.var(r.standard_normal((m, k)).astype(np.float32), False)
    idx = np.argsort(r.standard_normal((m, v)), axis=1)[:, :top]
    t = rounded(r.standard_normal((m, top)) * 2, F32)
    lab = idx[:, 0].astype(np.float64)
    lab[::5] = -1
    T, alpha = 2.0, 0.75
    made = s.forward(x)
    y = lib.value(made[1]).astype(np.float64)
    for n in reversed(made):
        lib.pg_node_free(n)

    def logsoft(a):
        a = a - a.max(1, keepdims=True)
        return a - np.log(np.exp(a).sum(1, keepdims=True))

    lp, lq, lr = logsoft(t / T), logsoft(y / T), logsoft(y)
    want = alpha * T * T * (np.exp(lp) * (lp - np.take_along_axis(lq, idx, 1))).sum()
    some = lab >= 0
    want -= (1 - alpha) * lr[some, lab[some].astype(int)].sum()
    tensors = [lib.tensor(t.astype(np.float32)), lib.tensor(idx.astype(np.float32)), lib.tensor(lab.astype(np.float32))]
    losses = []
    for _ in range(3):
        n = s.step(x, *tensors, DistillCfg(T, alpha, 1.0 / m))
        losses.append(float(lib.value(n)[0]))
        lib.pg_node_free(n)
    # terms of some 2^4 in f32 over exponentials good to 2^-20
    assert abs(losses[0] - want / m) <= 2.0 ** -14 * max(1, want / m)
    assert losses[2] < losses[1] < losses[0]
    for tensor in tensors:
        lib.pg_tensor_free(tensor)
    lib.pg_node_free(x)
    s.free()


@pytest.mark.parametrize("rows", [1, 2, 16, 17, 300])
def test_served_rows_do_not_depend_on_their_batch(lib, rows):
    """A row alone and in a batch: the sums' order may differ, the rounding of
    h to bf16 and then to 4 bits may go the other way in a few places."""
    r = np.random.default_rng(rows)
    s = distill.Student(lib, 64, 96, 50, r)
    served = s.freeze()
    x = r.standard_normal((rows, 64)).astype(np.float32)
    all_rows = served.logits(x)
    w, b, wo, bo = (lib.value(p).astype(np.float64) for p in s.params)
    z = rounded(x, BF16) @ rounded(w, BF16) + b
    h = z[:, :96] / (1 + np.exp(-z[:, :96])) * z[:, 96:]
    y = h @ wo + bo
    # 4 bits: within a quarter of each value's own power or a sixteenth of the block's largest
    noise = np.abs(h).max() * np.abs(wo).max() * np.sqrt(96) * 0.5
    assert np.abs(all_rows - y).max() <= noise
    assert np.abs(all_rows[:1] - served.logits(x[:1])).max() <= noise / 4
    served.free()
    s.free()


def served_model(s, x):
    """The student's logits as they are served, in 64 bits, and a bound of each.

    h is rounded to bf16 and then to 4 bits; both are certain but where the f32
    sums could fall on either side.  With lo and hi the two ends, each rounded to
    bf16, a block of one power on both sides has Q(h) between Q(lo) and Q(hi),
    one whose power could be either is off by at most 4 of the larger units."""
    w, b, wo, bo = (s.lib.value(p).astype(np.float64) for p in s.params)
    h, e = gated.model(rounded(x, BF16), rounded(w, BF16), b, None, "silu", BF16)["h"]
    lo, mid, hi = (rounded(v, BF16) for v in (h - e, h, h + e))
    qlo, q, qhi = (mx4.quantized(v) for v in (lo, mid, hi))
    off = np.maximum(np.abs(qhi - q), np.abs(q - qlo))
    for i in range(0, h.shape[1], 32):
        small = np.minimum(np.abs(lo[:, i:i + 32]), np.abs(hi[:, i:i + 32]))
        small[np.sign(lo[:, i:i + 32]) != np.sign(hi[:, i:i + 32])] = 0
        large = np.maximum(np.abs(lo[:, i:i + 32]), np.abs(hi[:, i:i + 32]))
        # the block's largest magnitude lies between these two
        a, z = (np.frexp(np.maximum(v.max(1), 2.0 ** -126))[1] for v in (small, large))
        off[:, i:i + 32] = np.where((a != z)[:, None], np.ldexp(4.0, z - 3)[:, None], off[:, i:i + 32])
    qo = mx4.quantized(wo.T).T
    y = q @ qo
    bound = off @ np.abs(qo) + (h.shape[1] + 2) * 2.0 ** -24 * ((np.abs(q) + off) @ np.abs(qo)) + 2.0 ** -24 * np.abs(y + bo)
    return y + bo, bound


@pytest.mark.parametrize("rows", [1, 2, 16, 17, 300])
def test_served_logits(lib, rows):
    """The gated layer in bf16 and the output layer in 4 bits, one after the other, against what they round."""
    r = np.random.default_rng(100 + rows)
    s = distill.Student(lib, 64, 96, 50, r)
    x = r.standard_normal((rows, 64)).astype(np.float32)
    want, bound = served_model(s, x)
    served = s.freeze()
    got, alone = served.logits(x), served.logits(x[:1])
    served.free()
    s.free()
    within(got, want, bound, "logits")
    within(alone, want[:1], bound[:1], "the first row alone")
    # the bounds tell wrong logits from right ones
    for wrong in (np.zeros_like(want), want[:, ::-1], np.roll(want, 1, 1), 1.01 * want):
        assert (np.abs(wrong - want) > bound).mean() > 0.5


def test_served_logits_of_a_trained_student(lib):
    """As above with biases and weights that are no longer where they began."""
    r = np.random.default_rng(5)
    m, k, f, v, top = 64, 32, 64, 60, 5
    s = distill.Student(lib, k, f, v, r)
    x = r.standard_normal((m, k)).astype(np.float32)
    idx = np.argsort(r.standard_normal((m, v)), axis=1)[:, :top]
    node = lib.var(x, False)
    tensors = [lib.tensor(a.astype(np.float32)) for a in (r.standard_normal((m, top)), idx, idx[:, 0])]
    for _ in range(20):
        lib.pg_node_free(s.step(node, *tensors, DistillCfg(2.0, 0.75, 1.0 / m)))
    want, bound = served_model(s, x)
    served = s.freeze()
    got = served.logits(x)
    served.free()
    for t in tensors:
        lib.pg_tensor_free(t)
    lib.pg_node_free(node)
    s.free()
    within(got, want, bound, "logits")
    for wrong in (np.zeros_like(want), want[:, ::-1], np.roll(want, 1, 1)):
        assert (np.abs(wrong - want) > bound).mean() > 0.5
