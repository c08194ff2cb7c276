"""picograd_amd/distill.py: a 4-bit teacher, its top logits, a gated student
trained on them and served."""
import numpy as np
import pytest

from op_tools import F32, rounded
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
