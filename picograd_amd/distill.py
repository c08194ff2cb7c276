"""A gated student trained on the top logits of a 4-bit teacher, over the C ABI.

    python -m picograd_amd.distill [--steps 500] [--rows 8192] [--classes 1000] [--norm] [--muon] [--bits 4]

The teacher is a frozen network of one gelu layer, its two matrices held in 4
bits (pg_amd_mx4_quantize).  It runs over the training rows once
(pg_amd_mx4_matmul); the k highest logits of each row, with their indices, are
what is kept of it.  The student is one gated layer (pg_amd_ag_gated16) and
one linear layer, trained with pg_amd_ag_distill on those and the rows' labels by AdamW.
Served, the student runs on 16-bit tensors without a graph: pg_amd_gated,
then its output layer in 4 bits.  With --norm its hidden values pass a layer norm
(pg_ag_layernorm; pg_amd_layernorm served), with --muon its two matrices step along
orthogonalised momenta (pg_amd_muon_*) and AdamW keeps the rest, with --bits 8 its
output layer is served in 8 bits (pg_amd_q8_matmul).

Data, teacher and student come from a seed; what is reported is how often the
student's highest logit is the teacher's on rows that neither saw.
"""
from __future__ import annotations

import argparse
import ctypes as C
import time

import numpy as np

from .capi import BF16, F32, AdamCfg, DistillCfg, MuonCfg, PgLib, load, shape_arg

ACT_NONE, ACT_SILU = 0, 3  # PG_ACT_*
NORM_EPS = 1e-5


class Mx4:
    """A frozen matrix W [K, N] in 4 bits; m(x) is a new tensor Q(x) W."""

    def __init__(self, lib: PgLib, w: int):
        self.lib, self.n = lib, lib.shape(w)[1]
        self.q = lib._check(lib.pg_amd_mx4_quantize(w, 0))

    def __call__(self, x: int, dtype: int = F32) -> int:
        y = empty(self.lib, (self.lib.shape(x)[0], self.n), dtype)
        if not self.lib.pg_amd_mx4_matmul(x, self.q, y):
            self.lib.pg_tensor_free(y)
            raise RuntimeError(self.lib.pg_autograd_last_error().decode())
        return y

    def free(self) -> None:
        self.lib.pg_amd_mx4_free(self.q)
        self.q = None


class Q8:
    """The same in 8 bits."""

    def __init__(self, lib: PgLib, w: int):
        self.lib, self.n = lib, lib.shape(w)[1]
        self.q = lib._check(lib.pg_amd_q8_quantize(w, 0))

    def __call__(self, x: int, dtype: int = F32) -> int:
        y = empty(self.lib, (self.lib.shape(x)[0], self.n), dtype)
        if not self.lib.pg_amd_q8_matmul(x, self.q, y):
            self.lib.pg_tensor_free(y)
            raise RuntimeError(self.lib.pg_autograd_last_error().decode())
        return y

    def free(self) -> None:
        self.lib.pg_amd_q8_free(self.q)
        self.q = None


def empty(lib: PgLib, shape, dtype: int = F32) -> int:
    nd, sh = shape_arg(shape)
    t = lib.pg_tensor_empty_dtype(dtype, nd, sh)
    if not t:
        raise RuntimeError(f"pg_tensor_empty_dtype: {lib.pg_amd_last_error().decode()}")
    return t


def to_bf16(a: np.ndarray) -> np.ndarray:
    """The bits of finite values, rounded to nearest even."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    return ((u + np.uint32(0x7FFF) + ((u >> 16) & np.uint32(1))) >> 16).astype(np.uint16)


class Teacher:
    """logits = gelu(Q(x) W1 + b1) W2, both matrices in 4 bits."""

    def __init__(self, lib: PgLib, w1: np.ndarray, b1: np.ndarray, w2: np.ndarray):
        self.lib = lib
        self.m = []
        for w in (w1, w2):
            t = lib.tensor(w)
            self.m.append(Mx4(lib, t))
            lib.pg_tensor_free(t)
        self.b1 = lib.var(b1, False)

    def logits(self, x: int) -> int:
        L = self.lib
        t = self.m[0](x)
        z = L._check(L.pg_var_from_tensor(t, False))
        s = L.op("add", z, self.b1)
        h = L.op("gelu", s)
        y = self.m[1](L.node(h).value)
        for n in (h, s, z):
            L.pg_node_free(n)
        L.pg_tensor_free(t)
        return y

    def top(self, x: np.ndarray, k: int, batch: int = 1024) -> tuple[np.ndarray, np.ndarray]:
        """The k highest logits of every row and their indices (f32), highest first."""
        values, idx = [], []
        for i in range(0, len(x), batch):
            t = self.lib.tensor(x[i:i + batch])
            y = self.logits(t)
            v = self.lib.read(y)
            at = np.argsort(-v, axis=1, kind="stable")[:, :k]
            values.append(np.take_along_axis(v, at, 1))
            idx.append(at.astype(np.float32))
            self.lib.pg_tensor_free(y)
            self.lib.pg_tensor_free(t)
        return np.concatenate(values), np.concatenate(idx)

    def free(self) -> None:
        for m in self.m:
            m.free()
        self.lib.pg_node_free(self.b1)


class Student:
    """A gated layer and a linear one, with a layer norm between them where asked: x [M, K] -> logits [M, classes]."""

    def __init__(self, lib: PgLib, k: int, f: int, classes: int, rng: np.random.Generator, dtype: int = BF16,
                 lr: float = 2e-3, norm: bool = False, muon: bool = False, muon_lr: float = 0.02):
        self.lib, self.dtype, self.norm, self.muon = lib, dtype, norm, None
        shapes = [(k, 2 * f), (2 * f,), (f, classes), (classes,)]
        self.params = [lib.var((rng.uniform(-1, 1, s) * s[0] ** -0.5 if len(s) == 2 else np.zeros(s)).astype(np.float32))
                       for s in shapes]
        if norm:  # weight and bias
            self.params += [lib.var(np.full(f, v, np.float32)) for v in (1.0, 0.0)]
        self.opt = lib._check(lib.pg_adam_new(C.byref(AdamCfg(lr, 0.9, 0.999, 1e-8, 1e-2, False, True))))
        if muon:
            self.muon = lib._check(lib.pg_amd_muon_new(C.byref(MuonCfg(muon_lr, 0.95, 1e-2, 0.0, 5, True))))
        for i, p in enumerate(self.params):
            if muon and i in (0, 2):
                if lib.pg_amd_muon_add_param(self.muon, p) != 0:
                    raise RuntimeError(lib.pg_autograd_last_error().decode())
            elif lib.pg_adam_add_param(self.opt, p) != 0:
                raise RuntimeError("pg_adam_add_param failed")

    def forward(self, x: int) -> list[int]:
        """The nodes of the hidden values (then of the normalised ones, with a norm) and the logits."""
        L, (w, b, wo, bo) = self.lib, self.params[:4]
        made = [L._check(L.pg_amd_ag_gated16(x, w, b, ACT_SILU, self.dtype))]
        if self.norm:
            made.append(L.op("layernorm", made[0], self.params[4], self.params[5], NORM_EPS))
        return made + [L._check(L.pg_amd_ag_linear16(made[-1], wo, bo, ACT_NONE, self.dtype))]

    def step(self, x: int, top: int, idx: int, labels: int, cfg: DistillCfg) -> int:
        """One training step; the loss as a node, for the caller to free."""
        L = self.lib
        L.pg_adam_zero_grad(self.opt)
        if self.muon:
            L.pg_amd_muon_zero_grad(self.muon)
        made = self.forward(x)
        loss = L._check(L.pg_amd_ag_distill(made[-1], top, idx, labels, C.byref(cfg)))
        L.pg_backward(loss)
        L.pg_adam_step(self.opt)
        if self.muon and not L.pg_amd_muon_step(self.muon):
            raise RuntimeError(L.pg_autograd_last_error().decode())
        for n in reversed(made):
            L.pg_node_free(n)
        return loss

    def freeze(self, bits: int = 4) -> "Served":
        return Served(self, bits)

    def free(self) -> None:
        self.lib.pg_adam_free(self.opt)
        if self.muon:
            self.lib.pg_amd_muon_free(self.muon)
        for p in self.params:
            self.lib.pg_node_free(p)


class Served:
    """A student's weights as they are served: the gated layer's in bf16, the
    output layer's in 4 or 8 bits."""

    def __init__(self, student: Student, bits: int = 4):
        L = self.lib = student.lib
        w, b, wo, bo = (L.value(p) for p in student.params[:4])
        self.f = w.shape[1] // 2
        self.w, self.b, self.bo = L.tensor(to_bf16(w), BF16), L.tensor(b), L.var(bo, False)
        self.norm = [L.tensor(L.value(p)) for p in student.params[4:]]
        t = L.tensor(wo)
        self.out = {4: Mx4, 8: Q8}[bits](L, t)
        L.pg_tensor_free(t)

    def logits(self, x: np.ndarray) -> np.ndarray:
        """Of any number of rows; one row is what a single answer costs."""
        L = self.lib
        t, h = L.tensor(to_bf16(x), BF16), empty(L, (len(x), self.f), BF16)
        if not L.pg_amd_gated(t, self.w, self.b, ACT_SILU, h, None):
            raise RuntimeError(L.pg_autograd_last_error().decode())
        if self.norm and not L.pg_amd_layernorm(h, *self.norm, NORM_EPS, h, None):
            raise RuntimeError(L.pg_autograd_last_error().decode())
        y = self.out(h)
        n = L._check(L.pg_var_from_tensor(y, False))
        s = L.op("add", n, self.bo)
        got = L.value(s)
        for node in (s, n):
            L.pg_node_free(node)
        for tensor in (y, h, t):
            L.pg_tensor_free(tensor)
        return got

    def free(self) -> None:
        for t in (self.w, self.b, *self.norm):
            self.lib.pg_tensor_free(t)
        self.lib.pg_node_free(self.bo)
        self.out.free()


def train(lib: PgLib, steps: int = 500, rows: int = 8192, classes: int = 1000, k: int = 64, hidden: int = 256, f: int = 192,
          top: int = 32, batch: int = 512, temperature: float = 2.0, alpha: float = 0.8, seed: int = 0, say=print,
          norm: bool = False, muon: bool = False, bits: int = 4) -> dict:
    """The losses, and the student's agreement with the teacher before and after."""
    rng = np.random.default_rng(seed)
    teacher = Teacher(lib, (rng.standard_normal((k, hidden)) * k ** -0.5).astype(np.float32),
                      (rng.standard_normal(hidden) * 0.1).astype(np.float32),
                      (rng.standard_normal((hidden, classes)) * 4 * hidden ** -0.5).astype(np.float32))
    held = max(256, rows // 8)
    centres = rng.standard_normal((64, k))  # the rows gather round a few points, as real ones do
    x = (centres[rng.integers(0, 64, rows + held)] + 0.15 * rng.standard_normal((rows + held, k))).astype(np.float32)
    values, idx = teacher.top(x, top)
    teacher.free()
    labels = idx[:, 0].copy()  # the teacher's choice, a tenth of them unknown
    labels[rng.random(len(labels)) < 0.1] = -1
    student = Student(lib, k, f, classes, rng, norm=norm, muon=muon)
    batch = min(batch, rows)
    cfg = DistillCfg(temperature, alpha, 1.0 / batch)
    batches = []
    for i in range(0, rows - batch + 1, batch):
        part = slice(i, i + batch)
        batches.append((lib.var(x[part], False), lib.tensor(values[part]), lib.tensor(idx[part]), lib.tensor(labels[part])))

    def agreement() -> float:
        served = student.freeze(bits)
        got = served.logits(x[rows:])
        served.free()
        return float((got.argmax(1) == idx[rows:, 0]).mean())

    before, losses = agreement(), []
    lib.sync()
    start = time.perf_counter()
    for i in range(steps):
        loss = student.step(*batches[i % len(batches)], cfg)
        if i % 100 == 0 or i + 1 == steps:
            losses.append(float(lib.value(loss)[0]))
            say(f"step {i}: loss {losses[-1]:.4f}")
        lib.pg_node_free(loss)
    lib.sync()
    ms = (time.perf_counter() - start) * 1e3 / max(steps, 1)
    after = agreement()
    served = student.freeze(bits)
    one = served.logits(x[rows:rows + 1])
    say(f"{ms:.3f} ms a step; agreement with the teacher on {held} rows {before:.3f} -> {after:.3f}; "
        f"row {rows} alone: class {int(one.argmax())}, the teacher's {int(idx[rows, 0])}")
    served.free()
    for node, *tensors in batches:
        lib.pg_node_free(node)
        for t in tensors:
            lib.pg_tensor_free(t)
    student.free()
    return {"losses": losses, "before": before, "after": after, "one": one, "ms": ms}


def main() -> None:
    p = argparse.ArgumentParser(description="Train a gated student on a 4-bit teacher's top logits.")
    p.add_argument("--steps", type=int, default=500)
    p.add_argument("--rows", type=int, default=8192)
    p.add_argument("--classes", type=int, default=1000)
    p.add_argument("--seed", type=int, default=0)
    p.add_argument("--norm", action="store_true", help="a layer norm behind the gated layer")
    p.add_argument("--muon", action="store_true", help="orthogonalised updates for the student's matrices")
    p.add_argument("--bits", type=int, choices=(4, 8), default=4, help="of the served output layer")
    a = p.parse_args()
    if min(a.steps, a.rows, a.classes) < 1 or a.classes < 32:
        p.error("at least one step and row, and 32 classes")
    train(load(), a.steps, a.rows, a.classes, seed=a.seed, norm=a.norm, muon=a.muon, bits=a.bits)


if __name__ == "__main__":
    main()
