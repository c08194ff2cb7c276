"""Training a normalised network with orthogonalised updates and serving it from 8-bit weights, as cases to time.

Three operators of this library, the pieces of one program: layers are
normalised, their weights learn by orthogonalised momentum, and what was
learnt is served as 8-bit products of the normalised rows.

  norm     y = (x - mean) rstd w + b over the last dimension of x [M, D], with
           rstd = 1 / sqrt(var + eps) and var the mean of (x - mean)^2, w and b
           f32 or left out (pg_amd_layernorm); with "train" also dx, of x's
           type, and dw, db (f32, the sums over the rows) for a given dy
           (pg_amd_layernorm_backward)
  ortho    the orthogonal factor of a matrix G by Newton-Schulz products:
           X = G / ||G||_F, then `steps` times X <- a X + (b S + c S S) X with
           S = X X^T (of a tall G its transpose is taken), (a, b, c) =
           (3.4445, -4.7750, 2.0315) (pg_amd_orthogonalise)
  muon     a step over a network's matrices W [K, N] with grads g: m <- mu m + g,
           u = g + mu m, W <- (1 - lr wd) W - lr sqrt(max(1, N / K)) O with O the
           orthogonal factor of u (pg_amd_muon_step)
  q8       y = Q(x) Q(W): every row of x [M, K] and column of W [K, N] rounded to
           whole numbers q of -127 .. 127 with a scale s of its own, s = max |v| /
           127 in f32 and q = v / s to nearest, ties to even; W is held in 8
           bits, x is rounded in the call (pg_amd_q8_matmul)
  q8_keep  a matrix rounded to that form and read back as the values it then
           stands for (pg_amd_q8_quantize, pg_amd_q8_dequantize)

prepare() makes what a program holds before the call, run() makes one pass,
exact() gives the same values from the definitions above in 64 bits.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

own = False  # True: run() calls this library; False: the plain form

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NS = (3.4445, -4.7750, 2.0315)
EPS = 1e-5  # of the norm
MU, LR, WD = 0.95, 0.02, 0.01  # of the step

# the largest cases that draw() gives
MOST_NORM = 8192 * 8192
MOST_NS = 4096 * 4096 * 4096
MOST_Q8 = 8192 * 4096 * 4096


def listed() -> list[dict]:
    return [
        # one token's row before a served layer: latency
        {"name": "norm-bf16-1x4096", "kind": "norm", "dtype": "bf16", "m": 1, "d": 4096, "affine": True, "train": False},
        # a step's rows at an odd width: rows start anywhere
        {"name": "norm-train-f32-1000x777", "kind": "norm", "dtype": "f32", "m": 1000, "d": 777, "affine": True,
         "train": True},
        # long rows, few of them, without weights
        {"name": "norm-train-f16-33x50001", "kind": "norm", "dtype": "f16", "m": 33, "d": 50001, "affine": False,
         "train": True},
        # a large step: 134 MB each of x, dy, y and dx
        {"name": "norm-train-bf16-8192x8192", "kind": "norm", "dtype": "bf16", "m": 8192, "d": 8192, "affine": True,
         "train": True},
        # the update of a small layer: the chain of dependent products
        {"name": "ortho-f32-64x64", "kind": "ortho", "dtype": "f32", "k": 64, "n": 64, "steps": 5},
        # a tall 16-bit grad of odd sizes
        {"name": "ortho-bf16-2049x777", "kind": "ortho", "dtype": "bf16", "k": 2049, "n": 777, "steps": 5},
        # one wide layer of the benchmark network
        {"name": "ortho-f32-1024x4096", "kind": "ortho", "dtype": "f32", "k": 1024, "n": 4096, "steps": 5},
        # a step over all of the benchmark network's matrices
        {"name": "muon-1024x4096x4096x4096x10", "kind": "muon", "dtype": "f32",
         "shapes": "1024x4096 4096x4096 4096x4096 4096x10", "steps": 5},
        # one token against a layer's 8-bit weights
        {"name": "q8-bf16-1x4096x4096", "kind": "q8", "dtype": "bf16", "out": "bf16", "m": 1, "k": 4096, "n": 4096},
        # ragged, from and to f32
        {"name": "q8-f32-333x1000x2049", "kind": "q8", "dtype": "f32", "out": "f32", "m": 333, "k": 1000, "n": 2049},
        # a large batch of served rows
        {"name": "q8-bf16-8192x4096x4096", "kind": "q8", "dtype": "bf16", "out": "bf16", "m": 8192, "k": 4096, "n": 4096},
        # a layer's f32 weights taken into 8 bits and read back
        {"name": "q8-keep-f32-4096x4096", "kind": "q8_keep", "dtype": "f32", "k": 4096, "n": 4096},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """Whole number from lo to hi, even over its logarithm; 32's multiples half of the time where they fit."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.5:
        v -= v % 32
    return min(max(v, lo), hi)


def _products(shapes) -> int:
    """Of a chain of steps over these matrices, in multiply-adds of one product with X."""
    return sum(k * n * min(k, n) for k, n in shapes)


def _shapes(case) -> list:
    if case["kind"] == "ortho":
        return [(case["k"], case["n"])]
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split()]


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "ortho", "ortho", "muon", "q8", "q8", "q8_keep"])
    while True:
        if kind == "norm":
            c = {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "m": _log(rng, 1, 16384),
                 "d": _log(rng, 8, 65536), "affine": rng.random() < 0.7, "train": rng.random() < 0.7}
            if c["m"] * c["d"] * (2 if c["dtype"] == "f32" else 1) <= MOST_NORM:
                return c
        elif kind == "ortho":
            return {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "k": _log(rng, 1, 4096),
                    "n": _log(rng, 1, 4096), "steps": rng.choice([3, 5, 5, 6])}
        elif kind == "muon":
            shapes = [(_log(rng, 8, 4096), _log(rng, 8, 4096)) for _ in range(rng.choice([1, 2, 3, 4]))]
            if _products(shapes) <= MOST_NS:
                return {"kind": kind, "dtype": "f32", "shapes": " ".join("%dx%d" % s for s in shapes), "steps": 5}
        elif kind == "q8":
            c = {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "out": rng.choice(["f32", "f16", "bf16"]),
                 "m": _log(rng, 1, 8192), "k": _log(rng, 32, 8192), "n": _log(rng, 16, 8192)}
            if c["m"] * c["k"] * c["n"] <= MOST_Q8:
                return c
        else:
            return {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "k": _log(rng, 32, 4096),
                    "n": _log(rng, 16, 4096)}


# ---------------------------------------------------------------- inputs, from the seed alone

def _inputs(case, seed) -> dict:
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    flat = lambda *shape: torch.rand(shape, generator=g, device="cuda")  # noqa: E731
    kind, dt = case["kind"], TORCH[case["dtype"]]

    def grad(k, n):
        """A sum over samples: some directions carry most of it."""
        r = min(k, n)
        strength = torch.exp(-4.0 * torch.arange(r, device="cuda") / r)
        return (normal(k, r) * strength) @ normal(r, n) * (1e-2 * (k * n) ** -0.25)

    if kind == "norm":
        m, d = case["m"], case["d"]
        # a few channels larger than the others, an offset per channel
        v = {"x": (normal(m, d) * torch.exp(normal(d) * 0.5) + 0.5 * normal(d)).to(dt)}
        if case["affine"]:
            v["w"], v["b"] = 1 + 0.2 * normal(d), 0.1 * normal(d)
        if case["train"]:
            v["dy"] = (normal(m, d) * 0.1).to(dt)
        return v
    if kind == "ortho":
        return {"g": grad(case["k"], case["n"]).to(dt)}
    if kind == "muon":
        v = {}
        for i, (k, n) in enumerate(_shapes(case)):
            v["w%d" % i] = (flat(k, n) * 2 - 1) * k ** -0.5
            v["g%d" % i] = grad(k, n)
            v["m%d" % i] = grad(k, n) * 8  # what earlier steps left
        return v
    if kind == "q8":
        m, k, n = case["m"], case["k"], case["n"]
        # a normalised row's channels under a norm's weights
        x = normal(m, k) * torch.exp(normal(k) * 0.5)
        return {"x": x.to(dt), "w": (flat(k, n) * 2 - 1) * k ** -0.5}
    return {"w": (normal(case["k"], case["n"]) * 0.02).to(dt)}


# ---------------------------------------------------------------- the state: what a program holds before the call

class _Memory:
    """Device memory of the library, for torch."""

    def __init__(self, ptr: int, shape, kind: str):
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": tuple(shape), "typestr": kind, "version": 3,
                                         "strides": None}


class _State:
    def __init__(self, case, v):
        self.case, self.v = case, v
        self.L, self.t, self.out, self.frees = None, {}, {}, []

    # the library's side
    def view(self, p, shape, dtype=torch.float32):
        from picograd_amd.capi import PgTensorAmd
        wide = dtype == torch.float32
        view = torch.as_tensor(_Memory(PgTensorAmd.from_address(p).dev, shape, "<f4" if wide else "<i2"), device="cuda")
        return view if wide else view.view(dtype)

    def fill(self, view, like):
        self.L.sync()
        view.copy_(like)
        torch.cuda.synchronize()

    def tensor(self, name, like=None, shape=None, dtype=None):
        """A device tensor of the library with `like`'s elements, or an unset one; its torch view."""
        from picograd_amd.capi import BF16, F16, F32, shape_arg
        dtype = like.dtype if like is not None else dtype
        size = torch.Size(like.shape if like is not None else shape)
        nd, sh = shape_arg(size)
        p = self.L.pg_tensor_empty_dtype({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}[dtype], nd, sh)
        if not p:
            raise RuntimeError(self.L.pg_amd_last_error().decode())
        self.frees.append((self.L.pg_tensor_free, p))
        view = self.view(p, size, dtype)
        if like is not None:
            self.fill(view, like)
        self.t[name] = p
        return view

    def result(self, name, shape, dtype):
        self.out[name] = self.tensor(name, shape=shape, dtype=dtype)

    def __del__(self):
        self.out = {}
        for f, p in reversed(self.frees):
            f(p)


_LIB = []


def _lib():
    import picograd_amd
    if not _LIB:
        L = picograd_amd.load()
        if L.pg_amd_init() != 0:
            raise RuntimeError(L.pg_amd_last_error().decode())
        _LIB.append(L)
    return _LIB[0]


def prepare(case, seed) -> _State:
    v = _inputs(case, seed)
    s = _State(case, v)
    if case["kind"] == "q8":
        v["wq"], v["ws"] = _q8(v["w"].t())  # the plain form's weights: whole numbers and scales in 32 bits
        v["wq"] = v["wq"].t().contiguous()
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


def _prepare_own(s) -> None:
    L = s.L = _lib()
    case, v, kind = s.case, s.v, s.case["kind"]
    dt = TORCH[case["dtype"]]
    if kind == "muon":
        from picograd_amd.capi import MuonCfg
        s.opt = L.pg_amd_muon_new(C.byref(MuonCfg(LR, MU, WD, 0.0, case["steps"], True)))
        if not s.opt:
            raise RuntimeError(L.pg_autograd_last_error().decode())
        s.frees.append((L.pg_amd_muon_free, s.opt))
        for i, shape in enumerate(_shapes(case)):
            s.tensor("g%d" % i, v["g%d" % i])
            s.tensor("w%d" % i, v["w%d" % i])
            n = L._check(L.pg_var_from_tensor(s.t["w%d" % i], True))
            s.frees.append((L.pg_node_free, n))
            zero = L._check(L.pg_var_scalar(0.0, False))
            loss = L.op("add", n, zero)
            L.pg_amd_backward_from(loss, s.t["g%d" % i])  # the node's grad
            for node in (loss, zero):
                L.pg_node_free(node)
            if L.pg_amd_muon_add_param(s.opt, n) != 0:
                raise RuntimeError(L.pg_autograd_last_error().decode())
            s.out["w%d" % i] = s.view(L.node(n).value, shape)
            s.out["m%d" % i] = s.view(L.pg_amd_muon_buffer(s.opt, i), shape)
            s.fill(s.out["m%d" % i], v["m%d" % i])
        L.sync()
        return
    for name in ("x", "w", "b", "dy", "g"):
        if name in v:
            s.tensor(name, v[name])
    if kind == "norm":
        m, d = case["m"], case["d"]
        s.result("y", (m, d), dt)
        if case["train"]:
            s.tensor("stats", shape=(m, 2), dtype=torch.float32)
            s.result("dx", (m, d), dt)
            s.result("dw", (d,), torch.float32)
            s.result("db", (d,), torch.float32)
    elif kind == "ortho":
        s.result("o", (case["k"], case["n"]), dt)
    elif kind == "q8":
        s.w8 = L.pg_amd_q8_quantize(s.t["w"], 0)
        if not s.w8:
            raise RuntimeError(L.pg_autograd_last_error().decode())
        s.frees.append((L.pg_amd_q8_free, s.w8))
        s.result("y", (case["m"], case["n"]), TORCH[case["out"]])
    else:
        s.source = s.t["w"]
        s.result("w", (case["k"], case["n"]), torch.float32)
    L.sync()


# ---------------------------------------------------------------- one pass

def run(s) -> dict:
    return (_OWN if own else _PLAIN)[s.case["kind"]](s)


def _ok(s, done):
    if not done:
        raise RuntimeError(s.L.pg_autograd_last_error().decode() or s.L.pg_amd_last_error().decode())


def _own_norm(s):
    t = s.t
    _ok(s, s.L.pg_amd_layernorm(t["x"], t.get("w"), t.get("b"), EPS, t["y"], t.get("stats")))
    if s.case["train"]:
        _ok(s, s.L.pg_amd_layernorm_backward(t["x"], t.get("w"), t["stats"], t["dy"], t["dx"], t["dw"], t["db"]))
    return s.out


def _own_ortho(s):
    _ok(s, s.L.pg_amd_orthogonalise(s.t["g"], s.case["steps"], s.t["o"]))
    return s.out


def _own_muon(s):
    _ok(s, s.L.pg_amd_muon_step(s.opt))
    return s.out


def _own_q8(s):
    _ok(s, s.L.pg_amd_q8_matmul(s.t["x"], s.w8, s.t["y"]))
    return s.out


def _own_q8_keep(s):
    q = s.L.pg_amd_q8_quantize(s.source, 0)
    _ok(s, q)
    _ok(s, s.L.pg_amd_q8_dequantize(q, s.t["w"]))
    s.L.pg_amd_q8_free(q)
    return s.out


_OWN = {"norm": _own_norm, "ortho": _own_ortho, "muon": _own_muon, "q8": _own_q8, "q8_keep": _own_q8_keep}


# ---------------------------------------------------------------- the plain form, in 32 bits

def _plain_norm(s):
    c, v = s.case, s.v
    dt = TORCH[c["dtype"]]
    x = v["x"].float()
    mean = x.mean(1, keepdim=True)
    r = x - mean
    rstd = 1 / torch.sqrt((r * r).mean(1, keepdim=True) + EPS)
    n = r * rstd
    y = n * v["w"] + v["b"] if c["affine"] else n
    out = {"y": y.to(dt)}
    if c["train"]:
        dy = v["dy"].float()
        h = dy * v["w"] if c["affine"] else dy
        dx = rstd * (h - h.mean(1, keepdim=True) - n * (h * n).mean(1, keepdim=True))
        out["dx"] = dx.to(dt)
        out["dw"] = (dy * n).sum(0)
        out["db"] = dy.sum(0)
    return out


def _factor(g, steps):
    """The orthogonal factor of g, in 32 bits (its norm summed in 64)."""
    a, b, c = NS
    size = torch.sqrt(g.double().square().sum())
    x = (g.double() / torch.where(size > 0, size, torch.ones_like(size))).float()
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.t().contiguous()
    for _ in range(steps):
        t = x @ x.t().contiguous()
        x = a * x + (b * t + c * (t @ t)) @ x
    return x.t().contiguous() if tall else x


def _plain_ortho(s):
    return {"o": _factor(s.v["g"].float(), s.case["steps"]).to(TORCH[s.case["dtype"]])}


def _plain_muon(s):
    v, out = s.v, {}
    for i, (k, n) in enumerate(_shapes(s.case)):
        w, g, m = v["w%d" % i], v["g%d" % i], v["m%d" % i]
        m.mul_(MU).add_(g)
        o = _factor(g + MU * m, s.case["steps"])
        w.mul_(1 - LR * WD).sub_(o * (LR * math.sqrt(max(1.0, n / k))))
        out["w%d" % i], out["m%d" % i] = w, m
    return out


def _q8(v):
    """v [R, K] as whole numbers in 32 bits and a scale for each row; quotients next to a border in 64."""
    v = v.float()
    scale = (v.abs().amax(1, keepdim=True).double() / 127).float()
    q = torch.round(v.double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double())
    return q.clamp(-127, 127).float(), scale


def _plain_q8(s):
    q, scale = _q8(s.v["x"])
    return {"y": ((q @ s.v["wq"]) * scale * s.v["ws"].t()).to(TORCH[s.case["out"]])}


def _plain_q8_keep(s):
    q, scale = _q8(s.v["w"].t())
    return {"w": (q * scale).t().contiguous()}


_PLAIN = {"norm": _plain_norm, "ortho": _plain_ortho, "muon": _plain_muon, "q8": _plain_q8, "q8_keep": _plain_q8_keep}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case) -> dict:
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    e = size[case["dtype"]]
    if kind == "norm":
        m, d = case["m"], case["d"]
        affine = 8 * d if case["affine"] else 0
        if not case["train"]:
            return {"bytes": 2 * m * d * e + affine, "flops": 8 * m * d}
        return {"bytes": 4 * m * d * e + affine + 8 * d, "flops": 22 * m * d}
    if kind in ("ortho", "muon"):
        flops = moved = 0
        for k, n in _shapes(case):
            lo, hi = min(k, n), max(k, n)
            # S and S S are symmetric: half of their products
            flops += case["steps"] * (lo * lo * hi + lo * lo * lo + 2 * lo * lo * hi)
            # g and o; or w and m in and out, and g
            moved += k * n * (2 * e if kind == "ortho" else 20)
        return {"bytes": moved, "flops": flops}
    k, n = case["k"], case["n"]
    if kind == "q8":
        m = case["m"]
        return {"bytes": m * k * e + n * (k + 4) + m * n * size[case["out"]], "flops": 2 * m * k * n}
    return {"bytes": k * n * (e + 4), "flops": 5 * k * n}


# ---------------------------------------------------------------- the same values in 64 bits

def _orthogonal(g, steps):
    """Of g in 64 bits: the products on the short side, over G G^T or G^T G."""
    size = torch.linalg.matrix_norm(g)
    x = g / size if float(size) > 0 else g
    one = torch.eye(min(x.shape), dtype=x.dtype, device=x.device)
    for _ in range(steps):
        xt = x.t().contiguous()
        t = x @ xt if x.shape[0] <= x.shape[1] else xt @ x
        p = NS[0] * one + t @ (NS[1] * one + NS[2] * t)
        x = p @ x if x.shape[0] <= x.shape[1] else x @ p
    return x


def _whole(v):
    """v [R, K] with its rows rounded to 8 bits, in 64 bits."""
    scale = (v.abs().max(1).values / 127).float().double().unsqueeze(1)
    t = v / torch.where(scale == 0, torch.full_like(scale, math.inf), scale)
    low = torch.floor(t)
    up = (t - low > 0.5) | ((t - low == 0.5) & (torch.remainder(low, 2) == 1))
    return torch.clamp(low + up, -127, 127) * scale


def exact(case, seed):
    v = {k: t.double() for k, t in _inputs(case, seed).items()}
    kind = case["kind"]
    if kind == "norm":
        x = v["x"].requires_grad_()
        d = case["d"]
        w = v.get("w", torch.ones(d, dtype=torch.float64, device="cuda")).requires_grad_()
        b = v.get("b", torch.zeros(d, dtype=torch.float64, device="cuda")).requires_grad_()
        with torch.enable_grad():
            centred = x - x.sum(1, keepdim=True) / d
            y = centred * torch.rsqrt((centred ** 2).sum(1, keepdim=True) / d + EPS) * w + b
            if not case["train"]:
                return {"y": y.detach()}
            grads = torch.autograd.grad(y, (x, w, b), v["dy"])
        return {"y": y.detach(), "dx": grads[0], "dw": grads[1], "db": grads[2]}
    if kind == "ortho":
        return {"o": _orthogonal(v["g"], case["steps"])}
    if kind == "muon":
        out = {}
        for i, (k, n) in enumerate(_shapes(case)):
            m = MU * v["m%d" % i] + v["g%d" % i]
            o = _orthogonal(v["g%d" % i] + MU * m, case["steps"])
            out["w%d" % i] = v["w%d" % i] * (1 - LR * WD) - LR * max(1.0, n / k) ** 0.5 * o
            out["m%d" % i] = m
        return out
    if kind == "q8":
        return {"y": _whole(v["x"]) @ _whole(v["w"].t().contiguous()).t().contiguous()}
    return {"w": _whole(v["w"].t().contiguous()).t().contiguous()}
