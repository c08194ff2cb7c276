"""Distilling a network into a gated one and serving it from 4-bit weights, as cases to time.

Three operators of this library, the pieces of one program: a teacher whose
layers are 4-bit products gives top logits, a student of gated feed-forward
layers learns from them through the distillation loss.

  gated    h = act(x Wg + bg) * (x Wu + bu) for x [M, K], W = [Wg | Wu] [K, 2F]
           and b = [bg | bu] [2F], all operands of one 16-bit type, b f32
           (pg_amd_gated); with "train" also dx, dW and db for a given dh
           (pg_amd_gated_backward)
  distill  per row of logits s [N, V], with the teacher's logits t_k at the
           indices i_k of its top entries (a negative index is padding):
           scale * (alpha T^2 KL(softmax(t / T) || softmax(s / T)) +
           (1 - alpha) CE(s, label)); a row without entries has no first
           part, one with a negative label no second (pg_amd_distill); with
           "train" also the grad of the logits, of the logits' type
  mx4      y = Q(x) Q(W), both rounded to 4-bit values (e2m1: 0, .5, 1, 1.5,
           2, 3, 4, 6 and their negatives) with one power of two for each 32
           values along the reduction: 2^(floor(log2(max |v|)) - 2); W is held
           in 4 bits, x is rounded in the call (pg_amd_mx4_matmul)
  mx4_keep a matrix rounded to that form along its rows' direction and
           read back as the values it then stands for (pg_amd_mx4_quantize,
           pg_amd_mx4_dequantize)

prepare() makes what a program holds before the call, run() makes one pass,
exact() gives the same values from the definitions above in 64 bits.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

own = False  # True: run() calls this library; False: the plain form

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3, "sigmoid": 4}  # PG_ACT_*
MX_BLOCK = 32

# the largest cases that draw() gives
MOST_GATED = 4096 * 4096 * 8192
MOST_LOGITS = 4096 * 131072
MOST_MX4 = 8192 * 4096 * 4096


def listed() -> list[dict]:
    return [
        # one token through a served layer: the weights stream past once, latency counts
        {"name": "gated-bf16-1x1024x4096", "kind": "gated", "dtype": "bf16", "m": 1, "k": 1024, "f": 4096,
         "act": "silu", "bias": False, "train": False},
        # a step of one layer at the benchmark network's widths and an ordinary batch
        {"name": "gated-train-bf16-512x1024x4096", "kind": "gated", "dtype": "bf16", "m": 512, "k": 1024, "f": 4096,
         "act": "silu", "bias": False, "train": True},
        # a ragged step: no size fits a tile, the halves of W do not start on 16 bytes
        {"name": "gated-train-f16-1023x777x2049", "kind": "gated", "dtype": "f16", "m": 1023, "k": 777, "f": 2049,
         "act": "gelu", "bias": True, "train": True},
        # a large step
        {"name": "gated-train-bf16-4096x4096x8192", "kind": "gated", "dtype": "bf16", "m": 4096, "k": 4096, "f": 8192,
         "act": "silu", "bias": False, "train": True},
        # the benchmark network's ten classes at its batch, labels beside a few teacher entries: latency
        {"name": "distill-train-f32-4096x10", "kind": "distill", "dtype": "f32", "n": 4096, "v": 10, "top": 4,
         "labels": True, "temperature": 2.0, "alpha": 0.7, "train": True},
        # an odd vocabulary at an ordinary batch, every option in use
        {"name": "distill-train-f32-1000x50001", "kind": "distill", "dtype": "f32", "n": 1000, "v": 50001, "top": 17,
         "labels": True, "temperature": 1.7, "alpha": 0.5, "train": True},
        # a large batch of long rows: 1 GiB of logits
        {"name": "distill-train-bf16-4096x131072", "kind": "distill", "dtype": "bf16", "n": 4096, "v": 131072,
         "top": 64, "labels": False, "temperature": 1.0, "alpha": 1.0, "train": True},
        # the loss alone over a few long rows, as an evaluation takes it
        {"name": "distill-f16-16x131072", "kind": "distill", "dtype": "f16", "n": 16, "v": 131072, "top": 32,
         "labels": True, "temperature": 2.0, "alpha": 0.5, "train": False},
        # one token against a layer's 4-bit weights
        {"name": "mx4-bf16-1x4096x4096", "kind": "mx4", "dtype": "bf16", "out": "bf16", "m": 1, "k": 4096, "n": 4096},
        # ragged, from and to f32: a reduction that ends inside a block
        {"name": "mx4-f32-333x1000x2049", "kind": "mx4", "dtype": "f32", "out": "f32", "m": 333, "k": 1000, "n": 2049},
        # a large batch of a teacher's rows
        {"name": "mx4-bf16-8192x4096x4096", "kind": "mx4", "dtype": "bf16", "out": "bf16", "m": 8192, "k": 4096,
         "n": 4096},
        # a layer's f32 weights taken into 4 bits and read back
        {"name": "mx4-keep-f32-4096x4096", "kind": "mx4_keep", "dtype": "f32", "k": 4096, "n": 4096},
    ]


def _log(rng, lo: int, hi: int) -> int:
    """Whole number from lo to hi, even over its logarithm; 32's multiples half of the time where they fit."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 64 and rng.random() < 0.5:
        v -= v % 32
    return min(max(v, lo), hi)


def draw(rng) -> dict:
    kind = rng.choice(["gated", "gated", "distill", "distill", "mx4", "mx4", "mx4_keep"])
    while True:
        if kind == "gated":
            train = rng.random() < 0.6
            act = rng.choice(["silu", "silu", "gelu", "sigmoid", "relu", "none"])
            # relu's derivative jumps at zero, where another order of a sum may fall on the other side
            bias = rng.random() < 0.5 and not (train and act == "relu")
            c = {"kind": kind, "dtype": rng.choice(["f16", "bf16"]), "m": _log(rng, 1, 4096), "k": _log(rng, 16, 4096),
                 "f": _log(rng, 16, 8192), "act": act, "bias": bias, "train": train}
            if c["m"] * c["k"] * c["f"] <= MOST_GATED:
                return c
        elif kind == "distill":
            c = {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "n": _log(rng, 1, 8192),
                 "v": _log(rng, 10, 262144), "top": _log(rng, 1, 128), "labels": rng.random() < 0.5,
                 "temperature": rng.choice([1.0, 1.7, 2.0, 4.0]), "alpha": rng.choice([0.3, 0.5, 0.9, 1.0]),
                 "train": rng.random() < 0.7}
            size = 2 if c["dtype"] != "f32" else 4
            if c["n"] * c["v"] * size <= 2 * MOST_LOGITS and c["top"] <= c["v"]:
                return c
        elif kind == "mx4":
            c = {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16"]), "out": rng.choice(["f32", "f16", "bf16"]),
                 "m": _log(rng, 1, 8192), "k": _log(rng, 32, 8192), "n": _log(rng, 16, 8192)}
            if c["m"] * c["k"] * c["n"] <= MOST_MX4:
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
    if kind == "gated":
        m, k, f = case["m"], case["k"], case["f"]
        v = {"x": normal(m, k).to(dt), "w": ((flat(k, 2 * f) * 2 - 1) * k ** -0.5).to(dt)}
        if case["bias"]:
            v["b"] = normal(2 * f) * 0.1
        if case["train"]:
            v["dh"] = (normal(m, f) * 0.1).to(dt)
        return v
    if kind == "distill":
        n, vocab, top = case["n"], case["v"], case["top"]
        # distinct indices: steps of 1 .. V / top, from a random start
        step = 1 + (flat(n, top) * (vocab // top - 1)).long()
        idx = (step.cumsum(1) - 1 + (flat(n, 1) * vocab).long()) % vocab
        t, _ = (normal(n, top) * 2 + 6).sort(1, descending=True)
        # the student has learnt a part of what the teacher says
        s = normal(n, vocab) * 2
        s.scatter_add_(1, idx, 0.5 * t + normal(n, top))
        s = s.to(dt)
        # short lists are padded; some rows have none (their masked positions)
        idx = torch.where((flat(n, top) < 0.1) | (flat(n, 1) < 0.05), torch.full_like(idx, -1), idx)
        v = {"s": s, "t": t, "idx": idx.float()}
        if case["labels"]:
            lab = (flat(n) * vocab).long()
            v["label"] = torch.where(flat(n) < 0.1, torch.full_like(lab, -1), lab).float()
        return v
    if kind == "mx4":
        m, k, n = case["m"], case["k"], case["n"]
        # activations with a few large channels
        x = normal(m, k) * torch.exp(normal(k) * 0.7)
        return {"x": x.to(dt), "w": (flat(k, n) * 2 - 1) * k ** -0.5}
    return {"w": (normal(case["k"], case["n"]) * 0.02).to(dt)}


def _scale(case) -> float:
    """Of a mean over the rows; 16-bit floats of narrow range take the loss scaled up."""
    return 64.0 if case["dtype"] == "f16" else 1.0 / case["n"]


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
    def tensor(self, name, like=None, shape=None, dtype=None):
        """A device tensor of the library with `like`'s elements, or an unset one; its torch view."""
        from picograd_amd.capi import BF16, F16, F32, PgTensorAmd, shape_arg
        dtype = like.dtype if like is not None else dtype
        nd, sh = shape_arg(like.shape if like is not None else shape)
        p = self.L.pg_tensor_empty_dtype({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}[dtype], nd, sh)
        if not p:
            raise RuntimeError(self.L.pg_amd_last_error().decode())
        self.frees.append((self.L.pg_tensor_free, p))
        size = torch.Size(like.shape if like is not None else shape)
        wide = dtype == torch.float32
        view = torch.as_tensor(_Memory(PgTensorAmd.from_address(p).dev, size, "<f4" if wide else "<i2"), device="cuda")
        view = view if wide else view.view(dtype)
        if like is not None:
            self.L.sync()
            view.copy_(like)
            torch.cuda.synchronize()
        self.t[name] = p
        return view

    def result(self, name, shape, dtype):
        self.out[name] = self.tensor(name, shape=shape, dtype=dtype)

    def __del__(self):
        self.out = {}
        for f, p in self.frees:
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
    if case["kind"] == "mx4":
        v["wq"] = _mx4(v["w"].t()).t().contiguous()  # the plain form's weights: the values in 32 bits
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


def _prepare_own(s) -> None:
    L = s.L = _lib()
    case, v, kind = s.case, s.v, s.case["kind"]
    dt = TORCH[case["dtype"]]
    for name in ("x", "w", "b", "dh", "s", "t", "idx", "label"):
        if name in v:
            s.tensor(name, v[name])
    if kind == "gated":
        m, k, f = case["m"], case["k"], case["f"]
        s.result("h", (m, f), dt)
        if case["train"]:
            s.tensor("z", shape=(m, 2 * f), dtype=torch.float32)
            s.result("dx", (m, k), dt)
            s.result("dw", (k, 2 * f), dt)
            if case["bias"]:
                s.result("db", (2 * f,), torch.float32)
    elif kind == "distill":
        from picograd_amd.capi import DistillCfg
        s.cfg = DistillCfg(case["temperature"], case["alpha"], _scale(case))
        s.result("loss", (case["n"],), torch.float32)
        if case["train"]:
            s.result("ds", (case["n"], case["v"]), dt)
    elif kind == "mx4":
        s.w4 = L.pg_amd_mx4_quantize(s.t["w"], 0)
        if not s.w4:
            raise RuntimeError(L.pg_autograd_last_error().decode())
        s.frees.append((L.pg_amd_mx4_free, s.w4))
        s.result("y", (case["m"], case["n"]), TORCH[case["out"]])
    else:
        s.result("w", (case["k"], case["n"]), torch.float32)
        s.source = s.tensor("source", v["w"])
    L.sync()


# ---------------------------------------------------------------- one pass

def run(s) -> dict:
    return (_OWN if own else _PLAIN)[s.case["kind"]](s)


def _ok(s, done):
    if not done:
        raise RuntimeError(s.L.pg_autograd_last_error().decode() or s.L.pg_amd_last_error().decode())


def _own_gated(s):
    t, act = s.t, ACTS[s.case["act"]]
    _ok(s, s.L.pg_amd_gated(t["x"], t["w"], t.get("b"), act, t["h"], t.get("z")))
    if s.case["train"]:
        _ok(s, s.L.pg_amd_gated_backward(t["x"], t["w"], t["z"], t["dh"], act, t["dx"], t["dw"], t.get("db")))
    return s.out


def _own_distill(s):
    t = s.t
    _ok(s, s.L.pg_amd_distill(t["s"], t["t"], t["idx"], t.get("label"), C.byref(s.cfg), t["loss"], t.get("ds")))
    return s.out


def _own_mx4(s):
    _ok(s, s.L.pg_amd_mx4_matmul(s.t["x"], s.w4, s.t["y"]))
    return s.out


def _own_mx4_keep(s):
    q = s.L.pg_amd_mx4_quantize(s.t["source"], 0)
    _ok(s, q)
    _ok(s, s.L.pg_amd_mx4_dequantize(q, s.t["w"]))
    s.L.pg_amd_mx4_free(q)
    return s.out


_OWN = {"gated": _own_gated, "distill": _own_distill, "mx4": _own_mx4, "mx4_keep": _own_mx4_keep}


# ---------------------------------------------------------------- the plain form, in 32 bits

def _act(g, act):
    """act(g) and its derivative."""
    if act == "none":
        return g, torch.ones_like(g)
    if act == "relu":
        return torch.relu(g), (g > 0).to(g.dtype)
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    sg = 1 / (1 + torch.exp(-g))
    if act == "sigmoid":
        return sg, sg * (1 - sg)
    return g * sg, sg * (1 + g * (1 - sg))


def _plain_gated(s):
    c, v = s.case, s.v
    dt, f = TORCH[c["dtype"]], c["f"]
    x, w = v["x"].float(), v["w"].float()
    z = x @ w
    if c["bias"]:
        z = z + v["b"]
    g, u = z[:, :f], z[:, f:]
    a, da = _act(g, c["act"])
    out = {"h": (a * u).to(dt)}
    if c["train"]:
        dh = v["dh"].float()
        dz = torch.cat([dh * u * da, dh * a], 1)
        out["dx"] = (dz @ w.t()).to(dt)
        out["dw"] = (x.t() @ dz).to(dt)
        if c["bias"]:
            out["db"] = dz.sum(0)
    return out


def _plain_distill(s):
    c, v = s.case, s.v
    T, alpha, scale = c["temperature"], c["alpha"], _scale(c)
    x, idx = v["s"].float(), v["idx"].long()
    there = idx >= 0
    at = idx.clamp(min=0)
    some = there.any(1, keepdim=True).float()
    t = torch.where(there, v["t"] / T, torch.full_like(v["t"], -math.inf))
    tmax = torch.where(some > 0, t.max(1, keepdim=True).values, torch.zeros_like(some))
    e = torch.exp(t - tmax)
    total = e.sum(1, keepdim=True)
    p = torch.where(there, e / torch.where(some > 0, total, torch.ones_like(total)), torch.zeros_like(e))
    logp = torch.where(there, t - tmax - torch.log(torch.where(some > 0, total, torch.ones_like(total))),
                       torch.zeros_like(t))
    y = x / T
    ymax = y.max(1, keepdim=True).values
    ey = torch.exp(y - ymax)
    sy = ey.sum(1, keepdim=True)
    logq = y.gather(1, at) - ymax - torch.log(sy)
    loss = scale * alpha * T * T * (p * (logp - logq)).sum(1)
    if c["labels"]:
        lab = v["label"].long().unsqueeze(1)
        has = (lab >= 0).float()
        xmax = x.max(1, keepdim=True).values
        ex = torch.exp(x - xmax)
        sx = ex.sum(1, keepdim=True)
        ce = xmax + torch.log(sx) - x.gather(1, lab.clamp(min=0))
        loss = loss + scale * (1 - alpha) * (has * ce).squeeze(1)
    out = {"loss": loss}
    if c["train"]:
        ds = (scale * alpha * T) * some * (ey / sy)
        ds.scatter_add_(1, at, (-scale * alpha * T) * p)
        if c["labels"]:
            ds = ds + (scale * (1 - alpha)) * has * (ex / sx)
            ds.scatter_add_(1, lab.clamp(min=0), (-scale * (1 - alpha)) * has)
        out["ds"] = ds.to(TORCH[c["dtype"]])
    return out


def _pow2(e):
    """2^e in 32 bits for whole e in -127 .. 127."""
    return ((e.clamp(min=-126) + 127) << 23).view(torch.float32) * torch.where(e < -126, 0.5, 1.0)


def _mx4(v):
    """v [R, K] rounded to 4-bit values with a scale for each 32 along its rows, in 32 bits."""
    r, k = v.shape
    v = v.float()
    pad = -k % MX_BLOCK
    if pad:
        v = torch.cat([v, v.new_zeros(r, pad)], 1)
    b = v.reshape(r, -1, MX_BLOCK)
    top = b.abs().amax(2, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, torch.full_like(top, -127).int()).int().clamp(-127, 127)
    a = (b * _pow2(-e)).abs()
    q = 0.5 * ((a > 0.25).float() + (a >= 0.75).float() + (a > 1.25).float() + (a >= 1.75).float())
    q = q + (a > 2.5).float() + (a >= 3.5).float() + 2 * (a > 5).float()
    return (torch.copysign(q, b) * _pow2(e)).reshape(r, -1)[:, :k]


def _plain_mx4(s):
    return {"y": (_mx4(s.v["x"]) @ s.v["wq"]).to(TORCH[s.case["out"]])}


def _plain_mx4_keep(s):
    return {"w": _mx4(s.v["w"].t()).t().contiguous()}


_PLAIN = {"gated": _plain_gated, "distill": _plain_distill, "mx4": _plain_mx4, "mx4_keep": _plain_mx4_keep}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case) -> dict:
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    e = size[case["dtype"]]
    if kind == "gated":
        m, k, f = case["m"], case["k"], case["f"]
        fwd = 2 * (m * k + 2 * k * f + m * f) + (8 * f if case["bias"] else 0)
        if not case["train"]:
            return {"bytes": fwd, "flops": 4 * m * k * f}
        return {"bytes": fwd + 2 * (m * f + m * k + 2 * k * f) + (8 * f if case["bias"] else 0),
                "flops": 12 * m * k * f}
    if kind == "distill":
        n, v = case["n"], case["v"]
        return {"bytes": n * v * e * (2 if case["train"] else 1) + n * (8 * case["top"] + 8),
                "flops": n * v * (12 if case["train"] else 6)}
    k, n = case["k"], case["n"]
    if kind == "mx4":
        m = case["m"]
        return {"bytes": m * k * e + n * k * 17 // 32 + m * n * size[case["out"]], "flops": 2 * m * k * n}
    return {"bytes": k * n * (e + 4), "flops": 12 * k * n}


# ---------------------------------------------------------------- the same values in 64 bits

def _grid(v):
    """v [R, K] to the nearest of the 4-bit values (ties to the even code), the block's power of two taken out and put back."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=v.device)
    mid = (grid[1:] + grid[:-1]) / 2
    k = v.shape[1]
    full = torch.nn.functional.pad(v, (0, -k % MX_BLOCK)).unflatten(1, (-1, MX_BLOCK))
    top = full.abs().amax(2, keepdim=True)
    power = torch.where(top > 0, torch.frexp(top).exponent.long() - 1, torch.full_like(top, -127).long())
    unit = ((torch.clamp(power - 2, -127, 127) + 1023) << 52).view(torch.float64)
    a = (full / unit).abs()
    low, high = torch.bucketize(a, mid, right=False), torch.bucketize(a, mid, right=True)  # the two differ at a tie
    code = torch.where(low % 2 == 0, low, high)
    return (torch.sign(full) * grid[code] * unit).flatten(1)[:, :k]


def exact(case, seed):
    v = {k: t.double() for k, t in _inputs(case, seed).items()}
    kind = case["kind"]
    if kind == "gated":
        f = case["f"]
        z = v["x"] @ v["w"] + v.get("b", 0.0)
        g, u = z[:, :f].clone().requires_grad_(), z[:, f:].clone().requires_grad_()
        with torch.enable_grad():
            a = {"none": lambda q: q, "relu": torch.relu, "sigmoid": torch.sigmoid, "silu": lambda q: q * torch.sigmoid(q),
                 "gelu": lambda q: q * torch.special.ndtr(q)}[case["act"]](g)
            h = a * u
            if case["train"]:
                dg, du = torch.autograd.grad(h, (g, u), v["dh"])
        out = {"h": h.detach()}
        if case["train"]:
            out["dx"] = dg @ v["w"][:, :f].t().contiguous() + du @ v["w"][:, f:].t().contiguous()
            xt = v["x"].t().contiguous()
            out["dw"] = torch.cat([xt @ dg, xt @ du], 1)
            if case["bias"]:
                out["db"] = torch.cat([dg.sum(0), du.sum(0)])
        return out
    if kind == "distill":
        return _exact_distill(case, v)
    if kind == "mx4":
        return {"y": _grid(v["x"]) @ _grid(v["w"].t().contiguous()).t().contiguous()}
    return {"w": _grid(v["w"].t().contiguous()).t().contiguous()}


def _exact_distill(case, v):
    T, alpha, scale = case["temperature"], case["alpha"], _scale(case)
    n, vocab = v["s"].shape
    rows = torch.arange(n, device="cuda").unsqueeze(1)
    there = v["idx"] >= 0
    some = there.any(1)
    at = v["idx"].long()
    p = torch.zeros_like(v["t"])
    p[some] = torch.softmax((v["t"] / T).masked_fill(~there, -math.inf)[some], 1)
    logq = torch.log_softmax(v["s"] / T, 1)
    terms = torch.where(there, p * (torch.log(p.clamp(min=1e-300)) - logq[rows, at.clamp(min=0)]), torch.zeros_like(p))
    loss = alpha * T * T * terms.sum(1)
    if case["labels"]:
        lab = v["label"].long()
        has = torch.nonzero(lab >= 0).squeeze(1)
        logs = torch.log_softmax(v["s"], 1)
        loss[has] -= (1 - alpha) * logs[has, lab[has]]
    out = {"loss": scale * loss}
    if case["train"]:
        ds = logq.exp_().mul_(alpha * T) * some.double().unsqueeze(1)
        r, c = torch.nonzero(there, as_tuple=True)
        ds.index_put_((r, at[r, c]), -alpha * T * p[r, c], accumulate=True)
        if case["labels"]:
            ds[has] += (1 - alpha) * logs[has].exp()
            ds[has, lab[has]] -= 1 - alpha
        out["ds"] = ds.mul_(scale)
    return out
