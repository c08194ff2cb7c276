"""Device tensors of a test and their values in 64 bits."""
from __future__ import annotations

import ctypes as C

import numpy as np

from picograd_amd.capi import BF16, F16, F32, shape_arg

# half a unit in the last place, relative
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}  # half the smallest subnormal
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}


def to_bits(a, dtype) -> np.ndarray:
    """a as f32, or as the bits of a 16-bit dtype (rounded to nearest even)."""
    a = np.asarray(a, np.float32)
    if dtype == F32:
        return a
    if dtype == F16:
        with np.errstate(over="ignore"):
            return a.astype(np.float16).view(np.uint16)
    u = np.atleast_1d(a).view(np.uint32)
    near = ((u + np.uint32(0x7FFF) + ((u >> 16) & np.uint32(1))) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), near.reshape(a.shape))


def from_bits(bits, dtype) -> np.ndarray:
    """The values in 64 bits."""
    if dtype == F32:
        return np.asarray(bits, np.float32).astype(np.float64)
    if dtype == F16:
        return np.asarray(bits).view(np.float16).astype(np.float64)
    return (np.asarray(bits).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def rounded(a, dtype) -> np.ndarray:
    """a's values rounded to dtype, in 64 bits."""
    return from_bits(to_bits(a, dtype), dtype)


class Bench:
    """Tensors and nodes that a test makes, freed at its end."""

    def __init__(self, lib):
        self.L, self.frees = lib, []
        for name, res, args in (("pg_tensor_permute_view", C.c_void_p, [C.c_void_p, C.POINTER(C.c_size_t)]),
                                ("pg_tensor_reshape_view", C.c_void_p,
                                 [C.c_void_p, C.c_size_t, C.POINTER(C.c_size_t)])):
            fn = getattr(lib.lib, name)
            fn.restype, fn.argtypes = res, args
            setattr(self, name, fn)

    def tensor(self, a, dtype=F32) -> int:
        t = self.L.tensor(to_bits(a, dtype), dtype)
        self.frees.append((self.L.pg_tensor_free, t))
        return t

    def transposed(self, a, dtype=F32) -> int:
        """A strided view with a's values."""
        base = self.tensor(np.ascontiguousarray(np.asarray(a).T), dtype)
        v = self.pg_tensor_permute_view(base, (C.c_size_t * 2)(1, 0))
        assert v
        self.frees.append((self.L.pg_tensor_free, v))
        return v

    def unset(self, shape, dtype=F32) -> int:
        """An output, full of a value that no test expects."""
        nd, sh = shape_arg(shape)
        t = self.L.pg_tensor_full_dtype(dtype, nd, sh, 777.0)
        assert t
        self.frees.append((self.L.pg_tensor_free, t))
        return t

    def var(self, a, requires_grad=True) -> int:
        n = self.L.var(np.asarray(a, np.float32), requires_grad)
        self.frees.append((self.L.pg_node_free, n))
        return n

    def node(self, n) -> int:
        assert n, self.L.pg_autograd_last_error().decode()
        self.frees.append((self.L.pg_node_free, n))
        return n

    def read(self, t) -> np.ndarray:
        return from_bits(self.L.read(t), self.L.tinfo(t).dtype)

    def ok(self, done):
        assert done, self.L.pg_autograd_last_error().decode() or self.L.pg_amd_last_error().decode()

    def refused(self, done, word):
        assert not done
        assert word in self.L.pg_autograd_last_error().decode()

    def close(self):
        self.L.sync()
        for f, p in reversed(self.frees):
            f(p)


def within(got, want, bound, what=""):
    """|got - want| <= bound, element for element; NaN and infinities where they are wanted."""
    got, want, bound = (np.asarray(v, np.float64) for v in (got, want, bound))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), what
    off = np.abs(got - want)[fine]
    lim = np.broadcast_to(bound, want.shape)[fine]
    assert (off <= lim).all(), f"{what}: off by {np.max(off / np.maximum(lim, 1e-300)):.3g} times the bound"
