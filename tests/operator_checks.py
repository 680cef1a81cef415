"""Helpers of the operator tests: 16-bit types in numpy, matrices with rows
apart from each other on the device, guarded outputs, and the operators'
definitions in 64 bits."""
import math

import numpy as np

from chimera_amd import capi

BITS = {"f32": 24, "f16": 11, "bf16": 8}  # significant bits


def to_type(x, name):
    """x rounded to the type (nearest even), as float64 values."""
    x = np.asarray(x, np.float32)
    if name == "f16":
        return x.astype(np.float16).astype(np.float64)
    if name == "bf16":
        return from_bf16(bf16_bits(x)).astype(np.float64)
    return x.astype(np.float64)


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def raw(x, name):
    """The array a device matrix of the type holds."""
    x = np.asarray(x, np.float32)
    return x if name == "f32" else x.astype(np.float16) if name == "f16" else bf16_bits(x)


class Matrix:
    """A device matrix [rows, cols] of a type with `pad` elements between rows
    and `shift` before the first; the elements outside it hold a pattern."""

    def __init__(self, ctx, x, name, pad=0, shift=0, shape=None):
        self.ctx, self.dtype = ctx, name
        self.shape = tuple(shape) if shape is not None else np.shape(x)
        cols = self.shape[-1]
        rows = int(np.prod(self.shape[:-1], dtype=np.int64))
        self.stride = cols + pad if len(self.shape) == 2 else None
        wide = cols + pad
        item = 4 if name == "f32" else 2
        word = np.uint32 if item == 4 else np.uint16
        self.at = shift + np.arange(rows)[:, None] * wide + np.arange(cols)
        self.host = np.full(shift + rows * wide + 64, 0x7FC17FC1 if item == 4 else 0x7FC1, word)
        if x is not None:
            self.host[self.at] = raw(x, name).reshape(rows, cols).view(word)
        self.buffer = ctx.to_device(self.host)
        self.ptr = self.buffer.ptr + shift * item

    def values(self):
        """The matrix as float64; fails if anything around it changed."""
        now = self.buffer.numpy()
        inside = np.zeros(now.size, bool)
        inside[self.at] = True
        assert np.array_equal(now[~inside], self.host[~inside]), "written outside the matrix"
        v = now[self.at]
        v = v.view(np.float32) if self.dtype == "f32" else v.view(np.float16) if self.dtype == "f16" else from_bf16(v)
        return v.astype(np.float64).reshape(self.shape)

    def free(self):
        self.buffer.free()


class Array:
    """A device array of any numpy type."""

    def __init__(self, ctx, x):
        self.buffer = ctx.to_device(np.ascontiguousarray(x))
        self.ptr, self.shape, self.dtype = self.buffer.ptr, self.buffer.shape, self.buffer.dtype

    def numpy(self):
        return self.buffer.numpy()

    def free(self):
        self.buffer.free()


def context():
    return capi.Context(None, 1, 1, 1, 1)


_erf = np.vectorize(math.erf, otypes=[np.float64])


def activation(z, act):
    """act(z) and act'(z) in 64 bits."""
    if act == "relu":
        return np.where(z > 0, z, 0.0), (z > 0).astype(np.float64)
    if act == "gelu":
        cdf = 0.5 * (1 + _erf(z / math.sqrt(2)))
        return z * cdf, cdf + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        s = 1 / (1 + np.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    return z, np.ones_like(z)


def linear(x, w, b, r, act, normalize):
    """z, act'(z), h, norms and y in 64 bits."""
    z = x @ w.T + (0.0 if b is None else b)
    h, slope = activation(z, act)
    h = h + (0.0 if r is None else r)
    norm = np.maximum(np.sqrt((h * h).sum(1, keepdims=True)), 1e-12)
    return z, slope, h, norm, h / norm if normalize else h


def linear_gradients(x, w, dy, y, slope, norm, normalize):
    dh = (dy - y * (y * dy).sum(1, keepdims=True)) / norm if normalize else dy
    dz = dh * slope
    return dh, dz, dz @ w, dz.T @ x, dz.sum(0)
