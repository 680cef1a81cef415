"""GELU's own error, on layers whose sums are the weights themselves.

Tolerances. The function of a 16-bit result is within 2^-18 of its size to -6,
so that the result is within that of the nearest 16-bit value. A 32-bit result
is within 2^-20 of its size down to -12.9, where it falls out of the normal
numbers, and a slope within 2^-20 of the sizes of its two terms."""
import math

import numpy as np
import pytest

from operator_checks import BITS, Matrix, context, linear, to_type
from test_gpu_linear import release, run_forward

pytestmark = pytest.mark.gpu


def gelu(z, type, out, rows):
    ctx = context()
    layer, d = run_forward(ctx, np.ones((rows, 1)), z[:, None], None, None, type, out, "gelu", False)
    have = d["y"].values()[-1]
    release(ctx, layer, d)
    ctx.close()
    return have, linear(np.ones((1, 1)), z[:, None], None, None, "gelu", False)[4][0]


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_results_of_16_bits_are_rounded_once(type, rows):
    z = np.unique(to_type(np.linspace(-6, 8, 20001), type))
    have, want = gelu(z, type, type, rows)
    size = np.abs(want)
    least = 2.0**-25 if type == "f16" else 0.0
    assert (np.abs(have - want) <= (2.0**-BITS[type] + 2.0**-18) * size + least).all()


_upper = np.vectorize(lambda z: 0.5 * math.erfc(-z / math.sqrt(2)), otypes=[np.float64])  # no difference below zero


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_results_of_32_bits_keep_their_digits(type, rows):
    z = np.unique(to_type(np.linspace(-12.9, 12.9, 20001), type))
    have, _ = gelu(z, type, "f32", rows)
    want = z * _upper(z)
    assert (np.abs(have - want) <= 2.0**-20 * np.abs(want)).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_errors_over_normal_arguments(rows):
    """The error's size over a layer's usual sums: two roundings (the function
    and its product with z) of at most 2^-24 each, so 2^-24 over the mean
    square with room to spare, of which rounding alone is about half."""
    z = to_type(np.random.default_rng(2).standard_normal(60_000), "f32")
    have, _ = gelu(z, "f32", "f32", rows)
    want = z * _upper(z)
    assert np.linalg.norm(have - want) <= 2.0**-24 * np.linalg.norm(want)


def test_slopes_keep_their_digits():
    z = np.unique(to_type(np.linspace(-12.9, 12.9, 20001), "f32"))[None]
    ctx = context()
    layer, d = run_forward(ctx, np.ones((1, 1)), z.T, None, None, "f32", "f32", "gelu", False, training=True)
    dy, dw = Matrix(ctx, np.ones(z.shape), "f32"), Matrix(ctx, None, "f32", shape=(z.size, 1))
    layer.backward(d["x"], dy, saved=d["saved"], dweight=dw)  # dW = dZ: the slopes
    cdf, rest = _upper(z[0]), z[0] * np.exp(-z[0] ** 2 / 2) / math.sqrt(2 * math.pi)
    assert (np.abs(dw.values()[:, 0] - (cdf + rest)) <= 2.0**-20 * (cdf + np.abs(rest))).all()
    release(ctx, layer, {**d, "dy": dy, "dw": dw})
    ctx.close()
