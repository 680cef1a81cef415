"""Layers whose sums come near the ends of the 32-bit range."""
import numpy as np
import pytest

from operator_checks import BITS, Matrix, context, to_type
from test_gpu_linear import release, run_forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [1, 40])
def test_activations_of_large_sums(type, act, rows):
    """Far from zero each activation is its argument or zero, its slope one or
    zero: exactly, as what is left is far below a last place."""
    z = to_type(np.array([[1e3, 1e6, 1e13, 1e19, 1e20, 1e30, 3e38]]), type)
    z = np.concatenate([z, -z], 1)
    ctx = context()
    layer, d = run_forward(ctx, np.ones((rows, 1)), z.T, None, None, type, type, act, False, training=True)
    assert np.array_equal(np.abs(d["y"].values()), np.tile(np.maximum(z, 0), (rows, 1)))
    dy = np.zeros((rows, z.size))
    dy[-1] = 1
    g = {"dy": Matrix(ctx, dy, type), "dw": Matrix(ctx, None, type, shape=(z.size, 1))}
    layer.backward(d["x"], g["dy"], saved=d["saved"], dweight=g["dw"])  # the last row's slopes
    assert np.array_equal(np.abs(g["dw"].values()[:, 0]), (z[0] > 0).astype(float))
    release(ctx, layer, {**d, **g})
    ctx.close()


@pytest.mark.parametrize("type,k,n,rows", [("f32", 8, 128, 40), ("f32", 8, 70, 5), ("f32", 8, 40, 70), ("bf16", 8, 128, 24_600),
                                           ("bf16", 8, 100, 300)])
def test_rows_of_any_length(type, k, n, rows):
    """Rows of length one from sums near 1e-10 to 1e38, whose squares leave
    32 bits; the lengths, and the gradient of the residual, come with them.
    The sums are the inputs' products with whole numbers: k roundings of 2^-24
    of terms that are at most 8 times the sum's size here, the length's and the
    division's of 2^-23 each."""
    rng = np.random.default_rng(n + rows)
    size = np.exp(rng.uniform(np.log(1e-9), np.log(1e36), rows))
    size[:4] = 3e36, 1e19, 2e19, 1e-8
    x = to_type(rng.integers(1, 9, (rows, k)) * size[:, None], type)
    w = rng.integers(1, 5, (n, k)).astype(np.float64)
    ctx = context()
    layer, d = run_forward(ctx, x, w, None, None, type, "f32", "none", True, training=True)
    h = x @ w.T
    norm = np.sqrt(np.square(h / size[:, None]).sum(1)) * size
    y = h / norm[:, None]
    off = (k + 8) * 2.0**-23
    fits = (np.abs(x) @ np.abs(w).T).max(1) < 3.4e38  # a sum past the 32-bit range is infinite
    assert fits[1:].sum() > rows // 2 and not np.isnan(d["y"].values()[fits]).any()
    assert (np.abs(d["y"].values() - y) <= off * np.abs(y))[fits].all()
    representable = fits & (norm < 3.4e38)
    assert (np.abs(d["norms"].values() / norm - 1)[representable] <= off).all()
    dy = rng.standard_normal((rows, n))
    g = {"dy": Matrix(ctx, dy, "f32"), "dr": Matrix(ctx, None, type, shape=(rows, n))}
    layer.backward(d["x"], g["dy"], y=d["y"], norms=d["norms"], dresidual=g["dr"])
    dy = g["dy"].values()
    want = (dy - y * (y * dy).sum(1, keepdims=True)) / norm[:, None]
    terms = (np.abs(dy) + np.abs(y) * np.abs(y * dy).sum(1, keepdims=True)) / norm[:, None]
    bound = (3 * off + n * 2.0**-23) * terms + 2.0**-BITS[type] * np.abs(want) + 2.0**-126
    assert (np.abs(g["dr"].values() - want) <= bound)[representable].all()
    release(ctx, layer, {**d, **g})
    ctx.close()
