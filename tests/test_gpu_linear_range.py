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
