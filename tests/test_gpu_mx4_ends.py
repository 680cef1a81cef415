"""The 4-bit layer's results in its own type: GELU and the 16-bit stores of every
walk and tile, without a residual (whose loads make a wave wait for the next
tile's) and with one, in blocks that walk several tiles.

A row of Y is its row of X's alone, so X is the same 331 rows over and over, which
no tile's are a multiple of, and every row has its known result. Tolerances as in
test_gpu_mx4."""
import math

import numpy as np
import pytest

from chimera_amd import operators
from dense_stack_shapes import MX4_LAYERS
from operator_checks import Matrix, activation, linear
from test_gpu_linear import forward_bounds
from test_gpu_mx4 import Layer, make

pytestmark = pytest.mark.gpu

PERIOD = 331
SHAPES = [(rows, k, n, type if type != "f32" else "bf16", 0) for rows, k, n, type, normalize, kernel in MX4_LAYERS
          if kernel[0] in ("walk", "tile")] + [(33_000, 300, 1000, "bf16", 5), (1_000, 300, 520, "f16", 1)]


@pytest.mark.parametrize("rows,k,n,type,pad", SHAPES)
@pytest.mark.parametrize("residual", [False, True])
def test_layers_in_their_own_type(rows, k, n, type, pad, residual):
    rng = np.random.default_rng(rows + k + n + residual)
    print(f"{rows} x {k} -> {n} {type}", flush=True)
    x, w, b, r = make(rng, PERIOD, k, n, type, True, residual)
    few = Layer(x, w, b, r, type, type, "gelu", False, garbage=True)
    z, _, h, length, y = linear(few.x, few.w, b, r, "gelu", False)
    _, _, ey = forward_bounds(few.x, few.w, b, h, length, y, type, False)
    ey += 2.0**-17 * np.abs(activation(z, "gelu")[0]) + (2.0**-25 if type == "f16" else 0.0)
    repeated = lambda v: np.resize(v, (rows, v.shape[1]))
    d_x, d_y = Matrix(few.ctx, repeated(x), type, pad, pad), Matrix(few.ctx, None, type, pad, pad, shape=(rows, n))
    d_r = Matrix(few.ctx, repeated(r), type, pad, pad) if residual else None
    layer = operators.Mx4Linear(few.ctx, few.d["codes"], few.d["scales"], k, few.d["b"], type=type, activation="gelu", max_rows=rows)
    layer.forward(d_x, d_y, residual=d_r)
    have, first = d_y.values(), d_y.buffer.numpy()
    for at in range(0, rows, PERIOD):
        part = have[at:at + PERIOD]
        assert (np.abs(part - y[: len(part)]) <= ey[: len(part)]).all(), at
    for _ in range(3):
        layer.forward(d_x, d_y, residual=d_r)
        assert np.array_equal(d_y.buffer.numpy(), first)
    layer.close()
    for v in (d_x, d_y, d_r):
        if v is not None:
            v.free()
    few.close()


@pytest.mark.parametrize("rows,k,n", [(1, 32, 400), (1000, 200, 800), (8200, 256, 4090), (500, 2100, 600), (2100, 2500, 2000)])
def test_gelu_far_below_zero(rows, k, n):
    """bf16 holds GELU down to -12.9, where the normal distribution's tail is no
    normal 32-bit number any more: of all biases from there to -6, in the kernels
    of few rows, of walks and of tiles. Rows of zeros leave the bias."""
    b = np.arange(0xC0C0, 0xC14F, dtype=np.uint32)  # -6 to -12.875
    b = np.resize((b << 16).view(np.float32).astype(np.float64), n)
    want = b * np.array([0.5 * math.erfc(-z / math.sqrt(2)) for z in b])
    few = Layer(np.zeros((1, k)), np.ones((n, k)), b, None, "bf16", "bf16", "gelu", False)
    d_x, d_y = Matrix(few.ctx, np.zeros((rows, k)), "bf16"), Matrix(few.ctx, None, "bf16", shape=(rows, n))
    layer = operators.Mx4Linear(few.ctx, few.d["codes"], few.d["scales"], k, few.d["b"], type="bf16", activation="gelu", max_rows=rows)
    layer.forward(d_x, d_y)
    assert (np.abs(d_y.values() - want) <= (2.0**-12 + 2.0**-8) * np.abs(want)).all()
    layer.close()
    d_x.free()
    d_y.free()
    few.close()
