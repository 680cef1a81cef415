"""Rows in microscaled 4-bit floating point, bit for bit, and the dense layer on
them against its definition in 64 bits.

Tolerances of the layer: products of codes are exact, so a sum of n of them in
32 bits is within n 2^-23 of the sum of their magnitudes; activations and the
rounding as for the dense layer, but GELU of 16-bit results, within 2^-17."""
import math

import numpy as np
import pytest

from chimera_amd import operators
from graph_replay import check_replays
from mx4_checks import LEVELS, quantise, without_signs_of_zeros
from operator_checks import BITS, Array, Matrix, activation, context, linear, to_type
from test_gpu_linear import forward_bounds

pytestmark = pytest.mark.gpu


def hard_values(rng, n, k, type):
    """Rows of all sizes with ties, zeros, one-value blocks and both ends of
    the type's range."""
    scale = 2.0 ** rng.integers(-130, 120, (n, -(-k // 32)))
    if type == "f16":
        scale = 2.0 ** rng.integers(-20, 10, scale.shape)
    x = rng.standard_normal((n, k)) * np.repeat(scale, 32, 1)[:, :k]
    ties = rng.random((n, k)) < 0.2
    x = np.where(ties, np.repeat(scale, 32, 1)[:, :k] * rng.choice(np.arange(-14, 15) / 4, (n, k)), x)
    x[rng.random((n, k)) < 0.05] = 0.0
    x[0] = 0.0
    if n > 3:
        x[1, : min(k, 32)] = 0.0
        x[2] = np.where(np.arange(k) % 32 == 5, -1.5, 0.0)
        x[3, 0] = 65504.0 if type == "f16" else 3.38e38
    return to_type(np.clip(x, -3.38e38, 3.38e38), type)


@pytest.mark.parametrize("n,k,type,pad,shift", [(1, 1, "f32", 0, 0), (4, 31, "f16", 3, 1), (7, 32, "bf16", 0, 0),
                                                (33, 257, "f32", 1, 0), (100, 777, "bf16", 5, 3), (64, 1024, "f16", 0, 0),
                                                (300, 4000, "f32", 0, 0), (2, 65536, "bf16", 0, 0), (40_001, 96, "bf16", 0, 0)])
def test_rows(n, k, type, pad, shift):
    rng = np.random.default_rng(n + k)
    print(f"{n} x {k} {type}", flush=True)
    x = hard_values(rng, n, k, type)
    codes, scales, values = quantise(x)
    ctx = context()
    row, blocks = operators.mx4_row(k)
    assert codes.shape == (n, row) and scales.shape == (n, blocks)
    d_x = Matrix(ctx, x, type, pad, shift)
    d_codes, d_scales = Array(ctx, np.full_like(codes, 0xEE)), Array(ctx, np.full_like(scales, 0xEE))
    operators.mx4_quantise(ctx, d_x, d_codes, d_scales)
    assert np.array_equal(d_scales.numpy(), scales)
    assert np.array_equal(without_signs_of_zeros(d_codes.numpy()), without_signs_of_zeros(codes))
    for out in ("f32", type):
        d_out = Matrix(ctx, None, out, pad, shift, shape=(n, k))
        operators.mx4_read(ctx, d_codes, d_scales, d_out)
        assert np.array_equal(d_out.values(), to_type(values, out))
        d_out.free()
    for v in (d_x, d_codes, d_scales):
        v.free()
    ctx.close()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_blocks_that_are_not_finite(type):
    """The block alone is lost, in either half of the padding's neighbours."""
    rng = np.random.default_rng(2)
    x = to_type(rng.standard_normal((6, 100)), type)
    x[0, 31], x[1, 32], x[2, 99], x[3, 0], x[3, 1] = np.nan, np.inf, -np.inf, np.nan, np.inf
    codes, scales, values = quantise(x)
    ctx = context()
    d = [Matrix(ctx, x, type), Array(ctx, np.zeros_like(codes)), Array(ctx, np.zeros_like(scales)),
         Matrix(ctx, None, type, shape=x.shape)]
    operators.mx4_quantise(ctx, *d[:3])
    operators.mx4_read(ctx, *d[1:])
    have = d[3].values()
    assert np.array_equal(d[2].numpy(), scales) and (scales == 255).sum() == 4
    assert np.array_equal(have, to_type(values, type), equal_nan=True)
    for v in d:
        v.free()
    ctx.close()


def test_every_code_and_scale_is_read_as_it_is_defined():
    ctx = context()
    scales = np.arange(256, dtype=np.uint8)
    codes = np.tile((np.arange(0, 16, 2) | np.arange(1, 17, 2) << 4).astype(np.uint8), (256, 2))
    wide = np.zeros((256, 8), np.uint8)
    wide[:, 0] = scales
    value = np.concatenate([LEVELS, -LEVELS])
    want = value[None] * np.exp2(scales.astype(np.float64) - 127)[:, None]
    want[255] = np.nan
    with np.errstate(over="ignore"):
        want = want.astype(np.float32)
    d = [Array(ctx, codes), Array(ctx, wide), Matrix(ctx, None, "f32", shape=(256, 32))]
    operators.mx4_read(ctx, *d)
    assert np.array_equal(d[2].values(), np.tile(want, (1, 2)).astype(np.float64), equal_nan=True)
    for v in d:
        v.free()
    ctx.close()


class Layer:
    def __init__(self, x, w, b, r, type, out, act, normalize, pad=0, shift=0, garbage=False):
        self.ctx = ctx = context()
        rows, k = x.shape
        codes, scales, self.w = quantise(w)
        if garbage:  # in the padding of the scales
            scales[:, -(-k // 32):] = 255
        self.x, self.b, self.r, self.out, self.act, self.normalize = quantise(x)[2], b, r, out, act, normalize
        self.d = {"codes": Array(ctx, codes), "scales": Array(ctx, scales), "x": Matrix(ctx, x, type, pad, shift),
                  "b": None if b is None else Matrix(ctx, b[None], type), "r": None if r is None else Matrix(ctx, r, type, pad, shift),
                  "y": Matrix(ctx, None, out, pad, shift, shape=(rows, w.shape[0]))}
        if b is not None:
            self.d["b"].shape = (w.shape[0],)
        self.layer = operators.Mx4Linear(ctx, self.d["codes"], self.d["scales"], k, self.d["b"], type=type, activation=act,
                                         normalize=normalize, max_rows=rows)

    def forward(self):
        self.layer.forward(self.d["x"], self.d["y"], residual=self.d["r"])

    def check(self):
        z, _, h, length, y = linear(self.x, self.w, self.b, self.r, self.act, self.normalize)
        _, _, ey = forward_bounds(self.x, self.w, self.b, h, length, y, self.out, self.normalize)
        if self.act == "gelu" and self.out != "f32":
            # 2^-17 of the activation's size, which a residual may take away; in a
            # row over its length, its own and y times the row's
            e = 2.0**-17 * np.abs(activation(z, "gelu")[0])
            ey = ey + ((e + np.abs(y) * np.sqrt((e * e).sum(1, keepdims=True))) / length if self.normalize else e)
        assert (np.abs(self.d["y"].values() - y) <= ey + (2.0**-25 if self.out == "f16" else 0.0)).all()
        self.d["x"].values()  # untouched around

    def close(self):
        self.layer.close()
        for v in self.d.values():
            if v is not None:
                v.free()
        self.ctx.close()


def make(rng, rows, k, n, type, bias, residual):
    size = np.exp(0.5 * rng.standard_normal(k))
    return (to_type(rng.standard_normal((rows, k)) * size, type), rng.standard_normal((n, k)) / np.sqrt(k),
            to_type(0.3 * rng.standard_normal(n), type) if bias else None,
            to_type(rng.standard_normal((rows, n)), type) if residual else None)


LAYERS = [
    # rows, k, n, type, out, act, bias, residual, normalize, pad, shift
    (1, 1, 1, "f32", "f32", "none", False, False, False, 0, 0),
    (1, 32, 16, "bf16", "bf16", "gelu", True, False, False, 0, 0),
    (1, 1024, 4096, "f16", "f16", "gelu", True, False, False, 0, 0),
    (2, 777, 130, "f16", "f16", "silu", True, True, False, 3, 1),
    (15, 4000, 33, "f32", "f32", "relu", False, True, False, 0, 0),
    (16, 256, 500, "bf16", "f32", "gelu_tanh", True, True, False, 8, 8),
    (17, 288, 128, "bf16", "bf16", "none", True, False, False, 0, 0),
    (1, 768, 128, "bf16", "f32", "none", False, False, True, 0, 0),
    (32, 768, 128, "bf16", "f32", "none", False, False, True, 0, 0),
    (33, 100, 96, "f32", "f32", "gelu", True, True, True, 4, 1),
    (17, 64, 1, "f16", "f32", "relu", True, False, True, 0, 0),
    (500, 1000, 48, "bf16", "bf16", "gelu_tanh", True, True, True, 1, 0),
    (9000, 160, 127, "f16", "f16", "silu", True, False, True, 0, 0),
    (65, 33, 5, "f16", "f16", "none", True, False, False, 1, 1),
    (300, 1056, 700, "bf16", "bf16", "silu", True, True, False, 5, 0),
    (2049, 511, 2050, "f32", "f32", "gelu", True, True, False, 0, 0),
    (4097, 513, 4099, "f16", "f16", "gelu", True, True, False, 3, 0),
    (4100, 2080, 512, "bf16", "f32", "none", False, False, False, 0, 0),
]


@pytest.mark.parametrize("rows,k,n,type,out,act,bias,residual,normalize,pad,shift", LAYERS)
def test_layer(rows, k, n, type, out, act, bias, residual, normalize, pad, shift):
    rng = np.random.default_rng(rows * 7 + k * 3 + n)
    print(f"{rows} x {k} -> {n} {type}", flush=True)
    layer = Layer(*make(rng, rows, k, n, type, bias, residual), type, out, act, normalize, pad, shift, garbage=True)
    layer.forward()
    layer.check()
    layer.close()


WHOLE = [(3, 1024, 333, "bf16"), (16, 3000, 17, "f16"), (40, 640, 200, "f32"), (1000, 777, 650, "bf16"), (3100, 456, 1720, "f16"),
         (5000, 2600, 1100, "bf16"), (70, 9000, 130, "f32")]


@pytest.mark.parametrize("rows,k,n,type", WHOLE)
def test_sums_of_whole_numbers(rows, k, n, type):
    """Codes of 0, 1, 2 and 4 in 32 bits: sums are exact, a wrong element shows."""
    rng = np.random.default_rng(rows + k)
    print(f"{rows} x {k} -> {n} {type}", flush=True)
    x, w = (rng.choice([0.0, 1.0, -1.0, 2.0, -4.0], s) for s in ((rows, k), (n, k)))
    b, r = rng.integers(-3, 4, n).astype(float), rng.integers(-3, 4, (rows, n)).astype(float)
    layer = Layer(x, w, b, r, type, "f32", "none", False)
    layer.forward()
    assert np.array_equal(layer.x, x) and np.array_equal(layer.w, w)
    assert np.array_equal(layer.d["y"].values(), x @ w.T + b + r)
    layer.close()


@pytest.mark.parametrize("rows,normalize", [(3, False), (8, True), (200, False), (200, True), (5000, True)])
def test_values_that_are_not_finite_stay_apart(rows, normalize):
    """A row of X reaches its row of Y, a row of W its column."""
    rng = np.random.default_rng(rows)
    x, w, _, _ = make(rng, rows, 300, 96, "bf16", False, False)
    x[1, 299] = np.nan
    w[7, 0] = np.inf
    layer = Layer(x, w, None, None, "bf16", "f32", "none", normalize)
    layer.forward()
    y = layer.d["y"].values()
    lost = np.zeros(y.shape, bool)
    lost[1] = True
    if normalize:
        lost[:] = True  # each row has a column that is NaN
    else:
        lost[:, 7] = True
    assert np.array_equal(np.isnan(y), lost)
    layer.close()


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("n", [20_000, 45_000])
def test_gelu_of_all_biases(n, type):
    """GELU of 16-bit results, over values from -6 on: rows of zeros leave the
    bias. Within 2^-17 of its size and half a step of the type, on few columns
    and on many; past -6 below 1e-8."""
    b = np.arange(1 << 16, dtype=np.uint16)
    with np.errstate(invalid="ignore"):
        b = (b.view(np.float16) if type == "f16" else (b.astype(np.uint32) << 16).view(np.float32)).astype(np.float64)
    b = np.sort(b[np.isfinite(b) & (b >= -3e4) & (np.abs(b) >= 2.0**-14)])
    b = b[:: max(1, -(-b.size // n))]
    b = np.concatenate([b, np.ones(n - b.size)])
    want = np.array([z * 0.5 * math.erfc(-z / math.sqrt(2)) for z in b])
    x, w = np.zeros((1, 32)), np.ones((n, 32))
    layer = Layer(x, w, b, None, type, type, "gelu", False)
    layer.forward()
    off = np.abs(layer.d["y"].values()[0] - want)
    bound = (2.0**-17 + 2.0**-BITS[type]) * np.abs(want) + (2.0**-25 if type == "f16" else 0)
    assert (off <= np.where(b >= -6, bound, 1e-8 + bound)).all()
    layer.close()


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [2, 900])
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu"])
def test_activations_of_sums_that_are_not_finite(rows, type, act):
    """Biases of NaN and both infinities: NaN stays, infinity too, and minus
    infinity gives zero or NaN (0 times it)."""
    b = np.array([np.nan, np.inf, -np.inf, 1.0] * 200)
    layer = Layer(np.zeros((rows, 40)), np.ones((800, 40)), b, None, type, type, act, False)
    layer.forward()
    y = layer.d["y"].values().reshape(rows, 200, 4)
    assert np.isnan(y[..., 0]).all() and np.isfinite(y[..., 3]).all()
    if act != "gelu_tanh":  # inf / inf in its argument's cube stays NaN or infinite
        assert (y[..., 1] == np.inf).all()
    assert (np.isnan(y[..., 2]) | (y[..., 2] == 0)).all()
    layer.close()


def test_graph_and_fewer_rows():
    rng = np.random.default_rng(5)
    x, w, b, _ = make(rng, 700, 520, 260, "bf16", True, False)
    layer = Layer(x, w, b, None, "bf16", "bf16", "silu", False)

    def few():  # on the same object
        for rows in (1, 20, 700):
            layer.d["x"].shape, layer.d["y"].shape = (rows, 520), (rows, 260)
            layer.forward()

    check_replays(layer.ctx, layer.forward, lambda: [layer.d["y"].values()], between=few)
    layer.check()
    with pytest.raises(Exception, match="workspace"):
        layer.d["x"].shape, layer.d["y"].shape = (7000, 520), (7000, 260)
        layer.forward()
    layer.d["x"].shape, layer.d["y"].shape = (0, 520), (0, 260)
    layer.forward()
    layer.d["x"].shape, layer.d["y"].shape = (700, 520), (700, 260)
    layer.close()
