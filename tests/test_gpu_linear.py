"""Dense layers against their definition in 64 bits.

Tolerances. A sum of n products in 32 bits is within n 2^-23 of the sum of
their magnitudes (twice the bound of rounding each step to nearest, for the
matrix cores' own rounding). The activations used here change by at most 1.13
times their argument's change and their slopes by at most 0.85 times; the
functions themselves are within 2^-20 of (1 + |z|). Rounding to a type of p
bits adds 2^-p of the value."""
import numpy as np
import pytest

from chimera_amd import operators
from operator_checks import BITS, Array, Matrix, context, linear, linear_gradients, to_type

pytestmark = pytest.mark.gpu


def make(rng, rows, k, n, type, bias, residual):
    x = to_type(rng.standard_normal((rows, k)), type)
    w = to_type(rng.standard_normal((n, k)) / np.sqrt(k), type)
    b = to_type(0.3 * rng.standard_normal(n), type) if bias else None
    r = to_type(rng.standard_normal((rows, n)), type) if residual else None
    return x, w, b, r


def forward_bounds(x, w, b, h, norm, y, out, normalize):
    """How far Z, H and Y may be off."""
    k = x.shape[1]
    ez = (k + 4) * 2.0**-23 * (np.abs(x) @ np.abs(w).T + (0.0 if b is None else np.abs(b)))
    eh = 1.13 * ez + 2.0**-20 * (1 + np.abs(h))
    ey = eh
    if normalize:
        en = np.sqrt((eh * eh).sum(1, keepdims=True))
        ey = (eh + np.abs(y) * en) / norm + 2.0**-20 * np.abs(y)
    return ez, eh, ey + 2.0**-BITS[out] * np.abs(y)


def run_forward(ctx, x, w, b, r, type, out, act, normalize, pads=(0, 0, 0), shift=0, training=False):
    rows, n = x.shape[0], w.shape[0]
    d = {"x": Matrix(ctx, x, type, pads[0], shift), "w": Matrix(ctx, w, type, pads[1], shift),
         "b": None if b is None else Matrix(ctx, b[None], type), "r": None if r is None else Matrix(ctx, r, type, pads[2], shift),
         "y": Matrix(ctx, None, out, pads[2], shift, shape=(rows, n))}
    if b is not None:
        d["b"].shape = (n,)
    if training:
        d["saved"] = Matrix(ctx, None, type, pads[2], shift, shape=(rows, n)) if act != "none" else None
        d["norms"] = Matrix(ctx, None, "f32", shape=(1, rows)) if normalize else None
        if normalize:
            d["norms"].shape = (rows,)
    layer = operators.Linear(ctx, d["w"], d["b"], activation=act, normalize=normalize, max_rows=rows, training=training)
    layer.forward(d["x"], d["y"], residual=d["r"], saved=d.get("saved"), norms=d.get("norms"))
    return layer, d


def release(ctx, layer, d):
    layer.close()
    for v in d.values():
        if v is not None:
            v.free()


FORWARD = [
    # rows, k, n, type, out, act, bias, residual, normalize, pads, shift
    (1, 1, 1, "f32", "f32", "none", False, False, False, (0, 0, 0), 0),
    (1, 8, 16, "bf16", "bf16", "gelu", True, False, False, (0, 0, 0), 0),
    (1, 777, 130, "f16", "f16", "silu", True, True, False, (0, 0, 0), 0),
    (32, 768, 128, "bf16", "f32", "none", False, False, True, (0, 0, 0), 0),
    (33, 100, 96, "f32", "f32", "gelu", True, True, True, (4, 4, 0), 0),
    (17, 64, 1, "f16", "f32", "relu", True, False, True, (0, 0, 0), 0),
    (64, 40, 48, "bf16", "bf16", "gelu_tanh", False, True, False, (8, 8, 8), 0),
    (65, 64, 48, "bf16", "bf16", "gelu_tanh", True, True, False, (8, 8, 8), 8),
    (65, 33, 5, "f16", "f16", "none", True, False, False, (0, 3, 1), 1),
    (129, 72, 128, "bf16", "f32", "silu", True, True, True, (0, 0, 0), 0),
    (300, 321, 127, "f32", "f32", "gelu_tanh", True, True, True, (3, 1, 2), 1),
    (257, 129, 129, "f32", "f32", "silu", True, False, False, (0, 0, 0), 0),
    (500, 256, 640, "f16", "f32", "gelu", True, True, False, (8, 0, 4), 0),
    (4100, 96, 4128, "bf16", "bf16", "none", True, False, False, (0, 0, 0), 0),
    (4097, 520, 4099, "f16", "f16", "gelu", True, True, False, (0, 0, 5), 0),
    (2049, 40, 2050, "f32", "f32", "none", False, False, False, (0, 4, 0), 0),
    (8200, 130, 100, "bf16", "bf16", "none", True, False, True, (0, 0, 0), 0),
]


@pytest.mark.parametrize("rows,k,n,type,out,act,bias,residual,normalize,pads,shift", FORWARD)
def test_forward(rows, k, n, type, out, act, bias, residual, normalize, pads, shift):
    rng = np.random.default_rng(rows * 7 + k * 3 + n)
    x, w, b, r = make(rng, rows, k, n, type, bias, residual)
    print(f"{rows} x {k} -> {n} {type}", flush=True)
    ctx = context()
    layer, d = run_forward(ctx, x, w, b, r, type, out, act, normalize, pads, shift, training=True)
    z, _, h, norm, y = linear(x, w, b, r, act, normalize)
    ez, _, ey = forward_bounds(x, w, b, h, norm, y, out, normalize)
    assert (np.abs(d["y"].values() - y) <= ey).all()
    if d["saved"] is not None:
        assert (np.abs(d["saved"].values() - z) <= ez + 2.0**-BITS[type] * np.abs(z)).all()
    for name in ("x", "w"):
        d[name].values()  # untouched around
    release(ctx, layer, d)
    ctx.close()


BACKWARD = [
    (1, 8, 16, "f32", "f32", "gelu", False, True, True, False),
    (3, 20, 5, "bf16", "bf16", "silu", True, False, False, False),
    (70, 64, 128, "bf16", "f32", "none", True, False, True, True),
    (129, 65, 96, "f32", "f32", "none", True, True, True, True),
    (200, 130, 100, "f16", "f16", "gelu_tanh", True, True, True, True),
    (513, 136, 264, "bf16", "bf16", "gelu", True, True, False, False),
    (1100, 72, 40, "f16", "f32", "silu", True, False, False, False),
    (2000, 33, 129, "f32", "f32", "silu", True, False, False, False),
    (5000, 48, 64, "bf16", "bf16", "none", True, True, False, False),
    (700, 1030, 2050, "bf16", "bf16", "gelu", True, False, False, False),
]


@pytest.mark.parametrize("rows,k,n,type,out,act,bias,residual,normalize,want_dr", BACKWARD)
def test_backward(rows, k, n, type, out, act, bias, residual, normalize, want_dr):
    rng = np.random.default_rng(rows + k + n)
    x, w, b, r = make(rng, rows, k, n, type, bias, residual)
    dy = to_type(rng.standard_normal((rows, n)), out)
    print(f"{rows} x {k} -> {n} {type}", flush=True)
    ctx = context()
    layer, d = run_forward(ctx, x, w, b, r, type, out, act, normalize, training=True)
    g = {"dy": Matrix(ctx, dy, out, 3, 1), "dx": Matrix(ctx, None, type, 5, 1, shape=(rows, k)),
         "dw": Matrix(ctx, None, type, 1, 0, shape=(n, k)), "db": Matrix(ctx, None, type, shape=(1, n)),
         "dr": Matrix(ctx, None, type, 8, 0, shape=(rows, n)) if want_dr else None}
    g["db"].shape = (n,)
    layer.backward(d["x"], g["dy"], saved=d["saved"], y=d["y"], norms=d["norms"], dx=g["dx"], dweight=g["dw"],
                   dbias=g["db"], dresidual=g["dr"])
    z, slope, h, norm, y = linear(x, w, b, r, act, normalize)
    ez, eh, ey = forward_bounds(x, w, b, h, norm, y, out, normalize)
    dh, dz, dx, dw, db = linear_gradients(x, w, dy, y, slope, norm, normalize)
    u = 2.0**-BITS[type]
    edh = 2.0**-21 * np.abs(dy)
    if normalize:
        dot = np.abs(y * dy).sum(1, keepdims=True)
        edot = (ey * np.abs(dy)).sum(1, keepdims=True) + (n + 4) * 2.0**-23 * dot
        en = np.sqrt((eh * eh).sum(1, keepdims=True)) / norm
        edh = (ey * dot + np.abs(y) * edot + 2.0**-21 * np.abs(dy)) / norm + np.abs(dh) * (en + 2.0**-20)
    # the saved sums are rounded to the type
    edz = edh * 1.13 + np.abs(dh) * (0.85 * (u * np.abs(z) + ez) + 2.0**-20 if act != "none" else 0.0)
    if want_dr:
        assert (np.abs(g["dr"].values() - dh) <= edh + u * np.abs(dh)).all()
    total = np.abs(dz) + edz
    assert (np.abs(g["db"].values() - db) <= edz.sum(0) + (rows + 4) * 2.0**-23 * total.sum(0) + u * np.abs(db)).all()
    edz = edz + u * total  # the products' operand
    edx = edz @ np.abs(w) + (n + 4) * 2.0**-23 * ((total + edz) @ np.abs(w))
    assert (np.abs(g["dx"].values() - dx) <= edx + u * np.abs(dx)).all()
    edw = edz.T @ np.abs(x) + (rows + 4) * 2.0**-23 * ((total + edz).T @ np.abs(x))
    assert (np.abs(g["dw"].values() - dw) <= edw + u * np.abs(dw)).all()
    # one gradient at a time, and the same sums again
    first = {name: v.values() for name, v in g.items() if v is not None}
    for name, key in (("dx", "dx"), ("dweight", "dw"), ("dbias", "db")):
        layer.backward(d["x"], g["dy"], saved=d["saved"], y=d["y"], norms=d["norms"], **{name: g[key]})
        assert np.array_equal(g[key].values(), first[key])
    release(ctx, layer, {**d, **g})
    ctx.close()


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_relu_gradient_is_exact_on_whole_numbers(type):
    """Small whole numbers: every sum is exact, zero among them, where the
    slope is zero."""
    rng = np.random.default_rng(3)
    rows, k, n = 90, 24, 40
    x = rng.integers(-1, 2, (rows, k)).astype(np.float64)
    w = rng.integers(-1, 2, (n, k)).astype(np.float64)
    dy = rng.integers(-1, 2, (rows, n)).astype(np.float64)
    ctx = context()
    layer, d = run_forward(ctx, x, w, None, None, type, type, "relu", False, training=True)
    z, slope, h, norm, y = linear(x, w, None, None, "relu", False)
    assert (z == 0).any()
    assert np.array_equal(d["y"].values(), y)
    g = {"dy": Matrix(ctx, dy, type), "dx": Matrix(ctx, None, type, shape=(rows, k)),
         "dw": Matrix(ctx, None, type, shape=(n, k))}
    layer.backward(d["x"], g["dy"], saved=d["saved"], dx=g["dx"], dweight=g["dw"])
    _, _, dx, dw, _ = linear_gradients(x, w, dy, y, slope, norm, False)
    assert np.array_equal(g["dx"].values(), to_type(dx, type))
    assert np.array_equal(g["dw"].values(), to_type(dw, type))
    release(ctx, layer, {**d, **g})
    ctx.close()


@pytest.mark.parametrize("act,normalize", [("gelu", False), ("gelu_tanh", True), ("silu", True), ("none", True)])
def test_gradient_against_differences(act, normalize):
    """<gradient, direction> against central differences of the definition in
    64 bits: h = 1e-4 leaves h^2 and 1e-16 / h, both far below the 32-bit
    gradients' error of about 2^-20 of the sum of magnitudes."""
    rng = np.random.default_rng(8)
    rows, k, n = 40, 24, 32
    x, w, b, r = make(rng, rows, k, n, "f32", True, True)
    dy = to_type(rng.standard_normal((rows, n)), "f32")
    ctx = context()
    layer, d = run_forward(ctx, x, w, b, r, "f32", "f32", act, normalize, training=True)
    g = {"dy": Matrix(ctx, dy, "f32"), "x": Matrix(ctx, None, "f32", shape=(rows, k)),
         "w": Matrix(ctx, None, "f32", shape=(n, k)), "b": Matrix(ctx, None, "f32", shape=(1, n)),
         "r": Matrix(ctx, None, "f32", shape=(rows, n)) if normalize else None}
    g["b"].shape = (n,)
    layer.backward(d["x"], g["dy"], saved=d["saved"], y=d["y"], norms=d["norms"], dx=g["x"], dweight=g["w"],
                   dbias=g["b"], dresidual=g["r"])
    at = {"x": x, "w": w, "b": b, "r": r}
    for name in ("x", "w", "b", "r"):
        grad = dy if g[name] is None else g[name].values()
        v = rng.standard_normal(at[name].shape)
        step = 1e-4

        def loss(s):
            p = {m: a + (s * v if m == name else 0.0) for m, a in at.items()}
            return (dy * linear(p["x"], p["w"], p["b"], p["r"], act, normalize)[4]).sum()

        want = (loss(step) - loss(-step)) / (2 * step)
        have = (grad.reshape(v.shape) * v).sum()
        assert abs(want - have) <= 2.0**-18 * np.abs(grad.reshape(v.shape) * v).sum() + 1e-5
    release(ctx, layer, {**d, **g})
    ctx.close()


@pytest.mark.parametrize("rows", [5, 200])
def test_rows_that_are_not_finite_stay_apart(rows):
    """NaN and infinity reach their own row only; a row of zeros normalizes to
    zeros, with the least norm."""
    rng = np.random.default_rng(4)
    x, w, _, _ = make(rng, rows, 72, 64, "bf16", False, False)
    x[1, 70], x[2, 0], x[3] = np.nan, np.inf, 0.0
    ctx = context()
    layer, d = run_forward(ctx, x, w, None, None, "bf16", "f32", "none", True, training=True)
    y = d["y"].values()
    assert np.isnan(y[1]).all() and not np.isfinite(y[2]).all()
    assert (y[3] == 0).all() and np.float32(d["norms"].values()[3]) == np.float32(1e-12)
    rest = np.r_[0, 4:rows]
    assert np.isfinite(y[rest]).all() and np.allclose((y[rest] ** 2).sum(1), 1, atol=1e-5)
    dy = rng.standard_normal((rows, 64))
    g = {"dy": Matrix(ctx, dy, "f32"), "dr": Matrix(ctx, None, "bf16", shape=(rows, 64))}
    layer.backward(d["x"], g["dy"], y=d["y"], norms=d["norms"], dresidual=g["dr"])
    dr = g["dr"].values()
    # the least norm is a constant: dY / 1e-12
    want = to_type(np.float32(dy[3]) / np.float32(1e-12), "bf16")
    assert np.allclose(dr[3], want, rtol=2.0**-8)
    assert np.isfinite(dr[rest]).all() and np.isnan(dr[1]).all()
    release(ctx, layer, {**d, **g})
    ctx.close()


def test_no_rows():
    ctx = context()
    rng = np.random.default_rng(1)
    w = Matrix(ctx, rng.standard_normal((24, 16)), "bf16")
    layer = operators.Linear(ctx, w, activation="none", max_rows=4, training=True)
    x, y = Matrix(ctx, np.zeros((1, 16)), "bf16"), Matrix(ctx, np.ones((1, 24)), "bf16")
    x.shape, y.shape = (0, 16), (0, 24)
    layer.forward(x, y)
    dw, db = Matrix(ctx, None, "bf16", 3, shape=(24, 16)), Matrix(ctx, None, "bf16", shape=(1, 24))
    db.shape = (24,)
    layer.backward(x, y, dweight=dw, dbias=db)
    assert (dw.values() == 0).all() and (db.values() == 0).all()
    y.shape = (1, 24)
    assert (y.values() == 1).all()
    layer.close()
    for v in (w, x, y, dw, db):
        v.free()
    ctx.close()


def test_graph_of_a_training_step():
    """The calls allocate nothing and wait for nothing: a captured step's
    replays give the eager results, with eager work between them."""
    import ctypes as C

    hip = C.CDLL("libamdhip64.so.7")
    rng = np.random.default_rng(12)
    x, w, b, _ = make(rng, 600, 128, 96, "bf16", True, False)
    dy = to_type(rng.standard_normal((600, 96)), "f32")
    ctx = context()
    layer, d = run_forward(ctx, x, w, b, None, "bf16", "f32", "gelu", True, training=True)
    g = {"dy": Matrix(ctx, dy, "f32"), "dx": Matrix(ctx, None, "bf16", shape=x.shape),
         "dw": Matrix(ctx, None, "bf16", shape=w.shape), "db": Matrix(ctx, None, "bf16", shape=(1, 96))}
    g["db"].shape = (96,)

    def step():
        layer.forward(d["x"], d["y"], saved=d["saved"], norms=d["norms"])
        layer.backward(d["x"], g["dy"], saved=d["saved"], y=d["y"], norms=d["norms"], dx=g["dx"], dweight=g["dw"],
                       dbias=g["db"])

    def results():
        return [v.values() for v in (d["y"], g["dx"], g["dw"], g["db"])]

    step()
    want = results()
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    from chimera_amd import capi
    capi.check(capi.lib().chimera_stream(ctx.handle, C.byref(stream)))
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    step()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for _ in range(3):
        assert hip.hipGraphLaunch(run, stream) == 0
        ctx.synchronize()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want))
        step()
        ctx.synchronize()
    hip.hipGraphExecDestroy(run)
    hip.hipGraphDestroy(graph)
    release(ctx, layer, {**d, **g})
    ctx.close()


@pytest.mark.parametrize("type,out", [("f32", "f32"), ("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("rows", [1, 40])
def test_gelu_over_its_range(type, out, rows):
    """Sums that are the weights themselves. Results in 32 bits are within
    2^-20 of 1 + |z|, and below zero, where they are small, within 2^-8 of
    their size to -6; those rounded to 16 bits within 2^-12 of their size to -4
    and 2^-8 to -6, before the rounding; infinities and NaN as in the formula."""
    z = to_type(np.concatenate([np.linspace(-12, 12, 4001), [0.0, 1e-3, -1e-3, 60000.0, -60000.0]])[None], type)
    special = to_type(np.array([[np.inf, -np.inf, np.nan]]), type)
    w = np.concatenate([z, special], axis=1).T
    x = np.ones((rows, 1))
    ctx = context()
    layer, d = run_forward(ctx, x, w, None, None, type, out, "gelu", False)
    have = d["y"].values()[-1]
    want = linear(x[:1], z.T, None, None, "gelu", False)[4][0]
    z = z[0]
    size = np.abs(want)
    off = 2.0**-20 * (1 + np.abs(z)) if out == "f32" else 2.0**-12 * size
    close = np.where(z < -6, 3e-8, np.where(z < -4, 2.0**-8 * size, np.maximum(2.0**-12 * size, off)))
    close = np.where((out == "f32") & (z < 0), np.minimum(off, np.maximum(2.0**-8 * size, 3e-8)), close)
    least = 2.0**-25 if out == "f16" else 0.0
    assert (np.abs(have[:-3] - want) <= close + 2.0**-BITS[out] * size + least).all()
    assert have[-3] == np.inf and np.isnan(have[-2:]).all()
    release(ctx, layer, d)
    ctx.close()
