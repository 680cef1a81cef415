"""Layer norm and its gradients against their definition in 64 bits.

Tolerances. u = 2^-24. A value passes at most D = 100 additions on its way into
a row's sum (64 in its thread, 6 in the wave, 16 between waves and a few more),
so such a sum is within D u of the sum of magnitudes. x - mean is rounded once
and its mean taken away again, so z is within (D + 8) u of |z| + 1: the mean of
|z| is at most 1, and the variance's error enters by half. A gradient g - mean
of g - z mean of g z has the errors of its three parts, 4 D u of their
magnitudes at most. A sum over rows passes at most as many additions as there
are rows, and 600 in the join. Rounding to a type of p bits adds 2^-p of the
value, and to f16 at least 2^-25."""
import numpy as np
import pytest

from chimera_amd import operators
from graph_replay import check_replays
from operator_checks import BITS, Matrix, context, to_type

pytestmark = pytest.mark.gpu

U, D = 2.0**-24, 100


def vector(ctx, x, type, n=None):
    v = Matrix(ctx, None if x is None else x[None], type, shape=(1, n if x is None else x.size))
    v.shape = (v.shape[1],)
    return v


def norm(x, w, b, eps):
    """z, rstd and y in 64 bits."""
    d = x - x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt((d * d).mean(1, keepdims=True) + np.float64(np.float32(eps)))
    z = d * rstd
    return z, rstd, z * w + b


def gradients(dy, z, rstd, w):
    g = dy * w
    return g, rstd * (g - g.mean(1, keepdims=True) - z * (g * z).mean(1, keepdims=True)), (dy * z).sum(0), dy.sum(0)


def rounding(v, type):
    return 2.0**-BITS[type] * np.abs(v) + (2.0**-25 if type == "f16" else 0.0)


class Case:
    """One norm with its arrays on the device."""

    def __init__(self, x, w, b, dy, type, out, pad=0, shift=0, eps=1e-5, training=True):
        self.ctx = ctx = context()
        rows, n = x.shape
        self.type, self.out, self.eps = type, out, eps
        self.x, self.w, self.b, self.dy = x, w, b, dy
        self.d = {"x": Matrix(ctx, x, type, pad, shift), "y": Matrix(ctx, None, out, pad, shift, shape=(rows, n)),
                  "w": None if w is None else vector(ctx, w, type), "b": None if b is None else vector(ctx, b, type)}
        if training:
            self.d.update(mean=vector(ctx, None, "f32", rows), rstd=vector(ctx, None, "f32", rows),
                          dy=Matrix(ctx, dy, out, pad, shift), dx=Matrix(ctx, None, type, pad, shift, shape=(rows, n)),
                          dw=vector(ctx, None, type, n), db=vector(ctx, None, type, n))
        self.norm = operators.LayerNorm(ctx, self.d["w"], self.d["b"], eps=eps, max_rows=rows, training=training, features=n,
                                        type=type)

    def forward(self):
        self.norm.forward(self.d["x"], self.d["y"], mean=self.d.get("mean"), rstd=self.d.get("rstd"))

    def backward(self, **out):
        out = out or {"dx": self.d["dx"], "dweight": self.d["dw"], "dbias": self.d["db"]}
        self.norm.backward(self.d["x"], self.d["dy"], self.d["mean"], self.d["rstd"], **out)

    def value(self, name):
        return self.d[name].values()

    def check(self):
        n = self.x.shape[1]
        w = np.ones(n) if self.w is None else self.w
        b = np.zeros(n) if self.b is None else self.b
        z, rstd, y = norm(self.x, w, b, self.eps)
        ez = (D + 8) * U * (np.abs(z) + 1)
        assert (np.abs(self.value("y") - y) <= np.abs(w) * ez + 2 * U * (np.abs(z * w) + np.abs(y)) + rounding(y, self.out)).all()
        if "dx" not in self.d:
            return
        assert (np.abs(self.value("rstd") - rstd[:, 0]) <= (D + 8) * U * rstd[:, 0]).all()
        dy = self.dy
        g, dx, dw, db = gradients(dy, z, rstd, w)
        mean = lambda v: np.abs(v).mean(1, keepdims=True)
        edx = rstd * 4 * D * U * (np.abs(g) + mean(g) + (np.abs(z) + 1) * (mean(g * z) + mean(g)))
        assert (np.abs(self.value("dx") - dx) <= edx + rounding(dx, self.type)).all()
        along = (self.x.shape[0] + 600) * U
        assert (np.abs(self.value("dw") - dw) <= (np.abs(dy) * ez).sum(0) + along * np.abs(dy * z).sum(0) + rounding(dw, self.type)).all()
        assert (np.abs(self.value("db") - db) <= along * np.abs(dy).sum(0) + rounding(db, self.type)).all()
        for name in ("x", "dy"):
            self.value(name)  # untouched around

    def close(self):
        self.norm.close()
        for v in self.d.values():
            if v is not None:
                v.free()
        self.ctx.close()


def make(rng, rows, n, type, out):
    size = np.exp(0.5 * rng.standard_normal(n))
    size[rng.integers(0, n)] *= 8
    x = to_type(rng.standard_normal((rows, n)) * size + 0.3 * size * rng.standard_normal(n), type)
    return (x, to_type(1 + 0.3 * rng.standard_normal(n), type), to_type(rng.standard_normal(n), type),
            to_type(rng.standard_normal((rows, n)), out))


CASES = [
    # rows, features, type, out, weight, bias, pad, shift
    (1, 1, "f32", "f32", True, True, 0, 0),
    (5, 2, "bf16", "f32", False, False, 1, 1),
    (1, 768, "bf16", "bf16", True, True, 0, 0),
    (33, 7, "f16", "f16", True, False, 0, 0),
    (100, 48, "f32", "f32", True, True, 3, 1),
    (1025, 128, "bf16", "bf16", True, True, 0, 0),
    (70, 129, "f16", "f32", False, True, 7, 3),
    (600, 512, "bf16", "f32", True, True, 8, 8),
    (601, 513, "f32", "f32", True, True, 0, 0),
    (2500, 777, "bf16", "bf16", True, True, 3, 0),
    (3000, 1024, "f16", "f16", True, True, 0, 0),
    (9, 1025, "f32", "f32", False, False, 0, 2),
    (700, 2000, "bf16", "bf16", True, True, 0, 0),
    (40, 2049, "bf16", "bf16", True, True, 1, 0),
    (300, 4096, "f16", "f32", True, False, 0, 0),
    (65, 8190, "f32", "f32", True, True, 2, 0),
    (3, 8193, "bf16", "bf16", True, True, 0, 0),
    (130, 20_000, "f32", "f32", True, True, 0, 1),
    (5, 32_769, "f16", "f16", True, True, 0, 0),
    (70, 65_536, "bf16", "f32", True, True, 0, 0),
]


@pytest.mark.parametrize("rows,n,type,out,weight,bias,pad,shift", CASES)
def test_forward_and_backward(rows, n, type, out, weight, bias, pad, shift):
    rng = np.random.default_rng(rows * 3 + n)
    x, w, b, dy = make(rng, rows, n, type, out)
    print(f"{rows} x {n} {type} -> {out}", flush=True)
    c = Case(x, w if weight else None, b if bias else None, dy, type, out, pad, shift)
    c.forward()
    c.backward()
    c.check()
    # one gradient at a time, and the same sums again
    first = {name: c.value(name) for name in ("dx", "dw", "db")}
    for name, key in (("dx", "dx"), ("dweight", "dw"), ("dbias", "db")):
        c.backward(**{name: c.d[key]})
        assert np.array_equal(c.value(key), first[key]), name
    c.close()


@pytest.mark.parametrize("n", [96, 512, 1000, 3000, 30_000])
def test_rows_far_from_zero_and_near_the_ends_of_the_range(n):
    """Rows of 1 + 1e-3 noise at 1e4, of values whose squares pass the 32-bit
    range at both ends, constant rows and rows of zeros."""
    rng = np.random.default_rng(n)
    x, w, b, dy = make(rng, 12, n, "f32", "f32")
    noise = rng.standard_normal((12, n))
    x[0], x[1] = 1e4 + noise[0], -3e6 + 100 * noise[1]
    x[2], x[3], x[4] = 1e19 * noise[2], 1e30 * noise[3], 1e37 * noise[4]
    x[5], x[6] = 1e-20 * noise[5], 1e-42 * noise[6]
    x[7], x[8] = 12345.678, 0.0
    x[9] = np.where(np.arange(n) % 2, 3.3e38, -3.3e38)
    x[10] = 3e38 + 3e37 * np.abs(noise[10]).clip(max=1)
    x = to_type(x, "f32")
    c = Case(x, w, b, dy, "f32", "f32", eps=1e-12)
    c.forward()
    c.backward()
    y = c.value("y")
    assert np.allclose(y[7:9], b, atol=1e-4 * np.abs(w).max())  # a constant's mean is within a rounding
    z, rstd, want = norm(x, w, b, 1e-12)
    # the statistics of huge rows are kept to 2^-21 of their size, which is below the normal numbers
    ez = ((D + 8) * U + 2.0**-21) * (np.abs(z) + 1)
    near = np.r_[0:7, 8:12]
    assert (np.abs(y - want)[near] <= (np.abs(w) * ez + 4 * U * (np.abs(z * w) + np.abs(want)))[near]).all()
    _, dx, _, _ = gradients(dy, z, rstd, w)
    g = np.abs(dy * w)
    mean = lambda v: np.abs(v).mean(1, keepdims=True)
    edx = rstd * (4 * D * U + 2.0**-18) * (g + mean(g) + (np.abs(z) + 1) * (mean(g * z) + mean(g))) + 2.0**-148
    assert (np.abs(c.value("dx") - dx)[near] <= edx[near]).all()
    c.close()


@pytest.mark.parametrize("eps", [1e-5, 1e-30])
@pytest.mark.parametrize("n", [5, 96, 1000, 3000, 30_000])
def test_rows_of_one_value(n, eps):
    """x - mean is what the mean's rounding left out, the same in all columns,
    and its mean is within D u of it, so z, over a deviation of at least 2^-9 of
    that, is below D u 2^9 + 2^-15 < 2^-8. Gradients are finite."""
    rng = np.random.default_rng(n)
    values = [0.0, 1.0, 12345.678, -3e6, 1e8, 1.7e19, 3e30, 2.0**115, 1e36, 2.0**127, 3e38, -3.4e38, 1e-30, 1e-42]
    x = to_type(np.repeat(np.array(values)[:, None], n, 1), "f32")
    w, b = to_type(1 + 0.3 * rng.standard_normal(n), "f32"), to_type(rng.standard_normal(n), "f32")
    dy = to_type(rng.standard_normal(x.shape), "f32")
    c = Case(x, w, b, dy, "f32", "f32", eps=eps)
    c.forward()
    c.backward()
    assert (np.abs(c.value("y") - b) <= 2.0**-8 * np.abs(w) + U * np.abs(b)).all()
    assert np.isfinite(c.value("dx")).all() and np.isfinite(c.value("dw")).all()
    rstd = 1 / np.sqrt(np.float64(np.float32(eps)))
    near = np.abs(x[:, 0]) <= 1e-30  # the others' means may be a rounding off, and eps below its square
    have = c.value("rstd").ravel()
    assert (np.abs(have - rstd)[near] <= 2.0**-20 * rstd).all()
    assert (have > 0).all() and (have <= rstd * (1 + 2.0**-20)).all()
    c.close()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [40, 300, 5000])
def test_rows_that_are_not_finite_stay_apart(type, n):
    rng = np.random.default_rng(n)
    x, w, b, dy = make(rng, 9, n, type, type)
    good = x.copy()
    x[1, n - 1], x[4, 0], x[5, 3] = np.nan, np.inf, -np.inf
    c = Case(x, w, b, dy, type, type)
    c.forward()
    c.backward()
    y, dx = c.value("y"), c.value("dx")
    bad = [1, 4, 5]
    assert np.isnan(y[bad]).all() and np.isnan(dx[bad]).all() and np.isnan(c.value("dw")).all()
    assert np.isfinite(c.value("db")).all()
    rest = np.setdiff1d(np.arange(9), bad)
    clean = Case(good, w, b, dy, type, type)
    clean.forward()
    clean.backward()
    assert np.array_equal(y[rest], clean.value("y")[rest]) and np.array_equal(dx[rest], clean.value("dx")[rest])
    c.close()
    clean.close()


@pytest.mark.parametrize("n", [24, 700])
def test_gradient_against_differences(n):
    """<gradient, direction> against central differences of the definition in
    64 bits: a step of 1e-4 leaves its square, about 1e-8 of the sum of
    magnitudes, far below the 2^-18 that the 32-bit gradients are given."""
    rng = np.random.default_rng(n)
    x, w, b, dy = make(rng, 30, n, "f32", "f32")
    c = Case(x, w, b, dy, "f32", "f32")
    c.forward()
    c.backward()
    at = {"x": x, "w": w, "b": b}
    for name in ("x", "w", "b"):
        grad = c.value("d" + name).reshape(at[name].shape)
        v = rng.standard_normal(at[name].shape)

        def loss(s):
            p = {m: a + (s * v if m == name else 0.0) for m, a in at.items()}
            return (dy * norm(p["x"], p["w"], p["b"], 1e-5)[2]).sum()

        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        assert abs(want - (grad * v).sum()) <= 2.0**-18 * np.abs(grad * v).sum() + 1e-5
    c.close()


def test_no_rows():
    rng = np.random.default_rng(1)
    x, w, b, dy = make(rng, 1, 200, "bf16", "bf16")
    c = Case(x, w, b, dy, "bf16", "bf16")
    for name in ("x", "y", "dy", "dx"):
        c.d[name].shape = (0, 200)
    for name in ("mean", "rstd"):
        c.d[name].shape = (0,)
    before = c.d["y"].buffer.numpy()
    c.forward()
    c.backward()
    assert np.array_equal(c.d["y"].buffer.numpy(), before)
    assert (c.value("dw") == 0).all() and (c.value("db") == 0).all()
    c.close()


@pytest.mark.parametrize("n", [100, 768, 10_000])
def test_graph_of_a_training_step(n):
    rng = np.random.default_rng(n)
    x, w, b, dy = make(rng, 300, n, "bf16", "bf16")
    c = Case(x, w, b, dy, "bf16", "bf16")

    def calls():
        c.forward()
        c.backward()

    check_replays(c.ctx, calls, lambda: [c.value(v) for v in ("y", "dx", "dw", "db")])
    c.close()


def test_fewer_rows_than_the_workspace_is_for():
    rng = np.random.default_rng(6)
    x, w, b, dy = make(rng, 2000, 260, "f32", "f32")
    c = Case(x, w, b, dy, "f32", "f32")
    for rows in (2000, 1, 17):
        c.x, c.dy = x[:rows], dy[:rows]
        for name in ("x", "y", "dy", "dx"):
            c.d[name].shape = (rows, 260)
        for name in ("mean", "rstd"):
            c.d[name].shape = (rows,)
        c.forward()
        c.backward()
        z, rstd, y = norm(c.x, w, b, 1e-5)
        _, dx, dw, db = gradients(c.dy, z, rstd, w)
        assert np.abs(c.d["y"].buffer.numpy().view(np.float32)[:rows * 260].reshape(rows, 260) - y).max() <= 1e-4
        assert np.abs(c.value("dw") - dw).max() <= 1e-3 and np.abs(c.value("db") - db).max() <= 1e-3
    c.close()
