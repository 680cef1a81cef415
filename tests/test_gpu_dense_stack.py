"""The dense stack's operators on the kernels of dense_stack_shapes, and a run of
them together as a training step and the queries after it make one."""
import numpy as np
import pytest

from chimera_amd import operators
from dense_stack_shapes import MX4_LAYERS, NORMS, UPDATES
from graph_replay import check_replays
from mx4_checks import quantise
from operator_checks import Array, Matrix, context, linear, to_type
from test_gpu_linear import forward_bounds
from test_gpu_mx4 import test_layer as check_layer, test_sums_of_whole_numbers as check_sums
from test_gpu_norm import Case, D, U, make, norm, rounding, vector
from test_gpu_orthogonal import ABC, steps_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,n,type,out,forward,backward", NORMS)
def test_norms(rows, n, type, out, forward, backward):
    rng = np.random.default_rng(rows + n)
    print(f"{rows} x {n} {type} -> {out}", flush=True)
    x, w, b, dy = make(rng, rows, n, type, out)
    odd = n % 2
    c = Case(x, w, b, dy, type, out, pad=odd, shift=odd)
    c.forward()
    c.backward()
    c.check()
    c.close()


@pytest.mark.parametrize("rows,k,n,type,normalize,kernel", MX4_LAYERS)
def test_4_bit_layers(rows, k, n, type, normalize, kernel):
    if normalize:
        check_layer(rows, k, n, type, "f32", "silu", True, True, True, 3, 0)
    else:
        check_sums(rows, k, n, type)


@pytest.mark.parametrize("rows,cols,symmetric,x", UPDATES)
def test_updates(rows, cols, symmetric, x):
    """Gradients of 16 equal singular values, whose two steps are the polynomial
    of those. A step's values have errors of 2^-22 of theirs, its products
    a few more, times |b| + 2 |c| at most: 32 2^-22 of X's length together,
    which is 1 at first, 3.5 after a step at most, whose slopes are at most 3.9:
    32 2^-22 (3.9 + 3.5). The gradient's own rounding, 2^-24 of it, grows by
    3.9^2. No element of the result is that small a part of it."""
    rng = np.random.default_rng(rows + cols)
    print(f"{rows} x {cols}", flush=True)
    left, right = (np.linalg.qr(rng.standard_normal((v, 16)))[0] for v in (rows, cols))
    g = to_type(left @ right.T, "f32")
    a, b, c = (np.float64(np.float32(v)) for v in ABC)
    s = 0.25
    for _ in range(2):
        s = a * s + b * s**3 + c * s**5
    ctx = context()
    update = operators.OrthogonalUpdate(ctx, rows, cols, steps=2)
    d_g, d_out = Matrix(ctx, g, "f32"), Matrix(ctx, None, "f32", shape=g.shape)
    update.orthogonalize(d_g, d_out)
    off = np.linalg.norm(d_out.values() - s * left @ right.T)
    assert off <= 32 * 2.0**-22 * 7.4 + 3.9**2 * 2.0**-24
    update.close()
    d_g.free()
    d_out.free()
    ctx.close()


class Stack:
    """Token states through a norm, a hidden layer and the layer of the
    embeddings, whose weight takes an orthogonal step from its gradient; then
    queries through both layers' 4-bit weights."""

    def __init__(self, rng, rows=600, queries=9, k=256, hidden=320, n=96, type="bf16"):
        self.ctx = ctx = context()
        self.type, self.k, self.hidden, self.n = type, k, hidden, n
        new = lambda rows, cols, t=type: Matrix(ctx, None, t, shape=(rows, cols))
        put = lambda scale, *shape: to_type(scale * rng.standard_normal(shape), type)
        w1, w2 = put(1 / np.sqrt(k), hidden, k), put(1 / np.sqrt(hidden), n, hidden)
        self.d = d = {
            "x": Matrix(ctx, put(1.0, rows, k), type), "q": Matrix(ctx, put(1.0, queries, k), type),
            "scale": vector(ctx, 1 + put(0.2, k), type), "shift": vector(ctx, put(0.2, k), type),
            "w1": Matrix(ctx, w1, type), "w2": Matrix(ctx, w2, type), "b1": vector(ctx, put(0.1, hidden), type),
            "master": Matrix(ctx, w2, "f32"), "next": new(n, hidden, "f32"), "momentum": Matrix(ctx, put(1e-3, n, hidden), "f32"),
            "next momentum": new(n, hidden, "f32"), "rounded": new(n, hidden),
            "y": new(rows, k), "h": new(rows, hidden), "saved": new(rows, hidden), "e": new(rows, n),
            "de": Matrix(ctx, put(1.0, rows, n), type), "dh": new(rows, hidden), "dw2": new(n, hidden),
            "dw1": new(hidden, k), "dy": new(rows, k), "dx": new(rows, k), "dscale": vector(ctx, None, type, k),
            "dshift": vector(ctx, None, type, k), "mean": vector(ctx, None, "f32", rows), "rstd": vector(ctx, None, "f32", rows),
            "qy": new(queries, k), "qh": new(queries, hidden), "qe": new(queries, n, "f32"),
        }
        for name, (o, i) in (("1", (hidden, k)), ("2", (n, hidden))):
            row, blocks = operators.mx4_row(i)
            d["codes" + name], d["scales" + name] = Array(ctx, np.zeros((o, row), np.uint8)), Array(ctx, np.zeros((o, blocks), np.uint8))
        self.norm = operators.LayerNorm(ctx, d["scale"], d["shift"], max_rows=rows, training=True)
        self.one = operators.Linear(ctx, d["w1"], d["b1"], activation="gelu", max_rows=rows, training=True)
        self.two = operators.Linear(ctx, d["w2"], max_rows=rows, training=True)
        self.update = operators.OrthogonalUpdate(ctx, n, hidden, type=type)
        self.small_one = operators.Mx4Linear(ctx, d["codes1"], d["scales1"], k, d["b1"], type=type, activation="gelu",
                                             max_rows=queries)
        self.small_two = operators.Mx4Linear(ctx, d["codes2"], d["scales2"], hidden, type=type, normalize=True, max_rows=queries)

    def run(self):
        d = self.d
        self.norm.forward(d["x"], d["y"], mean=d["mean"], rstd=d["rstd"])
        self.one.forward(d["y"], d["h"], saved=d["saved"])
        self.two.forward(d["h"], d["e"])
        self.two.backward(d["h"], d["de"], dx=d["dh"], dweight=d["dw2"])
        self.one.backward(d["y"], d["dh"], saved=d["saved"], dx=d["dy"], dweight=d["dw1"])
        self.norm.backward(d["x"], d["dy"], d["mean"], d["rstd"], dx=d["dx"], dweight=d["dscale"], dbias=d["dshift"])
        self.update.step(d["dw2"], d["master"], d["next"], rate=0.02, decay=0.01, momentum=d["momentum"],
                         new_momentum=d["next momentum"], mu=0.9, rounded=d["rounded"])
        operators.mx4_quantise(self.ctx, d["w1"], d["codes1"], d["scales1"])
        operators.mx4_quantise(self.ctx, d["rounded"], d["codes2"], d["scales2"])
        self.norm.forward(d["q"], d["qy"])
        self.small_one.forward(d["qy"], d["qh"])
        self.small_two.forward(d["qh"], d["qe"])

    RESULTS = ("y", "h", "e", "dx", "dscale", "dshift", "dw1", "dw2", "next", "rounded", "qe")

    def results(self):
        return [self.d[v].values() for v in self.RESULTS]

    def check(self):
        """Each operator's result from what it read on the device."""
        v = {name: m.values() for name, m in self.d.items() if isinstance(m, Matrix)}
        scale, shift = v["scale"].ravel(), v["shift"].ravel()
        for x, y in (("x", "y"), ("q", "qy")):
            z, rstd, want = norm(v[x], scale, shift, 1e-5)
            ez = (D + 8) * U * (np.abs(z) + 1)
            assert (np.abs(v[y] - want) <= np.abs(scale) * ez + 2 * U * (np.abs(z * scale) + np.abs(want))
                    + rounding(want, self.type)).all()
        z, rstd, _ = norm(v["x"], scale, shift, 1e-5)
        dw, db = (v["dy"] * z).sum(0), v["dy"].sum(0)
        off = (D + 1200) * U
        for have, want, parts in (("dscale", dw, v["dy"] * (np.abs(z) + 1)), ("dshift", db, v["dy"])):
            assert (np.abs(v[have].ravel() - want) <= off * np.abs(parts).sum(0) + rounding(want, self.type)).all()
        # the step: momentum and gradient, orthogonal, then the weight
        mu, rate = np.float64(np.float32(0.9)), np.float64(np.float32(0.02))
        keep = np.float64(np.float32(1) - np.float32(0.01))
        m = v["next momentum"]
        assert (np.abs(m - (mu * v["momentum"] + v["dw2"])) <= 2.0**-24 * np.abs(m) + 1e-45).all()
        x = (keep * v["master"] - v["next"]) / rate
        # read off the weight, X has the roundings of two 32-bit values of its size over the rate
        lost = 2.0**-23 * np.linalg.norm(v["master"]) / rate
        u = to_type(v["dw2"] + mu * m, "f32")
        exact = steps_of(u, np.float64)
        off = 4 * np.linalg.norm(steps_of(u, np.float32) - exact) + 2.0**-22 * np.linalg.norm(exact)
        assert np.linalg.norm(x - exact) <= off + lost
        assert np.array_equal(v["rounded"], to_type(v["next"], self.type))
        # the queries through the 4-bit weights
        for x, w, b, act, normalize, y, out in (("qy", "w1", v["b1"].ravel(), "gelu", False, "qh", self.type),
                                                ("qh", "rounded", None, "none", True, "qe", "f32")):
            x, w = quantise(v[x])[2], quantise(v[w])[2]
            _, _, h, length, want = linear(x, w, b, None, act, normalize)
            _, _, ey = forward_bounds(x, w, b, h, length, want, out, normalize)
            assert (np.abs(v[y] - want) <= ey + (2.0**-17 * np.abs(want) if act == "gelu" else 0.0)).all()

    def close(self):
        for v in (self.norm, self.one, self.two, self.update, self.small_one, self.small_two):
            v.close()
        for v in self.d.values():
            v.free()
        self.ctx.close()


def test_a_training_step_and_the_queries_after_it():
    stack = Stack(np.random.default_rng(1))
    stack.run()
    stack.ctx.synchronize()
    stack.check()
    stack.close()


def test_the_step_and_its_queries_in_a_graph():
    stack = Stack(np.random.default_rng(2), rows=130, queries=1)
    check_replays(stack.ctx, stack.run, stack.results)
    stack.check()
    stack.close()


def test_two_contexts_at_once():
    """Calls on two streams, neither waiting for the other, give what each gives
    alone."""
    stacks = [Stack(np.random.default_rng(3 + i), rows=900 + 100 * i) for i in range(2)]
    want = []
    for s in stacks:
        s.run()
        s.ctx.synchronize()
        want.append(s.results())
    for _ in range(5):
        for s in stacks:
            s.run()
    for s, w in zip(stacks, want):
        s.ctx.synchronize()
        assert all(np.array_equal(a, b) for a, b in zip(s.results(), w))
        s.close()
