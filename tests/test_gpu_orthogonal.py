"""The orthogonal update against its definition in 64 bits.

Tolerances. Errors grow with the steps as the singular values do, so they are
held against those of the same steps in 32-bit arithmetic: values of 22 bits
instead of 24 have four times its rounding errors, so the result is within four
times the distance that 32 bits have from 64, and 2^-22 of its size. Rounding
to a type of p bits adds 2^-p."""
import numpy as np
import pytest

from chimera_amd import operators
from graph_replay import check_replays
from operator_checks import BITS, Matrix, context, to_type

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)


def steps_of(u, kind, count=5, abc=ABC):
    """X after the steps, in float64 or float32."""
    a, b, c = (kind(np.float32(v)) for v in abc)
    turned = u.shape[0] > u.shape[1]
    x = np.asarray(u, np.float64)
    size = np.sqrt((x * x).sum())
    x = (x / size if size > 0 else x).astype(kind)
    x = x.T if turned else x
    for _ in range(count):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return (x.T if turned else x).astype(np.float64)


def close_to(have, u, type, count=5, abc=ABC):
    want = steps_of(u, np.float64, count, abc)
    size = np.linalg.norm(want)
    off = 4 * np.linalg.norm(steps_of(u, np.float32, count, abc) - want) + 2.0**-22 * size
    assert np.linalg.norm(have - want) <= off + 2.0**-BITS[type] * size + (2.0**-25 * np.sqrt(want.size) if type == "f16" else 0)


def gradient(rng, rows, cols, kind, type):
    few = max(1, min(rows, cols) // 8)
    g = rng.standard_normal((rows, cols))
    if kind == "strong":
        g = rng.standard_normal((rows, few)) @ rng.standard_normal((few, cols)) / np.sqrt(few) + 0.3 * g
    elif kind == "low rank":
        g = rng.standard_normal((rows, few)) @ rng.standard_normal((few, cols)) / np.sqrt(few)
    return to_type(1e-3 * g, type)


CASES = [
    # rows, cols, type, out, kind, pad, shift
    (1, 1, "f32", "f32", "noise", 0, 0),
    (1, 300, "bf16", "f32", "noise", 0, 0),
    (70, 1, "f16", "f16", "noise", 2, 1),
    (2, 3, "f32", "f32", "noise", 0, 0),
    (31, 33, "f32", "f32", "noise", 1, 1),
    (64, 64, "bf16", "bf16", "strong", 0, 0),
    (65, 63, "f32", "f32", "strong", 0, 0),
    (128, 768, "f32", "f32", "strong", 0, 0),
    (500, 129, "f16", "f32", "low rank", 3, 0),
    (200, 260, "bf16", "f32", "strong", 0, 2),
    (1000, 300, "f32", "f32", "strong", 4, 0),
    (384, 1030, "f32", "f32", "low rank", 0, 0),
    (640, 600, "bf16", "bf16", "noise", 0, 0),
    (1100, 1090, "f32", "f32", "strong", 0, 0),
    (96, 8000, "f16", "f32", "strong", 0, 0),
    (4100, 257, "f32", "f32", "noise", 0, 0),
]


def run(ctx, g, type, out, pad=0, shift=0, **kw):
    rows, cols = g.shape
    update = operators.OrthogonalUpdate(ctx, rows, cols, type=type, **kw)
    d_g, d_out = Matrix(ctx, g, type, pad, shift), Matrix(ctx, None, out, pad, shift, shape=g.shape)
    update.orthogonalize(d_g, d_out)
    have = d_out.values()
    update.orthogonalize(d_g, d_out)
    assert np.array_equal(d_out.values(), have, equal_nan=True)
    d_g.values()  # untouched around
    update.close()
    for v in (d_g, d_out):
        v.free()
    return have


@pytest.mark.parametrize("rows,cols,type,out,kind,pad,shift", CASES)
def test_update(rows, cols, type, out, kind, pad, shift):
    rng = np.random.default_rng(rows * 3 + cols)
    print(f"{rows} x {cols} {type} {kind}", flush=True)
    g = gradient(rng, rows, cols, kind, type)
    ctx = context()
    close_to(run(ctx, g, type, out, pad, shift), g, out)
    ctx.close()


@pytest.mark.parametrize("count", [1, 2, 8])
def test_steps_and_coefficients(count):
    """Coefficients that bring singular values to one and keep them."""
    rng = np.random.default_rng(count)
    g = gradient(rng, 90, 150, "noise", "f32")
    ctx = context()
    abc = (15 / 8, -10 / 8, 3 / 8)
    close_to(run(ctx, g, "f32", "f32", steps=count, coefficients=abc), g, "f32", count, abc)
    ctx.close()


@pytest.mark.parametrize("rows,cols", [(64, 64), (100, 700), (700, 100), (513, 1030)])
def test_orthogonal_rows_follow_the_polynomial(rows, cols):
    """Rows (or columns) that are orthogonal already: every singular value is
    1 / sqrt(m), and the result is the input times what the polynomial makes of
    it. One nonzero a row, so a misplaced element shows; sums have one term, so
    each step's error is that of a few roundings of 22 bits, which the slopes
    of the five steps (at most 3.9 each) multiply by at most 3.9^4 + ... + 1."""
    rng = np.random.default_rng(rows)
    m, k = min(rows, cols), max(rows, cols)
    g = np.zeros((m, k))
    g[np.arange(m), rng.permutation(k)[:m]] = rng.choice([-1.0, 1.0], m)
    s = 1 / np.sqrt(m)
    for _ in range(5):
        s = ABC[0] * s + ABC[1] * s**3 + ABC[2] * s**5
    ctx = context()
    for u in (g, 2.0**-90 * g, 2.0**90 * g):
        have = run(ctx, u.T if rows > cols else u, "f32", "f32")
        have = have.T if rows > cols else have
        assert np.array_equal(have != 0, g != 0)
        assert np.abs(have - s * g).max() <= 315 * 8 * 2.0**-22
    ctx.close()


def test_sizes_and_sides_do_not_matter():
    """A power of two times the gradient, or its transpose, gives the same bits."""
    rng = np.random.default_rng(9)
    g = gradient(rng, 150, 330, "strong", "f32")
    ctx = context()
    want = run(ctx, g, "f32", "f32")
    for scale in (2.0**-100, 2.0**100):
        assert np.array_equal(run(ctx, g * scale, "f32", "f32"), want)
    assert np.array_equal(run(ctx, g.T, "f32", "f32"), want.T)
    ctx.close()


def test_gradients_of_zeros_and_not_finite():
    rng = np.random.default_rng(10)
    ctx = context()
    assert (run(ctx, np.zeros((40, 70)), "bf16", "bf16") == 0).all()
    g = gradient(rng, 40, 70, "noise", "f32")
    g[3, 4] = np.nan
    assert np.isnan(run(ctx, g, "f32", "f32")).all()
    g[3, 4] = np.inf
    assert not np.isfinite(run(ctx, g, "f32", "f32")).any()
    ctx.close()


@pytest.mark.parametrize("rows,cols,type", [(128, 200, "f32"), (300, 90, "bf16"), (64, 64, "f16")])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("in_place", [True, False])
def test_step(rows, cols, type, nesterov, in_place):
    rng = np.random.default_rng(rows + nesterov)
    g = gradient(rng, rows, cols, "strong", type)
    m, w = (to_type(v, "f32") for v in (2e-3 * rng.standard_normal(g.shape), rng.standard_normal(g.shape) / np.sqrt(cols)))
    mu, rate, decay = 0.9, 0.03, 0.01
    ctx = context()
    update = operators.OrthogonalUpdate(ctx, rows, cols, type=type)
    d = {"g": Matrix(ctx, g, type, 1, 1), "m": Matrix(ctx, m, "f32", 3), "w": Matrix(ctx, w, "f32", 0, 1),
         "rounded": Matrix(ctx, None, type, 2, shape=g.shape), "x": Matrix(ctx, None, "f32", shape=g.shape)}
    new_m = d["m"] if in_place else Matrix(ctx, None, "f32", 1, shape=g.shape)
    new_w = d["w"] if in_place else Matrix(ctx, None, "f32", 5, shape=g.shape)
    update.step(d["g"], d["w"], None if in_place else new_w, rate=rate, decay=decay, momentum=d["m"],
                new_momentum=None if in_place else new_m, mu=mu, nesterov=nesterov, rounded=d["rounded"], out=d["x"])
    mu32, rate32, keep = np.float64(np.float32(mu)), np.float64(np.float32(rate)), np.float64(np.float32(1) - np.float32(decay))
    want_m = mu32 * m + g
    assert (np.abs(new_m.values() - want_m) <= 2.0**-24 * np.abs(want_m) + 1e-45).all()
    m32 = new_m.values()
    u = to_type(g + mu32 * m32, "f32") if nesterov else m32
    close_to(d["x"].values(), u, "f32")
    want_w = keep * w - rate32 * d["x"].values()
    have_w = new_w.values()
    assert (np.abs(have_w - want_w) <= 2.0**-23 * (np.abs(want_w) + rate32 * np.abs(d["x"].values()))).all()
    assert np.array_equal(d["rounded"].values(), to_type(have_w, type))
    if not in_place:
        assert np.array_equal(d["m"].values(), m) and np.array_equal(d["w"].values(), w)
        new_m.free()
        new_w.free()
    update.close()
    for v in d.values():
        v.free()
    ctx.close()


def test_step_without_momentum_and_out():
    rng = np.random.default_rng(3)
    g, w = gradient(rng, 60, 130, "noise", "f32"), to_type(rng.standard_normal((60, 130)), "f32")
    ctx = context()
    update = operators.OrthogonalUpdate(ctx, 60, 130)
    d_g, d_w, d_new = Matrix(ctx, g, "f32"), Matrix(ctx, w, "f32"), Matrix(ctx, None, "f32", shape=g.shape)
    update.step(d_g, d_w, d_new, rate=1.0, decay=1.0)
    close_to(-d_new.values(), g, "f32")
    update.close()
    for v in (d_g, d_w, d_new):
        v.free()
    ctx.close()


def test_graph_of_a_step():
    rng = np.random.default_rng(4)
    g, w, m = (to_type(rng.standard_normal((130, 200)), "f32") for _ in range(3))
    ctx = context()
    update = operators.OrthogonalUpdate(ctx, 130, 200)
    d = [Matrix(ctx, v, "f32") for v in (g, w, m)]
    new = [Matrix(ctx, None, "f32", shape=g.shape) for _ in range(2)]
    check_replays(ctx, lambda: update.step(d[0], d[1], new[0], momentum=d[2], new_momentum=new[1]),
                  lambda: [v.values() for v in new])
    update.close()
    for v in (*d, *new):
        v.free()
    ctx.close()
