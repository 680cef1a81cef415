"""The orthogonal update of gradients whose rows or columns differ in size, as
those of seldom used embeddings do: the small ones' values are far below the
largest one's, and the steps multiply them by up to 485.

Tolerance: close_to's, four times the distance that the same steps have in 32
bits, as values are held to 22 bits instead of 24, and 2^-22 of the size. It
needs the 22 bits at every size that counts: with a spacing of d for small
values the result is off by about 485 d / 3.5 sqrt(rows cols), which at 1,024 x
1,024 is 1.6e-8 for d = 2^-43 and 1.6e-5 for 2^-33."""
import numpy as np
import pytest

from operator_checks import context, to_type
from test_gpu_orthogonal import close_to, run, steps_of

pytestmark = pytest.mark.gpu

# each kernel of the products; see UPDATES in dense_stack_shapes
SHAPES = [(100, 300), (200, 330), (768, 760), (900, 880), (1300, 1000), (1500, 1450), (1400, 2600)]


def graded(rng, rows, cols, kind, small):
    """One large row, one large column, or rows of all sizes down to `small`."""
    g = rng.standard_normal((rows, cols))
    if kind == "row":
        g[1:] *= small
    elif kind == "column":
        g[:, 1:] *= small
    else:
        g *= small ** rng.random((rows, 1))
    return to_type(1e-3 * g, "f32")


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("kind", ["row", "column", "all sizes"])
def test_rows_and_columns_of_different_sizes(rows, cols, kind):
    ctx = context()
    for small in (1e-3, 1e-5) if rows < 1000 else (1e-4,):
        g = graded(np.random.default_rng(rows + cols), rows, cols, kind, small)
        print(f"{rows} x {cols} {kind} {small}", flush=True)
        close_to(run(ctx, g, "f32", "f32"), g, "f32")
    ctx.close()


@pytest.mark.parametrize("rows,cols", [(1, 5), (100, 300), (200, 330), (600, 640)])
def test_singular_values_up_to_the_documented_size(rows, cols):
    """A gradient of rank one, whose singular value of 1 becomes 15 after a step,
    so that A is 225 in the next, and B up to 250 in size. Each of X, A and B has
    the errors of a few roundings of 2^-22 of its size, 4 taken here, and the
    result a X + B X those of the three: 4 2^-22 of |a s| + 3 |B s|."""
    rng = np.random.default_rng(rows)
    left, right = rng.standard_normal(rows), rng.standard_normal(cols)
    g = to_type(np.outer(left / np.linalg.norm(left), right / np.linalg.norm(right)), "f32")
    ctx = context()
    for steps, abc in ((2, (15.0, 0.0, 0.0)), (2, (15.5, -0.5, 0.0)), (1, (10.0, -250.0, 0.0))):
        a, b, _ = abc
        s = 1.0 if steps == 1 else a + b  # before the last step
        have = run(ctx, g, "f32", "f32", steps=steps, coefficients=abc)
        off = 4 * 2.0**-22 * (abs(a * s) + 3 * abs(b * s**3)) + (steps - 1) * 4 * 2.0**-22 * abs(a + 3 * b * s**2) * s
        assert np.linalg.norm(have - steps_of(g, np.float64, steps, abc)) <= off
    ctx.close()
