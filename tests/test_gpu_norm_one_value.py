"""Layer norm of rows whose values are equal, or a few units in the last place
apart: the mean's own rounding is as large as what is left of the row, or larger
than sqrt(eps). Their statistics, results and gradients are those of the
definition, within the tolerances of test_gpu_norm, which have no term for it."""
import numpy as np
import pytest

from operator_checks import to_type
from test_gpu_norm import Case, make

pytestmark = pytest.mark.gpu


def steps_of(v, type):
    """The distance of v from its neighbours in the type."""
    if type == "bf16":
        return 2.0 ** (np.floor(np.log2(np.abs(v))) - 7)
    return np.abs(np.spacing(np.asarray(v, np.float16 if type == "f16" else np.float32))).astype(np.float64)


def check(x, type, out, eps, pad=0):
    rng = np.random.default_rng(x.size)
    _, w, b, dy = make(rng, *x.shape, type, out)
    c = Case(to_type(x, type), w, b, dy, type, out, pad=pad, eps=eps)
    c.forward()
    c.backward()
    c.check()
    c.close()


VALUES = {"f32": [1.0, 12345.678, 1e6 / 3, -3e6, 1e8, 123456789.0, -7e9, 1e15 / 7, 1.7e19, -1e-3], "f16": [1.0, 60000.0, -3.3, 0.1],
          "bf16": [1.0, 1e8, -3e6, 1e15, 0.3]}
# gradients of f16 end at 65,504, and rstd is 1e6 and more with the smaller ones
EPS = {"f32": (1e-5, 1e-12, 1e-30), "f16": (1e-5,), "bf16": (1e-5, 1e-12, 1e-30)}


@pytest.mark.parametrize("type,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("n", [5, 96, 300, 1000, 3000, 7001, 9001, 30_000])
def test_rows_of_one_value(n, type, out):
    values = to_type(np.array(VALUES[type]), type)
    print(f"{n} {type}", flush=True)
    for eps in EPS[type]:
        check(np.repeat(values[:, None], n, 1), type, out, eps, pad=n % 2)


@pytest.mark.parametrize("type,out", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("n", [24, 96, 300, 1000, 3000, 7001, 9001, 30_000])
def test_rows_of_neighbouring_values(n, type, out):
    """A value and its neighbours, and rows in which one column differs."""
    rng = np.random.default_rng(n)
    values = to_type(np.array([v for v in VALUES[type] if abs(v) < 1e10]), type)[:, None]
    step = steps_of(values, type)
    few, one = rng.integers(-1, 3, (values.size, n)), np.zeros((values.size, n))
    one[:, n // 3] = 1
    print(f"{n} {type}", flush=True)
    for eps in EPS[type][:2]:
        check(np.concatenate([values + step * few, values + step * one]), type, out, eps)
