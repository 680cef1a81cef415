"""GELU's own error, on layers whose sums are the weights themselves.

Tolerances. The function of a 16-bit result is within 2^-18 of its size to -6,
so that the result is within that of the nearest 16-bit value."""
import numpy as np
import pytest

from operator_checks import BITS, context, linear, to_type
from test_gpu_linear import release, run_forward

pytestmark = pytest.mark.gpu


def gelu(z, type, out, rows):
    ctx = context()
    layer, d = run_forward(ctx, np.ones((rows, 1)), z[:, None], None, None, type, out, "gelu", False)
    have = d["y"].values()[-1]
    release(ctx, layer, d)
    ctx.close()
    return have, linear(np.ones((1, 1)), z[:, None], None, None, "gelu", False)[4][0]


@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40])
def test_results_of_16_bits_are_rounded_once(type, rows):
    z = np.unique(to_type(np.linspace(-6, 8, 20001), type))
    have, want = gelu(z, type, type, rows)
    size = np.abs(want)
    least = 2.0**-25 if type == "f16" else 0.0
    assert (np.abs(have - want) <= (2.0**-BITS[type] + 2.0**-18) * size + least).all()
