"""4-bit rows of so many blocks that they take two launches, bit for bit."""
from types import SimpleNamespace

import numpy as np
import pytest

from chimera_amd import operators
from mx4_checks import quantise, without_signs_of_zeros
from operator_checks import bf16_bits, context, from_bf16, to_type

pytestmark = pytest.mark.gpu


def test_rows_past_a_launch():
    """Two values a row, three apart, in 2^20 blocks of 32 rows and three more.
    The same 101 rows over and over, which no launch's are a multiple of."""
    rows, n, period = (1 << 25) + 70, 2, 101
    rng = np.random.default_rng(1)
    few = to_type(rng.standard_normal((period, n)), "bf16")
    codes, scales, values = quantise(few)
    x = np.full((period, n + 1), 0x7FC1, np.uint16)
    x[:, :n] = bf16_bits(few)
    ctx = context()
    d_x, d_out = ctx.to_device(np.resize(x, (rows, n + 1))), ctx.to_device(np.full((rows, n + 1), 0x7FC1, np.uint16))
    d_codes, d_scales = ctx.to_device(np.full((rows + 1, 16), 0xEE, np.uint8)), ctx.to_device(np.full((rows + 1, 8), 0xEE, np.uint8))
    matrix = lambda d: SimpleNamespace(ptr=d.ptr, shape=(rows, n), dtype="bf16", stride=n + 1)
    array = lambda d, wide: SimpleNamespace(ptr=d.ptr, shape=(rows, wide), dtype=np.dtype(np.uint8))
    c, s = array(d_codes, 16), array(d_scales, 8)
    operators.mx4_quantise(ctx, matrix(d_x), c, s)
    operators.mx4_read(ctx, c, s, matrix(d_out))

    def repeats(have, want):
        whole = rows // period * period
        assert np.array_equal(have[:whole].reshape(-1, *want.shape), np.broadcast_to(want, (whole // period, *want.shape)))
        assert np.array_equal(have[whole:rows], want[:rows - whole])

    have = d_codes.numpy()
    assert (have[rows] == 0xEE).all()
    repeats(without_signs_of_zeros(have), without_signs_of_zeros(codes))
    have = d_scales.numpy()
    assert (have[rows] == 0xEE).all()
    repeats(have[:, :1], scales[:, :1])
    out = d_out.numpy()
    assert (out[:, n] == 0x7FC1).all()
    repeats(from_bf16(out[:, :n]), values.astype(np.float32))
    for d in (d_x, d_out, d_codes, d_scales):
        d.free()
    ctx.close()
