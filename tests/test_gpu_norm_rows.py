"""A layer norm made for many rows, called with fewer: all results of the rows
that a call has, and nothing behind them."""
import numpy as np
import pytest

from test_gpu_norm import Case, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,type", [(7, "f32"), (100, "bf16"), (260, "f32"), (1500, "f16"), (5000, "bf16"), (9000, "f32")])
def test_calls_of_fewer_rows(n, type):
    """In turn: arrays as large as the most rows' hold what the call before left
    behind the rows of a smaller one. mean and rstd too, whose arrays lie alone."""
    most = 600
    rng = np.random.default_rng(n)
    x, w, b, dy = make(rng, most, n, type, type)
    all_rows = Case(x, w, b, dy, type, type)
    d = all_rows.d
    whole = {name: d[name].at for name in ("x", "y", "dy", "dx", "mean", "rstd")}
    for rows in (most, 1, 17, 599, 300):
        print(f"{rows} x {n} {type}", flush=True)
        before = {name: d[name].buffer.numpy() for name in ("y", "dx", "mean", "rstd")}
        for name, at in whole.items():
            d[name].shape = (rows, n) if name in ("x", "y", "dy", "dx") else (rows,)
        all_rows.forward()
        all_rows.backward()
        for name in before:  # behind the rows
            end = rows * n if name in ("y", "dx") else rows
            assert np.array_equal(d[name].buffer.numpy()[end:], before[name][end:]), name
        # the rows themselves, by the checks of a case of their number
        part = Case.__new__(Case)
        part.x, part.w, part.b, part.dy, part.type, part.out, part.eps = x[:rows], w, b, dy[:rows], type, type, all_rows.eps
        part.d = d

        def value(name):
            v = d[name]
            if name not in whole:
                return v.values()
            shape, v.shape = v.shape, (most, n) if name in ("x", "y", "dy", "dx") else (1, most)
            v.host = v.buffer.numpy()  # what lies around is compared above
            have = v.values()
            v.shape = shape
            return have[:rows] if have.shape[0] == most else have[0, :rows]

        part.value = value
        part.check()
        mean = part.x.mean(1)
        assert (np.abs(value("mean") - mean) <= 100 * 2.0**-24 * np.abs(part.x).mean(1) + 2.0**-24 * np.abs(mean)).all()
    all_rows.close()
