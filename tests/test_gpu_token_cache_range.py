"""Queries of any size that 32 bits hold."""
import numpy as np
import pytest

from operator_checks import Array, Matrix, context, to_type
from test_gpu_token_cache import Cache, corpus, quantise, spread

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("split", [False, True])
def test_the_largest_and_the_least_queries(type, split):
    """Tokens of up to 2^127 and down to 2^-125 against documents whose values bring
    the products back: each score within 2^-20 |q||x| of a token, and 2^-126
    where a sum falls out of the normal numbers."""
    rng = np.random.default_rng(31)
    page, dim, q_len = 16, 128, 5
    lens = np.array([40, 700 if split else 33, 3], np.int32)
    start, pages, slots, total = corpus(rng, lens, page)
    ctx = context()
    c = Cache(ctx, total * page, "int8", dim, 64, page)
    exponents = np.array([127, 118, 90, -90, -118, -125])
    unit = rng.standard_normal((exponents.size, q_len, dim))
    unit /= np.abs(unit).max(2, keepdims=True)
    q = to_type(unit * 2.0**exponents[:, None, None], type)
    rows, at = Matrix(ctx, rng.standard_normal((total * page, dim)) * 2.0**-7, "f32"), Array(ctx, np.arange(total * page))
    c.cache.write(rows, at)
    _, s, value = quantise(rows.values().astype(np.float32), "int8", 64)
    tokens = spread(value, s, 64, dim).astype(np.float64)
    ids = np.tile(np.arange(3, dtype=np.int32), (exponents.size, 1))
    dev = [Matrix(ctx, q, type), Array(ctx, start), Array(ctx, lens), Array(ctx, pages), Array(ctx, ids),
           Matrix(ctx, None, "f32", shape=ids.shape)]
    c.cache.maxsim(*dev[:4], int(lens.max()), dev[4], dev[5])
    have = dev[5].values()
    for i in range(exponents.size):
        for d in range(3):
            want = (q[i] @ tokens[slots[d]].T).max(1).sum()
            off = q_len * 2.0**-20 * np.linalg.norm(q[i], axis=1).max() * np.linalg.norm(tokens, axis=1).max()
            assert abs(have[i, d] - want) <= off + q_len * 2.0**-126, (exponents[i], d)
    for v in (rows, at, c, *dev):
        v.free()
    ctx.close()
