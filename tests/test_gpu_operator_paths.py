"""The operators on the kernels of operator_shapes. Layers of small whole
numbers: every sum is exact in 32 bits, so results are the reference's rounded
once, to the bit; a wrong element anywhere shows."""
import numpy as np
import pytest

from operator_checks import Array, Matrix, context, to_type
from operator_shapes import GRADIENTS, LARGE, LAYERS, NORMALIZED, WALKS
from test_gpu_linear import release, run_forward, test_forward as check_forward
from test_gpu_token_cache import Cache, corpus, quantise, spread

pytestmark = pytest.mark.gpu


def whole(rng, shape, most=1):
    return rng.integers(-most, most + 1, shape).astype(np.float32)


@pytest.mark.parametrize("rows,k,n,type,kernel,odd", LAYERS)
def test_layers(rows, k, n, type, kernel, odd):
    rng = np.random.default_rng(rows)
    print(f"{rows} x {k} -> {n} {type}", flush=True)
    x, w, b, r = whole(rng, (rows, k)), whole(rng, (n, k)), whole(rng, n, 3), whole(rng, (rows, n), 3)
    z = x @ w.T + b
    ctx = context()
    for residual, act in ((r, "relu"), (None, "none")):
        # X's and W's rows as they lie; those of Y, the saved sums and the residual apart where odd
        layer, d = run_forward(ctx, x, w, b, residual, type, type, act, False, (0, 0, 3 if odd else 0), 0, training=True)
        h = (np.maximum(z, 0) if act == "relu" else z) + (0 if residual is None else residual)
        assert np.array_equal(d["y"].values(), to_type(h, type))
        if act == "relu":
            assert np.array_equal(d["saved"].values(), to_type(z, type))
        release(ctx, layer, d)
    layer, d = run_forward(ctx, x, w, b, r, type, "f32", "none", False, (0, 0, 1 if odd else 0), 1 if odd else 0)
    assert np.array_equal(d["y"].values(), z + r)
    release(ctx, layer, d)
    ctx.close()


@pytest.mark.parametrize("rows,k,n,type,kernel", NORMALIZED)
def test_normalized_layers(rows, k, n, type, kernel):
    check_forward(rows, k, n, type, "f32", "silu", True, True, True, (0, 0, 2), 0)


@pytest.mark.parametrize("rows,k,n,type,dx,dw,joined", GRADIENTS)
def test_gradients(rows, k, n, type, dx, dw, joined):
    rng = np.random.default_rng(rows + 1)
    print(f"{rows} x {k} -> {n} {type}", flush=True)
    x, w, dy = whole(rng, (rows, k)), whole(rng, (n, k)), whole(rng, (rows, n))
    z = x @ w.T
    dz = dy * (z > 0)
    want = {"dx": dz @ w, "dw": dz.T @ x, "db": dz.sum(0, dtype=np.float64)[None]}
    ctx = context()
    # dY read through the slope, with bias gradients, then as it lies
    layer, d = run_forward(ctx, x, w, None, None, type, type, "relu", False, training=True)
    g = {"dy": Matrix(ctx, dy, type), "dx": Matrix(ctx, None, type, 3, 1, shape=(rows, k)),
         "dw": Matrix(ctx, None, type, 1, 0, shape=(n, k)), "db": Matrix(ctx, None, type, shape=(1, n))}
    g["db"].shape = (n,)
    layer.backward(d["x"], g["dy"], saved=d["saved"], dx=g["dx"], dweight=g["dw"], dbias=g["db"])
    for name in ("dx", "dw", "db"):
        assert np.array_equal(g[name].values().reshape(want[name].shape), to_type(want[name], type)), name
    release(ctx, layer, {**d, **{m: g[m] for m in ("dx", "dw", "db")}})
    layer, d = run_forward(ctx, x, w, None, None, type, type, "none", False, training=True)
    out = {"dx": Matrix(ctx, None, type, shape=(rows, k)), "dw": Matrix(ctx, None, type, shape=(n, k))}
    layer.backward(d["x"], g["dy"], dx=out["dx"], dweight=out["dw"])
    assert np.array_equal(out["dx"].values(), to_type(dy @ w, type))
    assert np.array_equal(out["dw"].values(), to_type(dy.T @ x, type))
    release(ctx, layer, {**d, **out, "dy": g["dy"]})
    ctx.close()


@pytest.mark.parametrize("format,type,nq,q_len,cap,items", WALKS)
def test_waves_that_walk_documents(format, type, nq, q_len, cap, items):
    """Documents of no, one and several tiles, absent ids between them, and
    the best k of more candidates than the sort's smallest block takes."""
    rng = np.random.default_rng(nq * cap)
    print(f"{nq} queries of {q_len}, {cap} candidates, {format}", flush=True)
    lens = np.array([0, 1, 31, 32, 33, 64, 65, 100, 7, 0, 300, 128, 2, 40], np.int32)
    page, dim, group = 16, 128, 64
    start, pages, slots, total = corpus(rng, lens, page)
    ctx = context()
    c = Cache(ctx, total * page, format, dim, group, page)
    x = rng.standard_normal((total * page, dim)).astype(np.float32)
    rows, at = Matrix(ctx, x, "f32"), Array(ctx, np.arange(total * page))
    c.cache.write(rows, at)
    _, s, value = quantise(x, format, group)
    tokens = spread(value, s, group, dim).astype(np.float64)
    q = to_type(rng.standard_normal((nq, q_len, dim)), type)
    q_lens = rng.integers(0, q_len + 1, nq).astype(np.int32)
    q_lens[0] = q_len
    ids = rng.integers(-1, lens.size + 1, (nq, cap)).astype(np.int32)
    ids[1] = -1  # nothing to score
    ids[2, 5:] = -1
    counts = np.full(nq, cap, np.int32)
    counts[-1] = cap - 70
    by_doc = np.full((nq, lens.size + 2), -np.inf)  # the last two: no documents
    for d, where in enumerate(slots):
        if len(where):
            best = (q.reshape(-1, dim) @ tokens[where].T).max(1).reshape(nq, q_len)
            by_doc[:, d] = np.where(np.arange(q_len) < q_lens[:, None], best, 0).sum(1)
    want = np.take_along_axis(by_doc, ids, 1)  # -1 is the last entry
    want[-1, counts[-1]:] = -np.inf
    k = min(cap, 50)
    dev = [Matrix(ctx, q, type), Array(ctx, start), Array(ctx, lens), Array(ctx, pages), Array(ctx, ids),
           Matrix(ctx, None, "f32", shape=(nq, cap)), Array(ctx, q_lens), Array(ctx, counts),
           Array(ctx, np.zeros((nq, k), np.int64)), Array(ctx, np.zeros((nq, k), np.float32)), Array(ctx, np.zeros(nq, np.int32))]
    c.cache.maxsim(*dev[:4], int(lens.max()), dev[4], dev[5], query_lens=dev[6], cand_counts=dev[7], k=k, top_ids=dev[8],
                   top_scores=dev[9], top_counts=dev[10])
    have = dev[5].values()
    assert np.array_equal(np.isneginf(have), np.isneginf(want))
    fin = np.isfinite(want)
    # 2^-20 |q||x| a token
    bound = q_len * 2.0**-20 * np.linalg.norm(q, axis=2).max() * np.linalg.norm(tokens, axis=1).max()
    assert np.abs(have[fin] - want[fin]).max() <= bound
    top, top_scores = dev[8].numpy(), dev[9].numpy()
    assert np.array_equal(dev[10].numpy(), np.minimum(k, counts))
    for i in range(nq):
        order = np.lexsort((-ids[i, :counts[i]].astype(np.int64), -have[i, :counts[i]]))[:k]
        assert np.array_equal(top[i], ids[i, order])
        assert np.array_equal(top_scores[i].astype(np.float64), have[i, order])
    for v in (rows, at, c, *dev):
        v.free()
    ctx.close()


@pytest.mark.parametrize("type,format,dim,n", LARGE)
def test_rows_past_the_caches(type, format, dim, n):
    rng = np.random.default_rng(n)
    print(f"{n} rows of {dim} {type}, {format}", flush=True)
    ctx = context()
    c = Cache(ctx, (n + 40) // 16 * 16, format, dim, 128)
    x = to_type(rng.standard_normal((n, dim), np.float32), type).astype(np.float32)
    where = rng.permutation(c.host_codes.shape[0])[:n].astype(np.int64)
    rows, at, out = Matrix(ctx, x, type), Array(ctx, where), Matrix(ctx, None, type, shape=(n, dim))
    c.cache.write(rows, at)
    c.cache.read(at, out)
    bits, scales, value = quantise(x, format, 128)
    want_codes, want_scales = c.host_codes.copy(), c.host_scales.copy()
    want_codes[where], want_scales[where] = bits, scales
    have = c.codes.numpy()
    if format == "fp8":  # -0 and 0 are the same value
        have, want_codes = np.where(have == 128, 0, have), np.where(want_codes == 128, 0, want_codes)
    assert np.array_equal(have, want_codes) and np.array_equal(c.scales.numpy(), want_scales)
    assert np.array_equal(out.values(), to_type(spread(value, scales, 128, dim), type))
    for v in (rows, at, out, c):
        v.free()
    ctx.close()
