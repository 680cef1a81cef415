"""The quantised token cache: codes and scales bit for bit against the
documented arithmetic in numpy, what is read back, and late interaction on it
against 64 bits. A product may be off by 2^-20 |q||x| (a query's two fp16
parts keep 22 bits, sums are 32-bit), so a score by that times the query's
tokens."""
import numpy as np
import pytest

from chimera_amd import operators
from operator_checks import Array, Matrix, context, raw, to_type

pytestmark = pytest.mark.gpu

TOP = {"int8": 127.0, "int4": 7.0, "fp8": 448.0}
# e4m3 values of the bytes 0..126
E4M3 = np.array([(m / 8 * 2.0**-6) if e == 0 else (1 + m / 8) * 2.0**(e - 7) for e in range(16) for m in range(8)][:127])


def e4m3_bits(v):
    """Nearest even e4m3 byte of |v| <= 448."""
    a = np.abs(v).astype(np.float64)
    hi = np.searchsorted(E4M3, a).clip(0, 126)
    lo = (hi - 1).clip(0)
    up, down = E4M3[hi] - a, a - E4M3[lo]
    pick = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    return (pick | np.where(np.signbit(v), 0x80, 0)).astype(np.uint8)


def quantise(x, format, group):
    """(bytes, scales, code values) of rows [n, dim], float32 arithmetic."""
    n, dim = x.shape
    groups = -(-dim // group)
    wide = -(-dim // 32) * 32
    x = x.astype(np.float32)
    codes = np.zeros((n, groups * 128), np.float32)
    scales = np.zeros((n, groups), np.float32)
    top = np.float32(TOP[format])
    with np.errstate(all="ignore"):
        for g in range(groups):
            part = x[:, g * group:(g + 1) * group]
            most = np.abs(part).max(1)
            bad = ~np.isfinite(part).all(1)
            zero = bad | (most < np.float32(2.0**-117))
            inv = np.where(zero, np.float32(0), top * (np.float32(1) / most)).astype(np.float32)
            scales[:, g] = np.where(bad, np.float32(np.nan), np.where(zero, np.float32(0), most * (np.float32(1) / top)))
            v = np.where(zero[:, None], np.float32(0), part * inv[:, None])
            v = np.clip(v if format == "fp8" else np.rint(v), -top, top)
            codes[:, g * group:g * group + part.shape[1]] = v
    codes = codes[:, :wide]
    if format == "fp8":
        b = e4m3_bits(codes)
        value = np.where(b >= 128, -1.0, 1.0) * E4M3[b & 127]
        return b, scales, value[:, :dim]
    if format == "int8":
        return codes.astype(np.int8).view(np.uint8), scales, codes[:, :dim].astype(np.float64)
    u = (codes + 8).astype(np.uint8)
    return u[:, 0::2] | (u[:, 1::2] << 4), scales, codes[:, :dim].astype(np.float64)


def spread(values, scales, group, dim):
    """code * scale in float32."""
    with np.errstate(invalid="ignore"):
        return (values.astype(np.float32) * np.repeat(scales, group, 1)[:, :dim]).astype(np.float32)


class Cache:
    def __init__(self, ctx, slots, format, dim, group, page=16):
        row, groups = operators.cache_row(format, dim, group)
        rng = np.random.default_rng(99)
        self.host_codes = rng.integers(0, 256, (slots, row)).astype(np.uint8)
        self.host_scales = np.full((slots, groups), 7.5, np.float32)
        self.codes, self.scales = Array(ctx, self.host_codes), Array(ctx, self.host_scales)
        self.cache = operators.TokenCache(ctx, self.codes, self.scales, format, dim, group, page)

    def free(self):
        self.cache.close()
        self.codes.free()
        self.scales.free()


def special_rows(rng, n, dim):
    x = rng.standard_normal((n, dim)).astype(np.float32) * np.exp(rng.uniform(-20, 20, (n, 1))).astype(np.float32)
    x[0] = 0
    if n > 8:
        x[1, dim // 2] = np.nan
        x[2, 0] = np.inf
        x[3] = 2.0**-130
        x[4] = np.float32(3e38)
        x[5] = np.tile([1.0, -1.0, 0.5, -0.5], 32)[:dim]  # codes at ties
        x[6, :] = -1.0
        x[7] = 2.0**-117
    return x


@pytest.mark.parametrize("format", ["int8", "int4", "fp8"])
@pytest.mark.parametrize("dim,group,type,pad,shift", [(128, 128, "f32", 0, 0), (128, 32, "bf16", 0, 0),
                                                      (96, 64, "f16", 8, 0), (100, 32, "f32", 1, 1), (1, 32, "f32", 0, 0),
                                                      (37, 128, "bf16", 3, 1), (64, 64, "f16", 0, 0)])
def test_write_and_read(format, dim, group, type, pad, shift):
    rng = np.random.default_rng(dim + group)
    n, slots = 101, 192
    x = special_rows(rng, n, dim)
    if type == "f16":
        x = np.where(np.abs(x) > 60000, np.sign(x) * 60000, x)
        x[2, 0] = np.inf
    x = to_type(x, type).astype(np.float32)
    where = rng.permutation(slots)[:n].astype(np.int64)
    where[10], where[11] = -1, slots  # outside: skipped, and read as zeros
    ctx = context()
    c = Cache(ctx, slots, format, dim, group)
    rows, at = Matrix(ctx, x, type, pad, shift), Array(ctx, where)
    c.cache.write(rows, at)
    bits, scales, value = quantise(x, format, group)
    ok = (where >= 0) & (where < slots)
    want_codes, want_scales = c.host_codes.copy(), c.host_scales.copy()
    want_codes[where[ok]], want_scales[where[ok]] = bits[ok], scales[ok]
    have = c.codes.numpy()
    if format == "fp8":  # -0 and 0 are the same value
        have, want_codes = np.where(have == 128, 0, have), np.where(want_codes == 128, 0, want_codes)
    assert np.array_equal(have, want_codes)
    assert np.array_equal(c.scales.numpy(), want_scales, equal_nan=True)
    with np.errstate(over="ignore", invalid="ignore"):
        want = to_type(spread(value, scales, group, dim), type)
    want[~ok] = 0
    out = Matrix(ctx, None, type, pad, shift, shape=(n, dim))
    c.cache.read(at, out)
    assert np.array_equal(out.values(), want, equal_nan=True)
    for v in (rows, at, out, c):
        v.free()
    ctx.close()


def test_one_token_and_none():
    ctx = context()
    c = Cache(ctx, 16, "int8", 128, 128)
    x = np.random.default_rng(0).standard_normal((1, 128)).astype(np.float32)
    rows, at, out = Matrix(ctx, x, "f32"), Array(ctx, np.array([15])), Matrix(ctx, None, "f32", shape=(1, 128))
    c.cache.write(rows, at)
    c.cache.read(at, out)
    bits, scales, value = quantise(x, "int8", 128)
    assert np.array_equal(out.values(), spread(value, scales, 128, 128))
    rows.shape = out.shape = (0, 128)
    at.shape = (0,)
    c.cache.write(rows, at)
    c.cache.read(at, out)
    for v in (rows, at, out, c):
        v.free()
    ctx.close()


def test_offsets_past_32_bits():
    """Slots whose codes lie past 4 GiB, written, read and scored."""
    ctx = context()
    slots, dim, page = 34_000_000, 128, 32
    codes, scales = ctx.empty((slots, 128), np.uint8), ctx.empty((slots, 4), np.float32)
    cache = operators.TokenCache(ctx, codes, scales, "int8", dim, 32, page)
    rng = np.random.default_rng(2)
    x = rng.standard_normal((64, dim)).astype(np.float32)
    pages = np.array([slots // page - 1, slots // page - 7], np.int32)
    where = (pages[:, None].astype(np.int64) * page + np.arange(page)).ravel()
    rows, at, out = Matrix(ctx, x, "f32"), Array(ctx, where), Matrix(ctx, None, "f32", shape=(64, dim))
    cache.write(rows, at)
    cache.read(at, out)
    _, s, value = quantise(x, "int8", 32)
    tokens = spread(value, s, 32, dim).astype(np.float64)
    assert np.array_equal(out.values(), tokens)
    q = rng.standard_normal((1, 5, dim))
    dq = Matrix(ctx, q, "f32")
    dev = [Array(ctx, v) for v in (np.array([0], np.int64), np.array([50], np.int32), pages, np.array([[0]], np.int32))]
    scores = Matrix(ctx, None, "f32", shape=(1, 1))
    cache.maxsim(dq, dev[0], dev[1], dev[2], 50, dev[3], scores)
    want = (to_type(q, "f32")[0] @ tokens[:50].T).max(1).sum()
    assert abs(scores.values()[0, 0] - want) <= 5 * 2.0**-20 * np.linalg.norm(q, axis=2).max() * np.linalg.norm(tokens, axis=1).max()
    cache.close()
    for v in (rows, at, out, dq, scores, codes, scales, *dev):
        v.free()
    ctx.close()




def corpus(rng, lens, page, spare=5):
    """Pages of the documents in no order: (page_start, pages, slots of every
    token, number of pages)."""
    owned = -(-lens.astype(np.int64) // page)
    start = np.concatenate([[0], np.cumsum(owned)])[:-1]
    total = int(owned.sum()) + spare
    pages = rng.permutation(total)[: total - spare].astype(np.int32)
    slots = [pages[s + np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page for s, n in zip(start, lens)]
    return start, pages, slots, total


def reference(queries, q_lens, tokens, slots, ids, counts):
    out = np.full(ids.shape, -np.inf)
    for q in range(ids.shape[0]):
        for j in range(min(ids.shape[1], counts[q])):
            d = ids[q, j]
            if 0 <= d < len(slots) and len(slots[d]):
                p = queries[q, :q_lens[q]] @ tokens[slots[d]].T
                out[q, j] = np.where(np.isnan(p), -np.inf, p).max(1).sum()
    return out


MAXSIM = [
    # format, dim, group, page, type, nq, query_len, lens, cap
    ("int8", 128, 128, 16, "f32", 3, 32, [0, 1, 15, 16, 17, 31, 32, 33, 64, 100, 129, 300], 20),
    ("int8", 128, 32, 8, "bf16", 2, 32, [5, 40, 0, 77], 7),
    ("int4", 96, 32, 32, "f16", 2, 19, [1, 2, 33, 200, 63], 9),
    ("int4", 100, 64, 1, "f32", 1, 1, [3, 50, 0, 31], 6),
    ("fp8", 48, 64, 64, "f32", 2, 33, [70, 1, 0, 130], 5),
    ("fp8", 128, 64, 256, "bf16", 1, 70, [300, 257, 255, 1], 4),
    ("int8", 1, 32, 4, "f32", 1, 3, [9, 1], 3),
    # few documents, long ones: split and joined
    ("int8", 128, 128, 16, "f32", 1, 32, [5000, 1, 0, 3100, 129], 5),
    ("int4", 128, 32, 64, "bf16", 2, 45, [2500, 4099, 128], 4),
    ("fp8", 64, 32, 2, "f16", 1, 7, [1000, 0, 640], 3),
    # many candidates
    ("int8", 64, 64, 16, "f32", 40, 16, [10, 40, 90, 33], 300),
]


@pytest.mark.parametrize("format,dim,group,page,type,nq,q_len,lens,cap", MAXSIM)
def test_maxsim(format, dim, group, page, type, nq, q_len, lens, cap):
    rng = np.random.default_rng(dim * q_len + nq)
    lens = np.array(lens, np.int32)
    start, pages, slots, total = corpus(rng, lens, page)
    ctx = context()
    c = Cache(ctx, total * page, format, dim, group, page)
    x = rng.standard_normal((total * page, dim)).astype(np.float32)
    x /= np.linalg.norm(x, axis=1, keepdims=True)
    if len(slots[-1]):
        x[slots[-1][0]] = np.nan  # a cached row that was not finite
    rows, at = Matrix(ctx, x, "f32"), Array(ctx, np.arange(total * page))
    c.cache.write(rows, at)
    _, s, value = quantise(x, format, group)
    tokens = spread(value, s, group, dim).astype(np.float64)
    q = to_type(rng.standard_normal((nq, q_len, dim)) * np.exp(rng.uniform(-3, 3, (nq, q_len, 1))), type)
    q_lens = rng.integers(1, q_len + 1, nq).astype(np.int32)
    q_lens[0] = q_len
    ids = rng.integers(-1, lens.size + 1, (nq, cap)).astype(np.int32)
    ids[0, :min(cap, lens.size)] = np.arange(lens.size)[:cap]
    counts = np.full(nq, cap, np.int32)
    counts[-1] = max(1, cap - 2)
    print(f"{format} {dim} {type}, {nq} queries of {q_len}", flush=True)
    dev = {"q": Matrix(ctx, q, type), "start": Array(ctx, start), "lens": Array(ctx, lens), "pages": Array(ctx, pages),
           "ids": Array(ctx, ids), "scores": Matrix(ctx, None, "f32", shape=(nq, cap)), "ql": Array(ctx, q_lens),
           "counts": Array(ctx, counts)}
    bound = q_len * 2.0**-20 * np.linalg.norm(q, axis=2).max() * np.nanmax(np.linalg.norm(tokens, axis=1))
    longest = int(lens.max())

    def score(k=0, **more):
        c.cache.maxsim(dev["q"], dev["start"], dev["lens"], dev["pages"], longest, dev["ids"], dev["scores"], k=k, **more)
        return dev["scores"].values()

    for q_all, n_all in ((False, True), (True, False)):
        want = reference(q, np.full(nq, q_len) if q_all else q_lens, tokens, slots, ids,
                         np.full(nq, cap) if n_all else counts)
        have = score(query_lens=None if q_all else dev["ql"], cand_counts=None if n_all else dev["counts"])
        assert np.array_equal(np.isneginf(have), np.isneginf(want))
        fin = np.isfinite(want)
        assert np.abs(have[fin] - want[fin]).max(initial=0.0) <= bound
    # the best k: by the scores just returned, ties to the larger id
    k = 3
    top = {"ids": Array(ctx, np.zeros((nq, k), np.int64)), "scores": Array(ctx, np.zeros((nq, k), np.float32)),
           "counts": Array(ctx, np.zeros(nq, np.int32))}
    have = score(k=k, cand_counts=dev["counts"], top_ids=top["ids"], top_scores=top["scores"], top_counts=top["counts"])
    for i in range(nq):
        n = min(k, counts[i])
        order = sorted(range(counts[i]), key=lambda j: (-have[i, j], -ids[i, j]))[:n]
        assert top["counts"].numpy()[i] == n
        assert np.array_equal(top["scores"].numpy()[i, :n].astype(np.float64), have[i, order])
        assert np.array_equal(top["ids"].numpy()[i, :n], ids[i, order])
    for v in (rows, at, c, *dev.values(), *top.values()):
        v.free()
    ctx.close()


@pytest.mark.parametrize("format", ["int8", "int4", "fp8"])
@pytest.mark.parametrize("type", ["f32", "f16"])
def test_maxsim_keeps_32_bits(format, type):
    """Single tokens against single documents of one token: the error is that
    of a sum of 128 products in 32 bits in about eight joins, and of a query in
    two halves of 11 bits. Both are near 2^-24 of a sum's size; 2^-22 over the
    mean square."""
    rng = np.random.default_rng(17)
    n, dim = 2048, 128
    start, pages, slots, total = corpus(rng, np.ones(n, np.int32), 8)
    ctx = context()
    c = Cache(ctx, total * 8, format, dim, 32, 8)
    x = rng.standard_normal((total * 8, dim)).astype(np.float32)
    rows, at = Matrix(ctx, x, "f32"), Array(ctx, np.arange(total * 8))
    c.cache.write(rows, at)
    _, s, value = quantise(x, format, 32)
    tokens = spread(value, s, 32, dim).astype(np.float64)
    q = to_type(rng.standard_normal((2, 1, dim)), type)
    ids = np.tile(np.arange(n, dtype=np.int32), (2, 1))
    dev = {"q": Matrix(ctx, q, type), "start": Array(ctx, start), "lens": Array(ctx, np.ones(n, np.int32)),
           "pages": Array(ctx, pages), "ids": Array(ctx, ids), "scores": Matrix(ctx, None, "f32", shape=(2, n))}
    c.cache.maxsim(dev["q"], dev["start"], dev["lens"], dev["pages"], 1, dev["ids"], dev["scores"])
    have = dev["scores"].values()
    want = reference(q, np.ones(2, np.int64), tokens, slots, ids, np.full(2, n))
    assert np.sqrt(np.square(have - want).mean()) <= 2.0**-22 * np.sqrt(np.square(want).mean())
    for v in (c, *dev.values(), rows, at):
        v.free()
    ctx.close()


def test_absent_tokens_and_empty_queries():
    """Pages outside the cache or the list and tokens past max_doc_tokens are
    absent; a query without tokens scores 0."""
    rng = np.random.default_rng(6)
    ctx = context()
    page, dim = 4, 32
    c = Cache(ctx, 10 * page, "int8", dim, 32, page)
    x = rng.standard_normal((10 * page, dim)).astype(np.float32)
    rows, at = Matrix(ctx, x, "f32"), Array(ctx, np.arange(10 * page))
    c.cache.write(rows, at)
    _, s, value = quantise(x, "int8", 32)
    tokens = spread(value, s, 32, dim).astype(np.float64)
    pages = np.array([3, -1, 10, 5, 6], np.int32)
    start = np.array([0, 3, 4, -2, 100], np.int64)
    lens = np.array([12, 8, 9, 4, 4], np.int32)  # document 2 runs past the list, 3 and 4 start outside it
    seen = [np.arange(12, 16), np.r_[20:24, 24:28], np.arange(24, 28), np.r_[[]], np.r_[[]]]
    q = to_type(rng.standard_normal((2, 6, dim)), "f32")
    dev = [Matrix(ctx, q, "f32"), Array(ctx, start), Array(ctx, lens), Array(ctx, pages),
           Array(ctx, np.tile(np.arange(5, dtype=np.int32), (2, 1))), Matrix(ctx, None, "f32", shape=(2, 5)),
           Array(ctx, np.array([6, 0], np.int32))]
    c.cache.maxsim(*dev[:4], 12, dev[4], dev[5], query_lens=dev[6])
    have = dev[5].values()
    for d in range(5):
        want = (q[0] @ tokens[seen[d].astype(int)].T).max(1).sum() if seen[d].size else -np.inf
        assert have[0, d] == want or abs(have[0, d] - want) <= 6 * 2.0**-20 * 64
    assert (have[1] == 0).all()
    c.cache.maxsim(*dev[:4], 5, dev[4], dev[5])
    want = (q[0] @ tokens[[20, 21, 22, 23, 24]].T).max(1).sum()
    assert abs(dev[5].values()[0, 1] - want) <= 6 * 2.0**-20 * 64
    for v in (rows, at, c, *dev):
        v.free()
    ctx.close()


def test_graph_of_writing_reading_and_scoring():
    """Captured calls replay with the eager results, with eager work between
    the replays."""
    import ctypes as C

    from chimera_amd import capi

    hip = C.CDLL("libamdhip64.so.7")
    rng = np.random.default_rng(3)
    ctx = context()
    page, dim = 16, 128
    lens = np.array([700, 30, 5], np.int32)  # split: two launches
    start, pages, slots, total = corpus(rng, lens, page)
    c = Cache(ctx, total * page, "int8", dim, 128, page)
    x = rng.standard_normal((total * page, dim)).astype(np.float32)
    rows, at, out = Matrix(ctx, x, "f32"), Array(ctx, np.arange(total * page)), Matrix(ctx, None, "f32", shape=x.shape)
    q = Matrix(ctx, rng.standard_normal((2, 32, dim)), "f32")
    dev = [Array(ctx, v) for v in (start, lens, pages, np.tile(np.arange(3, dtype=np.int32), (2, 1)))]
    scores = Matrix(ctx, None, "f32", shape=(2, 3))
    top = [Array(ctx, np.zeros((2, 2), np.int64)), Array(ctx, np.zeros((2, 2), np.float32)), Array(ctx, np.zeros(2, np.int32))]

    def step():
        c.cache.write(rows, at)
        c.cache.read(at, out)
        c.cache.maxsim(q, dev[0], dev[1], dev[2], 700, dev[3], scores, k=2, top_ids=top[0], top_scores=top[1],
                       top_counts=top[2])

    def results():
        return [out.values(), scores.values(), c.codes.numpy(), c.scales.numpy(), *(t.numpy() for t in top)]

    step()
    want = results()
    stream, graph, run = C.c_void_p(), C.c_void_p(), C.c_void_p()
    capi.check(capi.lib().chimera_stream(ctx.handle, C.byref(stream)))
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    step()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for _ in range(3):
        assert hip.hipGraphLaunch(run, stream) == 0
        ctx.synchronize()
        assert all(np.array_equal(a, b) for a, b in zip(results(), want))
        step()
        ctx.synchronize()
    hip.hipGraphExecDestroy(run)
    hip.hipGraphDestroy(graph)
    for v in (rows, at, out, q, *dev, scores, *top, c):
        v.free()
    ctx.close()
