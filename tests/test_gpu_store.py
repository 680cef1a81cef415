"""The store of changing documents and the example that runs the operators
together."""
import importlib.util
from pathlib import Path

import numpy as np
import pytest

from chimera_amd.store import TokenStore
from operator_checks import context

pytestmark = pytest.mark.gpu


def unit(rng, n, dim):
    x = rng.standard_normal((n, dim)).astype(np.float32)
    return x / np.linalg.norm(x, axis=1, keepdims=True)


def test_documents_come_and_go():
    rng = np.random.default_rng(5)
    ctx = context()
    store = TokenStore(ctx, num_pages=40, dim=64, format="int8", group=64, page_tokens=8)
    held = {}

    def add(lens):
        x = unit(rng, sum(lens), 64)
        for doc, part in zip(store.add(x, lens), np.split(x, np.cumsum(lens)[:-1])):
            held[doc] = part
            yield doc

    def check():
        q = unit(rng, 2 * 7, 64).reshape(2, 7, 64)
        ids = np.tile(np.arange(-1, 8, dtype=np.int32), (2, 1))
        scores, top, top_scores, counts = store.rescore(q, ids, k=3)
        for j, d in enumerate(ids[0]):
            if d not in held or not len(held[d]):
                assert np.isneginf(scores[:, j]).all()
                continue
            back = store.read(d)
            # int8: half a code of the largest value, at most 1 / 254
            assert back.shape == held[d].shape and np.abs(back - held[d]).max() <= 1 / 254
            want = (q.astype(np.float64) @ back.astype(np.float64).T).max(2).sum(1)
            assert np.abs(scores[:, j] - want).max() <= 7 * 2.0**-20
        assert np.array_equal(top_scores, -np.sort(-scores, 1)[:, :3])

    a, b, c = add([3, 17, 0])
    check()
    store.append(c, (x := unit(rng, 1, 64)))
    held[c] = x
    store.append(a, (x := unit(rng, 30, 64)))
    held[a] = np.concatenate([held[a], x])
    check()
    store.remove(b)
    del held[b]
    with pytest.raises(KeyError):
        store.read(b)
    check()
    free = store.free_tokens
    with pytest.raises(MemoryError):
        store.add(unit(rng, free + 1, 64), [free + 1])
    assert store.free_tokens == free
    (d,) = add([free])
    assert d == b and store.free_tokens == 0
    check()
    with pytest.raises(MemoryError):
        store.append(d, unit(rng, 8, 64))
    with pytest.raises(ValueError):
        store.add(unit(rng, 4, 64), [3])
    store.close()
    ctx.close()


def test_the_example():
    path = Path(__file__).resolve().parents[1] / "examples" / "changing_corpus.py"
    spec = importlib.util.spec_from_file_location("changing_corpus", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    r = module.main()
    assert r["losses"][-1] < 0.8 * r["losses"][0]
    found = r["top"][:, 0] == r["targets"]
    assert found[1:].all() and r["removed"] not in r["top"]
