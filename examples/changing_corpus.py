"""From hidden states to ranked documents while the corpus changes:

1. a dense stack (a residual layer with an activation, then the layer that
   ends in embeddings of length one) is trained for a few steps, so that a
   query's tokens come near their document's,
2. it turns the documents' hidden states into token embeddings, from which an
   index is built and which go into a quantised store as well,
3. documents are added to the store after the build, and one is removed,
4. a query's candidates, the index's and the new documents, are ranked by late
   interaction on the store.

Hidden states are synthetic. Run: python examples/changing_corpus.py
"""
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from chimera_amd import capi  # noqa: E402
from chimera_amd.operators import Linear  # noqa: E402
from chimera_amd.store import TokenStore  # noqa: E402

HIDDEN, DIM, QUERY_LEN = 256, 128, 32


class Head:
    """H = x + gelu(x W1^T + b1), y = H W2^T / |H W2^T|, in 32 bits."""

    def __init__(self, ctx, rng, max_rows):
        self.ctx, self.rows = ctx, max_rows
        self.host = {"w1": rng.standard_normal((HIDDEN, HIDDEN)).astype(np.float32) / HIDDEN**0.5,
                     "b1": np.zeros(HIDDEN, np.float32),
                     "w2": rng.standard_normal((DIM, HIDDEN)).astype(np.float32) / HIDDEN**0.5}
        self.p = {name: ctx.to_device(v) for name, v in self.host.items()}
        self.g = {name: ctx.empty(v.shape, np.float32) for name, v in self.host.items()}
        self.first = Linear(ctx, self.p["w1"], self.p["b1"], activation="gelu", max_rows=max_rows, training=True)
        self.last = Linear(ctx, self.p["w2"], normalize=True, max_rows=max_rows, training=True)

    def forward(self, x, keep=None):
        """Embeddings [rows, DIM] of device hidden states; `keep` gets what
        the backward pass reads."""
        rows = x.shape[0]
        h, y = self.ctx.empty((rows, HIDDEN), np.float32), self.ctx.empty((rows, DIM), np.float32)
        saved = norms = None
        if keep is not None:
            saved, norms = self.ctx.empty((rows, HIDDEN), np.float32), self.ctx.empty((rows,), np.float32)
            keep.update(x=x, h=h, y=y, saved=saved, norms=norms)
        self.first.forward(x, h, residual=x, saved=saved)
        self.last.forward(h, y, norms=norms)
        if keep is None:
            self.ctx.synchronize()
            h.free()
        return y

    def step(self, keep, dy, rate):
        """One step of gradient descent from dL/dy (host)."""
        ctx, rows = self.ctx, dy.shape[0]
        d_dy, dh = ctx.to_device(dy), ctx.empty((rows, HIDDEN), np.float32)
        self.last.backward(keep["h"], d_dy, y=keep["y"], norms=keep["norms"], dx=dh, dweight=self.g["w2"])
        self.first.backward(keep["x"], dh, saved=keep["saved"], dweight=self.g["w1"], dbias=self.g["b1"])
        for name, value in self.host.items():
            value -= rate * self.g[name].numpy()
            capi.check(capi.lib().chimera_copy_to_device(ctx.handle, capi.P(self.p[name].ptr), capi._ptr(value),
                                                         value.nbytes))
        for a in (d_dy, dh, keep["h"], keep["y"], keep["saved"], keep["norms"]):
            a.free()

    def close(self):
        self.first.close()
        self.last.close()
        for a in (*self.p.values(), *self.g.values()):
            a.free()


def noisy(rng, x):
    """Hidden states of the same words in another place."""
    return (x + 0.7 * rng.standard_normal(x.shape)).astype(np.float32)


def train(ctx, head, rng, hidden, steps=30):
    """Pulls a token's embedding towards that of its noisy copy and away from
    the other tokens': L = mean over i of log sum_j exp(s_ij) - s_ii with
    s = 8 <a_i, b_j>. Returns the losses."""
    losses = []
    n = head.rows // 2
    for _ in range(steps):
        pick = rng.choice(hidden.shape[0], n, replace=False)
        x = ctx.to_device(np.concatenate([hidden[pick], noisy(rng, hidden[pick])]))
        keep = {}
        y = head.forward(x, keep).numpy()
        a, b = y[:n], y[n:]
        s = 8 * a @ b.T
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        losses.append(float(-np.log(p[np.arange(n), np.arange(n)]).mean()))
        ds = 8 * (p - np.eye(n, dtype=np.float32)) / n
        head.step(keep, np.concatenate([ds @ b, ds.T @ a]).astype(np.float32), rate=0.5)
        x.free()
    return losses


def embed(ctx, head, hidden):
    x = ctx.to_device(hidden)
    y = head.forward(x)
    out = y.numpy()
    x.free()
    y.free()
    return out


def main(docs=400, added=20, queries=8, seed=1):
    rng = np.random.default_rng(seed)
    lens = rng.integers(20, 90, docs + added).astype(np.int32)
    ptrs = np.concatenate([[0], np.cumsum(lens)])
    topics = rng.standard_normal((docs + added, HIDDEN)).astype(np.float32)
    hidden = np.repeat(topics, lens, 0) + rng.standard_normal((int(ptrs[-1]), HIDDEN)).astype(np.float32)

    # the index's context, and one for the operators
    index = capi.Context(None, 8, 100, 40, 3, max_batch=queries)
    ctx = capi.Context(None, 1, 1, 1, 1)
    head = Head(ctx, rng, max_rows=int(ptrs[-1]))
    head.rows = 512
    losses = train(ctx, head, rng, hidden)
    tokens = embed(ctx, head, hidden)

    old = int(ptrs[docs])
    index.build(tokens[:old], lens[:docs], n_clusters=256, ex_bits=4)
    store = TokenStore(ctx, num_pages=int((-(-lens // 16)).sum()), format="int8")
    ids = store.add(tokens[:old], lens[:docs])
    new = store.add(tokens[old:], lens[docs:])

    # half of the queries ask for new documents; the first old target goes
    targets = np.concatenate([rng.choice(docs, queries - queries // 2, replace=False),
                              docs + rng.choice(added, queries // 2, replace=False)])
    pick = ptrs[targets][:, None] + (rng.random((queries, QUERY_LEN)) * lens[targets][:, None]).astype(np.int64)
    q = embed(ctx, head, noisy(rng, hidden[pick].reshape(-1, HIDDEN))).reshape(queries, QUERY_LEN, DIM)
    store.remove(ids[targets[0]])

    found, _, _ = index.search(q, k=40)
    cands = np.concatenate([found.astype(np.int32), np.tile(np.array(new, np.int32), (queries, 1))], 1)
    _, top, top_scores, _ = store.rescore(q, cands, k=5)
    store.close()
    head.close()
    index.close()
    ctx.close()
    return {"losses": losses, "targets": targets, "top": top, "scores": top_scores, "removed": int(targets[0])}


if __name__ == "__main__":
    r = main()
    print(f"loss {r['losses'][0]:.3f} -> {r['losses'][-1]:.3f}")
    for t, ids, scores in zip(r["targets"], r["top"], r["scores"]):
        note = " (removed)" if t == r["removed"] else ""
        print(f"target {t}{note}: best {ids.tolist()}, scores {np.round(scores, 3).tolist()}")
