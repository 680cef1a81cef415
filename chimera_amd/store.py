"""Token embeddings of documents that come and go, quantised on the device:
what an index does not hold between two builds. Pages of a TokenCache go to
documents as they are added, grow or are removed; late interaction rescores
candidates (of an index's search, or all documents) on them.
"""
from __future__ import annotations

from contextlib import ExitStack

import numpy as np

from . import capi
from .operators import TokenCache, cache_row


def _freed(stack: ExitStack, array: capi.DeviceArray) -> capi.DeviceArray:
    """The array, which the stack frees."""
    stack.callback(array.free)
    return array


class TokenStore:
    """A cache of num_pages pages and the tables that say which of them a
    document has. Documents are numbered from 0 on; the number of a removed
    document is used again. The tables are made again and uploaded, all of
    them, at the first call of rescore() after a change, and rescore() takes
    and gives back its buffers: where that counts, keep the tables and buffers
    and call `cache` with tables()."""

    def __init__(self, ctx: capi.Context, num_pages: int, dim: int = 128, format: str = "int8", group: int = 128,
                 page_tokens: int = 16):
        row, scales = cache_row(format, dim, group, page_tokens)
        if num_pages < 1:
            raise ValueError("a store needs pages")
        self.ctx, self.dim, self.page_tokens = ctx, dim, page_tokens
        with ExitStack() as made:
            self._codes = _freed(made, ctx.empty((num_pages * page_tokens, row), np.uint8))
            self._scales = _freed(made, ctx.empty((num_pages * page_tokens, scales), np.float32))
            self.cache = TokenCache(ctx, self._codes, self._scales, format, dim, group, page_tokens)
            made.pop_all()
        self._free = list(range(num_pages - 1, -1, -1))
        self._docs: list[list[int] | None] = []  # pages of each document, None: removed
        self._lens: list[int] = []
        self._unused: list[int] = []  # numbers of removed documents
        self._tables = None  # on the device, as long as nothing changes

    def close(self) -> None:
        if self.cache is None:
            return
        self.ctx.synchronize()
        self._drop_tables()
        self.cache.close()
        self._codes.free()
        self._scales.free()
        self.cache = None

    def _drop_tables(self) -> None:
        for a in self._tables or ():
            a.free()
        self._tables = None

    @property
    def free_tokens(self) -> int:
        """Tokens that the pages no document has can hold."""
        return len(self._free) * self.page_tokens

    def doc_len(self, doc: int) -> int:
        self._check(doc)
        return self._lens[doc]

    def _check(self, doc: int) -> None:
        if not 0 <= doc < len(self._docs) or self._docs[doc] is None:
            raise KeyError(f"no document {doc}")

    def _slots(self, pages: list[int], begin: int, end: int) -> np.ndarray:
        t = np.arange(begin, end)
        return np.asarray(pages, np.int64)[t // self.page_tokens] * self.page_tokens + t % self.page_tokens

    def _next_pages(self, count: int) -> list[int]:
        """The pages that the next document gets; they stay free until they
        are taken."""
        if count > len(self._free):
            raise MemoryError(f"{count} pages are needed, {len(self._free)} are free")
        return self._free[len(self._free) - count:][::-1]

    def _take(self, pages: list[int]) -> None:
        del self._free[len(self._free) - len(pages):]

    def _write(self, embeddings, slots: np.ndarray) -> None:
        if slots.size == 0:
            return
        with ExitStack() as bufs:
            if isinstance(embeddings, np.ndarray):
                embeddings = _freed(bufs, self.ctx.to_device(np.ascontiguousarray(embeddings, np.float32)))
            self.cache.write(embeddings, _freed(bufs, self.ctx.to_device(slots)))
            self.ctx.synchronize()

    def add(self, embeddings, doc_lens) -> list[int]:
        """Adds documents: embeddings [tokens, dim], one document's tokens
        after the other's (a numpy array or a device array), and the number of
        tokens of each. Returns their numbers."""
        lens = [int(n) for n in doc_lens]
        if len(embeddings.shape) != 2 or embeddings.shape[1] != self.dim or any(n < 0 for n in lens) or \
                sum(lens) != embeddings.shape[0]:
            raise ValueError(f"the lengths must add up to the rows of embeddings [tokens, {self.dim}]")
        owned = [-(-n // self.page_tokens) for n in lens]
        pages = self._next_pages(sum(owned))
        ends = np.cumsum([0, *owned]).tolist()
        per_doc = [pages[a:b] for a, b in zip(ends, ends[1:])]
        slots = [self._slots(p, 0, n) for p, n in zip(per_doc, lens)]
        self._write(embeddings, np.concatenate(slots).astype(np.int64) if slots else np.zeros(0, np.int64))
        # nothing has changed up to here, so a refused write leaves the store as it was
        self._take(pages)
        ids = []
        for p, n in zip(per_doc, lens):
            doc = self._unused.pop() if self._unused else len(self._docs)
            if doc == len(self._docs):
                self._docs.append(None)
                self._lens.append(0)
            self._docs[doc], self._lens[doc] = p, n
            ids.append(doc)
        self._drop_tables()
        return ids

    def append(self, doc: int, embeddings) -> None:
        """Adds tokens at a document's end."""
        self._check(doc)
        if len(embeddings.shape) != 2 or embeddings.shape[1] != self.dim:
            raise ValueError(f"embeddings must be [tokens, {self.dim}]")
        begin, end = self._lens[doc], self._lens[doc] + embeddings.shape[0]
        pages = self._next_pages(-(-end // self.page_tokens) - len(self._docs[doc]))
        self._write(embeddings, self._slots(self._docs[doc] + pages, begin, end).astype(np.int64))
        self._take(pages)
        self._docs[doc] = self._docs[doc] + pages
        self._lens[doc] = end
        self._drop_tables()

    def remove(self, doc: int) -> None:
        self._check(doc)
        self._free.extend(self._docs[doc])
        self._docs[doc], self._lens[doc] = None, 0
        self._unused.append(doc)
        self._drop_tables()

    def read(self, doc: int) -> np.ndarray:
        """The document's embeddings as the cache has them [tokens, dim]."""
        self._check(doc)
        n = self._lens[doc]
        if n == 0:
            return np.zeros((0, self.dim), np.float32)
        with ExitStack() as bufs:
            slots = _freed(bufs, self.ctx.to_device(self._slots(self._docs[doc], 0, n).astype(np.int64)))
            out = _freed(bufs, self.ctx.empty((n, self.dim), np.float32))
            self.cache.read(slots, out)
            return out.numpy()

    def tables(self):
        """(page_start, doc_lens, pages) on the device and the longest
        document's length, as TokenCache.maxsim takes them."""
        if self._tables is None:
            owned = [d or [] for d in self._docs]
            start = np.concatenate([[0], np.cumsum([len(d) for d in owned], dtype=np.int64)])[:-1]
            pages = np.array([p for d in owned for p in d] or [0], np.int32)
            with ExitStack() as made:
                self._tables = [_freed(made, self.ctx.to_device(a))
                                for a in (start.astype(np.int64) if len(owned) else np.zeros(1, np.int64),
                                          np.array(self._lens or [0], np.int32), pages)]
                made.pop_all()
        return (*self._tables, max(self._lens, default=0))

    def rescore(self, queries: np.ndarray, cand_ids: np.ndarray, k: int, query_lens=None):
        """The best k of each query's candidates [nq, cap] (-1: none) for
        queries [nq, query_len, dim]: (scores of all candidates [nq, cap], ids
        [nq, k], scores [nq, k], counts [nq])."""
        q = np.ascontiguousarray(queries, np.float32)
        ids = np.asarray(cand_ids).astype(np.int64)
        ids = np.where((ids >= -(1 << 31)) & (ids < 1 << 31), ids, -1).astype(np.int32)  # past 32 bits: no document's
        nq, cap = ids.shape
        start, lens, pages, longest = self.tables()
        with ExitStack() as bufs:
            d_q, d_ids = (_freed(bufs, self.ctx.to_device(v)) for v in (q, ids))
            d_scores, d_top, d_top_scores, d_counts = (
                _freed(bufs, self.ctx.empty(shape, dtype))
                for shape, dtype in (((nq, cap), np.float32), ((nq, k), np.int64), ((nq, k), np.float32), ((nq,), np.int32)))
            d_lens = None
            if query_lens is not None:
                d_lens = _freed(bufs, self.ctx.to_device(np.clip(query_lens, 0, q.shape[1]).astype(np.int32)))
            self.cache.maxsim(d_q, start, lens, pages, longest, d_ids, d_scores, query_lens=d_lens, k=k, top_ids=d_top,
                              top_scores=d_top_scores, top_counts=d_counts)
            return d_scores.numpy(), d_top.numpy(), d_top_scores.numpy(), d_counts.numpy()
