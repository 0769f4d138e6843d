"""Paged caches for the tests: a pool with its tables and lengths on the device, and the operators'
definitions in 64 bits over the same arrays."""
import numpy as np

from graph_horizon_amd import GhKvPaged
from graph_horizon_amd import _ffi as F

D = 128


def pages_of(n, page):
    return -(-n // page)


class Paged:
    """A pool and a batch over it. Positions that no row holds are NaN, so that whatever reads them shows.
    k, v: [layers][slots][heads][128] FP16; table, lengths, score as on the device."""

    def __init__(self, hip, rng, lengths, page, heads, layers=1, extra_pages=3, width=None, scored=False, slots=None,
                 score=None, garbage=np.float16(np.nan)):
        self.hip, self.page, self.heads, self.layers, self.rows = hip, page, heads, layers, len(lengths)
        need = [pages_of(n, page) for n in lengths]
        self.width = width or max(1, max(need))
        pages = sum(need) + extra_pages
        self.slots = slots or pages * page
        order = rng.permutation(self.slots // page)[:sum(need)]
        # places past a row's pages hold numbers beyond the pool: they are never looked at
        self.table = np.full((self.rows, self.width), 0xFFFFFFF0, np.uint32)
        at = 0
        for r, c in enumerate(need):
            self.table[r, :c] = order[at:at + c]
            at += c
        self.lengths = np.asarray(lengths, np.uint32)
        self.k = np.full((layers, self.slots, heads, D), garbage, np.float16)
        self.v = self.k.copy()
        for r, n in enumerate(lengths):
            s = self.cells(r, n)
            self.k[:, s] = rng.standard_normal((layers, n, heads, D)).astype(np.float16)
            self.v[:, s] = rng.standard_normal((layers, n, heads, D)).astype(np.float16)
        self.score = None
        if scored:
            shape = (layers, self.rows, heads, self.width * page)
            self.score = np.ascontiguousarray(rng.random(shape) if score is None else np.broadcast_to(score, shape), np.float32)
        self.bufs = {}
        self.upload()

    def cells(self, r, n):
        """Slots of row r's first n positions."""
        j = np.arange(n)
        return self.table[r, j // self.page].astype(np.int64) * self.page + j % self.page

    def upload(self):
        for name in ("k", "v", "table", "lengths", "score"):
            x = getattr(self, name)
            if x is None:
                continue
            if name not in self.bufs:
                self.bufs[name] = self.hip.alloc_buffer(x.nbytes)
            self.hip.upload(self.bufs[name], x)

    def handle(self):
        b = self.bufs
        kv = F.GhKv(b["k"], b["v"], F.KV_F16, self.layers, self.slots, self.heads, D, D)
        return GhKvPaged(kv, b["table"], b["lengths"], b.get("score", F.GhBuf()), self.page, self.width, self.rows)

    def read(self, name):
        x = getattr(self, name)
        return self.hip.download(self.bufs[name], x.dtype, x.size).reshape(x.shape)

    def free(self):
        for b in self.bufs.values():
            self.hip.free_buffer(b)
        self.bufs = {}


def attend(q, k, v):
    """q [G][128] over k, v [n][128] in 64 bits: (out, weights, error bounds of both). The bounds count FP32
    roundings: a score's sum of 128 exact products is off by at most 128 half steps of Σ|q k| and two more for
    its scaling; the weight moves by that factor and by 2^-21 (exp2, the two FP16 parts); sums of n terms
    in any order by n half steps."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    half, n = 2.0 ** -24, len(k)
    s = q @ k.T / np.sqrt(D)
    ds = (128 * half * (np.abs(q) @ np.abs(k).T) / np.sqrt(D) + 4 * half * (np.abs(s) + 15)).max(1, keepdims=True)
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    rel = 2 * ds + 2.0 ** -21 + (n + 64) * half
    out = w @ v
    # a weight's two parts are at least 2^-24 of the 2^15 that the largest of its split has
    tail = 2.0 ** -38 * w.max(1, keepdims=True) * np.abs(v).sum(0)
    out_bound = 2 * rel * (w @ np.abs(v)) + tail + np.abs(out) * 2.0 ** -11 + 2.0 ** -25
    return out, w, out_bound, w * 2 * rel


def check_attention(p, layer, q, out, before=None, after=None):
    """Outputs [rows][heads·G][128] (and scores) of one call against attend()."""
    g = q.shape[1] // p.heads
    for r, n in enumerate(p.lengths):
        n = int(n)
        if n == 0:
            assert not out[r].view(np.uint16).any(), "a free row's output"
        s = p.cells(r, n)
        for h in range(p.heads):
            hs = slice(h * g, h * g + g)
            if n:
                want, w, ob, wb = attend(q[r, hs], p.k[layer, s, h], p.v[layer, s, h])
                err = np.abs(out[r, hs].astype(np.float64) - want)
                assert np.all(err <= ob), (r, h, float((err / ob).max()))
            if before is not None:
                old, new = before[layer, r, h], after[layer, r, h]
                if n:
                    total = old[:n].astype(np.float64) + w.sum(0)
                    bound = wb.sum(0) + (g + 1) * 2.0 ** -24 * np.abs(total)
                    err = np.abs(new[:n] - total)
                    assert np.all(err <= bound), (r, h, float((err / bound).max()))
                assert np.array_equal(new[n:].view(np.uint32), old[n:].view(np.uint32)), "scores past the row"
    if before is not None:
        others = [i for i in range(p.layers) if i != layer]
        assert np.array_equal(before[others], after[others]), "other layers' scores"


def order_key(x):
    b = x.astype(np.float32).view(np.int32).astype(np.int64)
    return np.where(b < 0, b ^ 0x7FFFFFFF, b)


def keep(score, budget, recent):
    """Positions that an eviction keeps of one head's scores, ascending."""
    n = len(score)
    older = order_key(score[:n - recent])
    best = np.lexsort((np.arange(len(older)), -older))[:budget - recent]
    return np.concatenate([np.sort(best), np.arange(n - recent, n)]).astype(np.uint32)
