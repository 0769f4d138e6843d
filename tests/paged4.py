"""Paged caches in 4 bits for the tests: vectors as bytes by the definition, and a pool like paged.Paged."""
import numpy as np

from graph_horizon_amd import GhKvPaged
from graph_horizon_amd import _ffi as F
from paged import D, Paged, attend

VECTOR = 80


def pack(x):
    """Values [...][128] as vectors [...][80] of bytes, by the definition in FP32."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], 4, 32)
    with np.errstate(all="ignore"):
        low, high = g.min(-1), g.max(-1)
        m, step = low.astype(np.float16), (high - low) / np.float32(15)
        d = step.astype(np.float16)
        d = np.where(d.astype(np.float32) > step, (d.view(np.uint16) - 1).view(np.float16), d)
        df = d.astype(np.float32)[..., None]
        c = np.where(df > 0, np.rint((g - m.astype(np.float32)[..., None]) / df), 0)
        odd = ~np.isfinite(g).all(-1)
    c = np.where(odd[..., None], 0, np.clip(np.nan_to_num(c), 0, 15)).astype(np.uint8).reshape(x.shape)
    d, m = (np.where(odd, np.uint16(0x7E00), y.view(np.uint16)) for y in (d, m))
    dm = np.stack([d, m], -1).astype("<u2").reshape(*x.shape[:-1], 8).view(np.uint8)
    return np.concatenate([c[..., 0::2] | c[..., 1::2] << 4, dm], -1)


def parts(b):
    """Codes [...][4][32], steps and minima [...][4] of vectors of bytes, in 64 bits."""
    c = np.stack([b[..., :64] & 15, b[..., :64] >> 4], -1).reshape(*b.shape[:-1], 4, 32).astype(np.float64)
    dm = np.ascontiguousarray(b[..., 64:]).view(np.float16).astype(np.float64)
    return c, dm[..., 0::2], dm[..., 1::2]


def values(b):
    """What vectors of bytes stand for, in 64 bits."""
    c, d, m = parts(b)
    return (m[..., None] + d[..., None] * c).reshape(*b.shape[:-1], D)


def unpack(b):
    """The same in FP16, as a read-back gives it."""
    return values(b).astype(np.float16)


def attend4(q, kb, vb):
    """paged.attend over vectors of bytes: (out, weights, error bounds of both). The bounds count, besides those of
    paged.attend: keys are sums of d·c and m, of which each product and sum is rounded in FP32 by itself (a half step of
    their sizes' sum for each of 32 dims, and eight more for the groups' sums); the query's sum over a group is held to 2^-22
    and to 2^-16 (an FP16 subnormal times 2^9); half of its dims to 2^-21 (a subnormal times 2^4); a value is rounded to FP16."""
    half = 2.0 ** -24
    k, v = values(kb), values(vb)
    out, w, bound, wb = attend(q, k, v)
    q = np.abs(q.astype(np.float64))
    c, d, m = parts(kb)
    dc, m = (d[..., None] * c).reshape(k.shape), np.repeat(np.abs(m), 32, -1)
    ds = (40 * half * (q @ (dc + m).T) + 2.0 ** -22 * (q @ m.T) + 2.0 ** -16 * m.sum(1) / 32 + 2.0 ** -21 * dc.sum(1)) / np.sqrt(D)
    ds = ds.max(1, keepdims=True)
    a = np.abs(v)
    return out, w, bound + 4 * ds * (w @ a) + 2.0 ** -11 * (w @ a), wb + 4 * ds * w


def check_attention4(p, layer, q, out, before=None, after=None):
    """paged.check_attention over the pool's bytes."""
    g = q.shape[1] // p.heads
    for r, n in enumerate(p.lengths):
        n = int(n)
        if n == 0:
            assert not out[r].view(np.uint16).any(), "a free row's output"
        s = p.cells(r, n)
        for h in range(p.heads):
            hs = slice(h * g, h * g + g)
            if n:
                want, w, ob, wb = attend4(q[r, hs], p.kb[layer, s, h], p.vb[layer, s, h])
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


class Paged4(Paged):
    """A pool of which kb, vb are the bytes, and k, v the FP16 values that a read-back gives."""

    def upload(self):
        if "k" not in self.bufs:
            for name in ("k", "v"):
                setattr(self, name + "b", pack(getattr(self, name)))
        self.k, self.v = unpack(self.kb), unpack(self.vb)
        for name, x in (("k", self.kb), ("v", self.vb), ("table", self.table), ("lengths", self.lengths), ("score", self.score)):
            if x is None:
                continue
            if name not in self.bufs:
                self.bufs[name] = self.hip.alloc_buffer(x.nbytes)
            self.hip.upload(self.bufs[name], x)

    def handle(self):
        b = self.bufs
        kv = F.GhKv(b["k"], b["v"], F.KV_Q4, self.layers, self.slots, self.heads, D, D)
        return GhKvPaged(kv, b["table"], b["lengths"], b.get("score", F.GhBuf()), self.page, self.width, self.rows)

    def read(self, name):
        if name not in ("k", "v"):
            return super().read(name)
        x = getattr(self, name + "b")
        return self.hip.download(self.bufs[name], np.uint8, x.size).reshape(x.shape)
