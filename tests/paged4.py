"""Paged caches in 4 bits for the tests: vectors as bytes by the definition, and a pool like paged.Paged."""
import numpy as np

from graph_horizon_amd import GhKvPaged
from graph_horizon_amd import _ffi as F
from paged import D, Paged

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


def unpack(b):
    """The FP16 values that vectors of bytes stand for."""
    c, d, m = parts(b)
    return (m[..., None] + d[..., None] * c).astype(np.float16).reshape(*b.shape[:-1], D)


class Paged4(Paged):
    """k, v are the FP16 values that the pool's bytes kb, vb stand for."""

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
