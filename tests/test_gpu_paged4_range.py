"""Operators over 4-bit caches at sizes of values other than 1: what they hold in fewer bits is relative to the values at hand."""
import numpy as np
import pytest

from paged import D, attend
from paged4 import Paged4, pack, parts, values
from test_gpu_paged4 import run_attention

pytestmark = pytest.mark.gpu


def attend_relative(q, kb, vb):
    """paged.attend over vectors of bytes: (out, weights, error bounds of both), as paged4.attend4 but for what the products hold of
    a query, by its largest |q|: that is brought to 2^15 or more before FP16's least steps count, which are 2^-16 of a group's sum
    and 2^-21 of half of the dims, so 2^-31 and 2^-36 of the largest."""
    half = 2.0 ** -24
    k, v = values(kb), values(vb)
    out, w, bound, wb = attend(q, k, v)
    q = np.abs(q.astype(np.float64))
    top = q.max(1, keepdims=True)
    c, d, m = parts(kb)
    dc, m = (d[..., None] * c).reshape(k.shape), np.repeat(np.abs(m), 32, -1)
    ds = (40 * half * (q @ (dc + m).T) + 2.0 ** -22 * (q @ m.T) + top * (2.0 ** -31 * m.sum(1) / 32 + 2.0 ** -36 * dc.sum(1))) / np.sqrt(D)
    ds = ds.max(1, keepdims=True)
    a = np.abs(v)
    return out, w, bound + 4 * ds * (w @ a) + 2.0 ** -11 * (w @ a), wb + 4 * ds * w


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("lengths,width", [([300, 40, 1], None), ([5000, 40, 3000, 17], 1200)])  # spans, chunks
@pytest.mark.parametrize("q_size,k_size", [(1e-3, 3e3), (2e-4, 1.2e4), (1e-6, 2e4), (1.0, 1.0), (1e3, 1e-3), (2e4, 1e-4)])
def test_attention_of_small_and_large_queries(hip, rng, q_size, k_size, lengths, width, scored):
    """Queries far from 1 against keys far on the other side: scores of the same spread, as near to the definition."""
    heads, group = 4, 3
    p = Paged4(hip, rng, lengths, 16, heads, width=width, scored=scored)
    k = np.clip(np.where(np.isnan(p.k), 0, k_size * p.k.astype(np.float64)), -60000, 60000).astype(np.float16)
    p.kb = pack(k)
    p.upload()
    q = np.clip(q_size * rng.standard_normal((len(lengths), heads * group, D)), -60000, 60000).astype(np.float16)
    q[:, 1] *= np.float16(0.01)       # each head by itself
    q[:, 2, ::3] = 0
    q[:, 3, 1:] *= np.float16(0.001)  # one dim above the others
    before = p.read("score") if scored else None
    q, out = run_attention(hip, p, heads * group, rng, q=q)
    after = p.read("score") if scored else None
    for r, n in enumerate(lengths):
        s = p.cells(r, n)
        for h in range(heads):
            hs = slice(h * group, (h + 1) * group)
            want, w, ob, wb = attend_relative(q[r, hs], p.kb[0, s, h], p.vb[0, s, h])
            err = np.abs(out[r, hs].astype(np.float64) - want)
            assert np.all(err <= ob), (r, h, float((err / ob).max()))
            if scored:
                total = before[0, r, h, :n].astype(np.float64) + w.sum(0)
                bound = wb.sum(0) + (group + 1) * 2.0 ** -24 * np.abs(total)
                err = np.abs(after[0, r, h, :n] - total)
                assert np.all(err <= bound), (r, h, float((err / bound).max()))
    p.free()
