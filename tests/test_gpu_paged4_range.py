"""Operators over 4-bit caches at sizes of values other than 1: what they hold in fewer bits is relative to the values at hand."""
import numpy as np
import pytest

from graph_horizon_amd import Yarn
from paged import D, attend
from paged4 import Paged4, pack, parts, values
from test_gpu_paged4 import run_attention, turned

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


def test_keys_next_to_the_end_of_fp16_stay_finite(hip, rng):
    """Rotated keys up to 65520, which FP16 rounds to 65504: the minimum of 32 may be rounded up, and no code may stand for more than
    the largest. A step: the values' range over 15, or, where that would reach 65520, what is left above the minimum."""
    tokens, heads = 3000, 4
    yarn = Yarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    p = Paged4(hip, rng, [tokens], 64, heads)
    k = rng.uniform(60000, 65504, (1, tokens, heads, D)).astype(np.float16)
    k[..., :64] = rng.standard_normal((1, tokens, heads, 64))  # pairs that turn further
    kb, pb, qb = hip.from_host(k), hip.from_host(np.zeros(1, np.uint32)), hip.from_host(np.zeros((1, tokens, 1, D), np.float16))
    out = [hip.alloc_buffer(k.nbytes) for _ in range(2)]
    hip.rope_kv_write_paged(p.handle(), qb, qb, kb, kb, 1, pb, tokens, tokens, yarn, 0)
    hip.kv_read_paged(out[0], out[1], p.handle(), tokens, 0)
    back = hip.download(out[0], np.float16, k.size).reshape(k.shape)[0]
    b = p.read("k")[0, p.cells(0, tokens)]
    want, bound = turned(k[0].astype(np.float64), yarn, np.arange(tokens), False)
    c, d, m = parts(b)
    g, e = want.reshape(c.shape), bound.reshape(c.shape).max(-1)
    low, high = g.min(-1), g.max(-1)
    fits, past = high + e < 65520, high - e >= 65520  # (between: either)
    assert np.isnan(m[past]).all() and np.isfinite(m[fits]).all()
    most = m[fits] + 15 * d[fits]
    assert np.all(most < 65520)
    assert np.all(most <= high[fits] + e[fits] + 2.0 ** -11 * np.abs(low[fits]))
    # m by its rounding, d at least the cut-off fifteenth of what is left
    assert np.all(np.abs(m - low)[fits] <= (e + 2.0 ** -11 * np.abs(low))[fits])
    left = np.minimum(high - low, high - m)[fits] - 2 * e[fits]
    assert np.all(d[fits] >= left / 15 * (1 - 2.0 ** -10) - 2.0 ** -23)
    err = np.abs(m[..., None] + d[..., None] * c - g).max(-1)
    assert np.all(err[fits] <= (d / 2 + e + 2.0 ** -11 * np.abs(low))[fits] + 2.0 ** -20)
    assert np.isfinite(back.reshape(c.shape)[fits]).all()
    # cases of each kind are there: the plain step would have reached 65520, and would not
    plain = np.floor((high - low) / 15 * 4) / 4  # steps of 256 to 511 are multiples of a quarter
    over = (low.astype(np.float16).astype(np.float64) + 15 * plain > 65520 + 1) & fits & (plain >= 256)
    assert over.sum() >= 20 and (fits & ~over).sum() >= 1000, (over.sum(), fits.sum())
    for x in (kb, pb, qb, *out):
        hip.free_buffer(x)
    p.free()


@pytest.mark.parametrize("eps", [1e-45, 1e-40, 1.2e-38, 1e-20])
def test_a_head_of_zeros_stays_zero_with_any_eps(hip, rng, eps):
    """0 over the root of eps is 0, with an eps below FP32's least normal number too; other heads are as with none."""
    q = rng.standard_normal((1, 2, D)).astype(np.float16)
    q[0, 0] = 0
    wb = hip.from_host(np.ones(D, np.float16))
    qb, kb, pb, zb = hip.from_host(q), hip.from_host(q), hip.from_host(np.zeros(1, np.uint32)), hip.from_host(q)
    yarn = Yarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    hip.norm_rope_batched(zb, kb, 2, 2, D, 0, 1, wb, wb, 0.0, yarn)
    plain = hip.download(zb, np.float16, q.size).reshape(q.shape)
    hip.upload(kb, q)
    hip.norm_rope_batched(qb, kb, 2, 2, D, 0, 1, wb, wb, eps, yarn)
    for b in (qb, kb):
        got = hip.download(b, np.float16, q.size).reshape(q.shape)
        assert not got[0, 0].view(np.uint16).any() and np.array_equal(got[0, 1], plain[0, 1])
    p = Paged4(hip, rng, [1], 16, 2)
    hip.upload(qb, q)
    hip.upload(kb, q)
    hip.norm_rope_kv_write_paged(p.handle(), qb, qb, kb, kb, 2, wb, wb, eps, pb, 1, 0, yarn, 0)
    assert not hip.download(qb, np.uint16, D).any()
    assert not p.read("k")[0, p.cells(0, 1)[0], 0].any()
    for b in (wb, qb, kb, pb, zb):
        hip.free_buffer(b)
    p.free()
