"""The operators over paged caches (gh_*_paged): append with RoPE, decode attention with and without the
accumulation of weights, eviction, and a run of all of them, against 64-bit definitions (tests/paged.py)."""
import threading

import numpy as np
import pytest

from graph_horizon_amd import GhError, GhKvPaged, HipBackend, HipModel, Yarn, synth
from graph_horizon_amd import _ffi as F
from paged import D, Paged, attend, check_attention, keep, pages_of

pytestmark = pytest.mark.gpu
YARN = Yarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)


def run_attention(hip, p, q_heads, rng, layer=0, max_len=0, q=None):
    if q is None:
        q = rng.standard_normal((p.rows, q_heads, D)).astype(np.float16)
    qb, ob = hip.from_host(q), hip.from_host(np.full_like(q, np.nan))
    try:
        hip.attention_decode_paged(ob, qb, p.handle(), q_heads, max_len, layer)
        out = hip.download(ob, np.float16, q.size).reshape(q.shape)
    finally:
        hip.free_buffer(qb)
        hip.free_buffer(ob)
    return q, out


# ---- attention ----

LENGTHS = {
    "one": [1],
    "tile_edges": [15, 16, 17, 0, 63, 64, 65, 1],
    "empty": [0, 0],
    "ragged": [1000, 3, 0, 257, 640, 129, 1],
    "long": [9001, 100],
}


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("name", list(LENGTHS))
@pytest.mark.parametrize("page,heads,group", [(16, 8, 4), (64, 2, 8), (32, 1, 1), (128, 5, 3), (16, 3, 16), (256, 1, 7)])
def test_attention(hip, rng, name, page, heads, group, scored):
    p = Paged(hip, rng, LENGTHS[name], page, heads, layers=2, scored=scored)
    before = None if not scored else p.read("score")
    q, out = run_attention(hip, p, heads * group, rng, layer=1)
    check_attention(p, 1, q, out, before, p.read("score") if scored else None)
    for name in ("k", "v", "table", "lengths"):
        assert np.array_equal(p.read(name).view(np.uint8), getattr(p, name).view(np.uint8)), name
    p.free()


@pytest.mark.parametrize("scored", [False, True])
def test_attention_past_the_cache(hip, rng, scored):
    """128 MiB of K and V, from which they are read with another cache policy."""
    p = Paged(hip, rng, [20000, 13000, 17], 64, 8, scored=scored)
    before = p.read("score") if scored else None
    q, out = run_attention(hip, p, 32, rng)
    check_attention(p, 0, q, out, before, p.read("score") if scored else None)
    p.free()


@pytest.mark.parametrize("max_len", [300, 320, 1000, 4096])
@pytest.mark.parametrize("group", [2, 4])
def test_attention_launch_longer_than_rows(hip, rng, max_len, group):
    """A table with room: the launch is sized by max_len, the rows end before it."""
    p = Paged(hip, rng, [300, 0, 17], 16, 4, width=256, scored=True)
    before = p.read("score")
    q, out = run_attention(hip, p, 4 * group, rng, max_len=max_len)
    check_attention(p, 0, q, out, before, p.read("score"))
    p.free()


def test_attention_row_groups(hip, rng):
    """More scratch than one group of rows may take: 300 rows of 16 heads over up to 32768 positions."""
    lengths = [int(n) for n in rng.integers(0, 40, 300)]
    lengths[-1] = 700
    p = Paged(hip, rng, lengths, 16, 1, width=2048, scored=True)
    before = p.read("score")
    q, out = run_attention(hip, p, 16, rng)
    check_attention(p, 0, q, out, before, p.read("score"))
    p.free()


def test_attention_repeats_bit_for_bit(hip, rng):
    p = Paged(hip, rng, [3000, 40, 1111], 32, 8)
    q, first = run_attention(hip, p, 32, rng)
    for _ in range(3):
        assert np.array_equal(run_attention(hip, p, 32, rng, q=q)[1].view(np.uint16), first.view(np.uint16))
    p.free()


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("lengths,width", [([0, 300, 17], 20), ([5000, 0, 40, 700], 313), ([3000, 2500, 9, 0] * 5, 188)])
def test_attention_into_its_queries(hip, rng, lengths, width, scored):
    """out is q's own buffer, in spans of one and more and in chunks: the bits of the call with two buffers."""
    p = Paged(hip, rng, lengths, 16, 4, width=width, scored=scored)
    q, want = run_attention(hip, p, 16, rng)
    buf = hip.from_host(q)
    hip.attention_decode_paged(buf, buf, p.handle(), 16, 0, 0)
    got = hip.download(buf, np.float16, q.size).reshape(q.shape)
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16))
    hip.free_buffer(buf)
    p.free()


def test_attention_equals_contiguous_decode(hip, rng):
    """Pages in order are the contiguous cache: both operators within twice the bound of each."""
    n, heads, group = 777, 8, 4
    p = Paged(hip, rng, [n], 16, heads, layers=2)
    q, out = run_attention(hip, p, heads * group, rng, layer=1)
    c = np.zeros((2, 800, heads, D), np.float16), np.zeros((2, 800, heads, D), np.float16)
    c[0][:, :n], c[1][:, :n] = p.k[:, p.cells(0, n)], p.v[:, p.cells(0, n)]
    kb, vb, qb, ob = hip.from_host(c[0]), hip.from_host(c[1]), hip.from_host(q), hip.alloc_buffer(q.nbytes)
    hip.attention_decode(ob, qb, F.GhKv(kb, vb, F.KV_F16, 2, 800, heads, D, D), heads * group, n - 1, 1)
    other = hip.download(ob, np.float16, q.size).reshape(q.shape).astype(np.float64)
    for h in range(heads):
        hs = slice(h * group, h * group + group)
        bound = attend(q[0, hs], c[0][1, :n, h], c[1][1, :n, h])[2]
        assert np.all(np.abs(other[0, hs] - out[0, hs]) <= 2 * bound)
    for b in (kb, vb, qb, ob):
        hip.free_buffer(b)
    p.free()


def test_attention_shared_and_repeated_pages(hip, rng):
    """Two rows over one prompt's pages, and a row that has the same page twice."""
    p = Paged(hip, rng, [200, 200, 64], 16, 2)
    p.table[1, :8] = p.table[0, :8]
    p.table[2, :4] = p.table[2, [0, 1, 0, 1]]
    p.upload()
    q, out = run_attention(hip, p, 8, rng)
    check_attention(p, 0, q, out)
    p.free()


@pytest.mark.parametrize("heads", [8, 1])
def test_attention_pool_past_4_gib(hip, rng, heads):
    """Pages whose byte offsets pass 32 bits (a pool of 4.5 GiB each for K and V)."""
    page, slots = 64, (9 << 29) // (256 * heads) // 64 * 64
    lengths = [130, 70]
    small = Paged(hip, rng, lengths, page, heads)
    kv = [hip.alloc_buffer(slots * heads * 256) for _ in range(2)]
    last = slots // page - 1
    table = small.table.copy()
    for r in range(2):
        for i in range(pages_of(lengths[r], page)):
            table[r, i] = last
            for b, x in zip(kv, (small.k, small.v)):
                at = int(small.table[r, i]) * page
                hip.upload(b, x[0, at:at + page], last * page * heads * 256)
            last -= 3 if i else slots // page // 2
            last %= slots // page
    tb, q = hip.from_host(table), rng.standard_normal((2, 4 * heads, D)).astype(np.float16)
    h = small.handle()
    h.kv = F.GhKv(kv[0], kv[1], F.KV_F16, 1, slots, heads, D, D)
    h.table = tb
    qb, ob = hip.from_host(q), hip.alloc_buffer(q.nbytes)
    hip.attention_decode_paged(ob, qb, h, 4 * heads, 0, 0)
    check_attention(small, 0, q, hip.download(ob, np.float16, q.size).reshape(q.shape))
    for b in (*kv, tb, qb, ob):
        hip.free_buffer(b)
    small.free()


def test_attention_peaked_and_flat_weights(hip, rng):
    """One key far above all others; 30000 keys of 2^-26 of the largest each, which together are 2^-11 of
    it; and a row of equal scores."""
    n = 30000
    p = Paged(hip, rng, [n, n, 500], 64, 1)
    q = np.zeros((3, 1, D), np.float16)
    q[:, 0, 0] = 8
    p.k[:] = 0
    p.v[:] = np.where(np.isnan(p.v), 0, p.v)
    a, b = p.cells(0, n), p.cells(1, n)
    p.k[0, a[1234], 0, 0] = 60
    p.k[0, b, 0, 0] = -25.5  # 8 * 25.5 / sqrt(128) = 18.03 = 26.01 ln 2
    p.k[0, b[77], 0, 0] = 0
    p.v[0, b, 0, 1] = 1000
    p.v[0, b[77], 0] = 0
    p.upload()
    q, out = run_attention(hip, p, 1, rng, q=q)
    check_attention(p, 0, q, out)
    assert 0.2 < out[1, 0, 1] < 0.7  # 30000 * 2^-26 * 1000
    p.free()


def test_attention_infinities_and_nan_stay_where_they_are_seen(hip, rng):
    """An infinite V, an infinite and a NaN K: the outputs of the definition, in their head and row alone; NaN
    and infinities behind the last position do not show (the pool is full of NaN elsewhere)."""
    p = Paged(hip, rng, [100, 100, 100, 100], 16, 2)
    cells = [p.cells(r, 100) for r in range(4)]
    p.v[0, cells[0][40], 1, 5] = np.inf
    p.v[0, cells[0][3], 1, 6] = -np.inf
    p.v[0, cells[0][40], 1, 7] = np.nan
    p.k[0, cells[1][50], 0] = np.nan
    p.k[0, cells[2][50], 0, 0] = np.inf
    p.upload()
    q = np.abs(rng.standard_normal((4, 8, D))).astype(np.float16)
    q[2, :, 0] = -1  # a score of -inf: weight 0
    q, out = run_attention(hip, p, 8, rng, q=q)
    assert np.all(out[0, 4:, 5] == np.inf) and np.all(out[0, 4:, 6] == -np.inf) and np.isnan(out[0, 4:, 7]).all()
    assert np.isnan(out[1, :4]).all()
    p.v[0, cells[0][[40, 40, 3]], 1, [5, 7, 6]] = 0
    p.k[0, cells[1][50], 0] = 0
    with np.errstate(invalid="ignore"):
        for r, h, dims in ((0, 0, slice(None)), (0, 1, slice(8, None)), (1, 1, slice(None)), (3, 0, slice(None)),
                           (3, 1, slice(None))):
            want, _, bound, _ = attend(q[r, 4 * h:4 * h + 4], p.k[0, cells[r], h], p.v[0, cells[r], h])
            assert np.all(np.abs(out[r, 4 * h:4 * h + 4] - want)[:, dims] <= bound[:, dims]), (r, h)
    rest = np.delete(cells[2], 50)
    want, _, bound, _ = attend(q[2, :4], p.k[0, rest, 0], p.v[0, rest, 0])
    assert np.all(np.abs(out[2, :4] - want) <= bound)
    p.free()


@pytest.mark.parametrize("lengths", [[200, 90], [7000, 3000]])  # both divisions of the work
def test_attention_a_query_that_is_not_finite_is_its_own(hip, rng, lengths):
    """A NaN and an infinity in two heads' queries: those heads are NaN, the others of the same kv head as ever,
    and scores are NaN where such a weight was added."""
    p = Paged(hip, rng, lengths, 16, 8, scored=True)
    before = p.read("score")
    q = rng.standard_normal((2, 32, D)).astype(np.float16)
    q[0, 5, 3], q[1, 30, 100] = np.nan, np.inf
    q, out = run_attention(hip, p, 32, rng, q=q)
    after = p.read("score")
    for r, odd in ((0, 5), (1, 30)):
        s = p.cells(r, lengths[r])
        for h in range(8):
            for i in range(4 * h, 4 * h + 4):
                if i == odd:
                    assert np.isnan(out[r, i]).all()
                    continue
                want, _, bound, _ = attend(q[r, i:i + 1], p.k[0, s, h], p.v[0, s, h])
                assert np.all(np.abs(out[r, i:i + 1] - want) <= bound), (r, i)
            assert np.isnan(after[0, r, h, :lengths[r]]).all() == (odd // 4 == h)
            assert np.array_equal(after[0, r, h, lengths[r]:], before[0, r, h, lengths[r]:])
    p.free()


def test_attention_without_scratch(rng):
    """Scratch that cannot be had is an error, and the next call works."""
    with HipBackend(0) as hip:
        p = Paged(hip, rng, [60000], 64, 8, scored=True)
        hip.set_scratch_limit(1 << 20)
        with pytest.raises(GhError) as e:
            run_attention(hip, p, 32, rng)
        assert e.value.code == -4
        hip.set_scratch_limit(0)
        before = p.read("score")
        q, out = run_attention(hip, p, 32, rng)
        check_attention(p, 0, q, out, before, p.read("score"))
        p.free()


@pytest.mark.parametrize("scored,lengths,limit", [(False, [400, 90, 0, 511, 33, 500, 17, 1], 4 << 20),
                                                  (True, [3000, 100, 2000, 1, 700], 20 << 20)])
def test_attention_with_scratch_for_some_rows(rng, scored, lengths, limit):
    """Rows take turns in what scratch there is (all of it: 4.3 and 25 MB)."""
    with HipBackend(0) as hip:
        p = Paged(hip, rng, lengths, 16, 8, scored=scored)
        for n in (limit, 0):
            hip.set_scratch_limit(n)
            before = p.read("score") if scored else None
            q, out = run_attention(hip, p, 128, rng)
            check_attention(p, 0, q, out, before, p.read("score") if scored else None)
        p.free()


# ---- append ----

@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("page,heads,tokens,lengths", [
    (16, 8, 1, [1, 16, 17, 0, 500]), (64, 2, 1, [64, 65]), (32, 1, 40, [40, 100, 0, 33, 7]), (16, 3, 300, [300]),
])
def test_write(hip, rng, page, heads, tokens, lengths, scored):
    p = Paged(hip, rng, lengths, page, heads, layers=3, scored=scored)
    k, v = (rng.standard_normal((p.rows, tokens, heads, D)).astype(np.float16) for _ in range(2))
    kb, vb = hip.from_host(k), hip.from_host(v)
    hip.kv_write_paged(p.handle(), kb, vb, tokens, 1)
    for r, n in enumerate(lengths):
        t = min(tokens, n)  # what lies before the row's first position is skipped
        at = p.cells(r, n)[n - t:]
        p.k[1, at], p.v[1, at] = k[r, tokens - t:], v[r, tokens - t:]
        if scored:
            p.score[1, r, :, n - t:n] = 0
    for name in ("k", "v") + (("score",) if scored else ()):
        assert np.array_equal(p.read(name).view(np.uint8), getattr(p, name).view(np.uint8)), name
    hip.free_buffer(kb)
    hip.free_buffer(vb)
    p.free()


@pytest.mark.parametrize("rope_dim", [128, 64, 6])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("heads,group,tokens", [(8, 4, 1), (2, 3, 5)])
def test_rope_write_has_the_bits_of_the_single_operations(hip, rng, rope_dim, in_place, heads, group, tokens):
    yarn = Yarn(rope_dim, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    lengths, q_heads = [20, 0, 6, 33], heads * group
    positions = np.array([0, 5, 20000, 700], np.uint32)
    p = Paged(hip, rng, lengths, 16, heads, layers=2)
    q = rng.standard_normal((4, tokens, q_heads, D)).astype(np.float16)
    k, v = (rng.standard_normal((4, tokens, heads, D)).astype(np.float16) for _ in range(2))
    qb, kb, vb, pb = (hip.from_host(x) for x in (q, k, v, positions))
    ob = qb if in_place else hip.from_host(np.full_like(q, 7))
    hip.rope_kv_write_paged(p.handle(), ob, qb, kb, vb, q_heads, pb, tokens, 20000 + tokens - 1, yarn, 1)
    got = hip.download(ob, np.float16, q.size).reshape(q.shape)
    want_q = (q if in_place else np.full_like(q, 7)).copy()
    for r, n in enumerate(lengths):
        for t in range(tokens) if n else ():
            row = {}
            for name, x, role in (("q", q[r, t], F.ROPE_QUERY), ("k", k[r, t], F.ROPE_KEY)):
                b = hip.from_host(x)
                hip.rope_yarn(b, len(x), D, int(positions[r]) + t, yarn, role)
                row[name] = hip.download(b, np.float16, x.size).reshape(x.shape)
                hip.free_buffer(b)
            want_q[r, t] = row["q"]
            at = p.cells(r, n)[n - tokens + t]
            p.k[1, at], p.v[1, at] = row["k"], v[r, t]
    assert np.array_equal(got.view(np.uint16), want_q.view(np.uint16))
    for name in ("k", "v"):
        assert np.array_equal(p.read(name).view(np.uint16), getattr(p, name).view(np.uint16)), name
    for b in (qb, kb, vb, pb) + (() if in_place else (ob,)):
        hip.free_buffer(b)
    p.free()


# ---- eviction ----

def evict_case(hip, rng, lengths, page, heads, layers, budget, recent, score=None, use_kept=True, alias=False):
    src = Paged(hip, rng, lengths, page, heads, layers, scored=True, score=score)
    dst = Paged(hip, rng, [budget if n > budget else 0 for n in lengths], page, heads, layers, scored=True,
                width=src.width if alias else pages_of(budget, page))
    dst.lengths = src.lengths.copy() if alias else np.arange(90, 90 + len(lengths), dtype=np.uint32)
    dst.upload()
    if alias:
        dst.score = src.score.copy()
        hip.free_buffer(dst.bufs["score"])
        hip.free_buffer(dst.bufs["lengths"])
        dst.bufs["score"], dst.bufs["lengths"] = src.bufs["score"], src.bufs["lengths"]
    kept = np.full((layers, len(lengths), heads, budget), 0xABCD, np.uint32)
    kb = hip.from_host(kept) if use_kept else None
    hip.kv_evict_paged(dst.handle(), src.handle(), kb, budget, recent)
    for r, n in enumerate(lengths):
        if n <= budget:
            continue
        dst.lengths[r] = budget
        old, new = src.cells(r, n), dst.cells(r, budget)
        for layer in range(layers):
            for h in range(heads):
                best = keep(src.score[layer, r, h, :n], budget, recent)
                kept[layer, r, h] = best
                dst.score[layer, r, h, :budget] = src.score[layer, r, h, best]
                dst.k[layer, new, h], dst.v[layer, new, h] = src.k[layer, old[best], h], src.v[layer, old[best], h]
    if use_kept:
        assert np.array_equal(hip.download(kb, np.uint32, kept.size).reshape(kept.shape), kept)
        hip.free_buffer(kb)
    for name in ("score", "lengths", "k", "v"):
        assert np.array_equal(dst.read(name).view(np.uint8), getattr(dst, name).view(np.uint8)), name
    for name in ("k", "v", "table") + (() if alias else ("lengths", "score")):
        assert np.array_equal(src.read(name).view(np.uint8), getattr(src, name).view(np.uint8)), "source " + name
    if alias:
        dst.bufs.pop("score"), dst.bufs.pop("lengths")
    src.free()
    dst.free()


@pytest.mark.parametrize("lengths,page,heads,layers,budget,recent", [
    ([2], 16, 1, 1, 1, 0), ([2], 16, 1, 1, 1, 1), ([17, 16, 0, 40], 16, 2, 2, 16, 3), ([600, 601, 64], 32, 8, 3, 560, 64),
    ([5000, 4097, 2049], 64, 2, 2, 2048, 256), ([300], 128, 3, 1, 299, 0), ([300], 16, 3, 1, 200, 200),
    ([20001], 256, 1, 1, 7001, 1), ([100, 50], 16, 5, 2, 200, 10),
    ([8300], 64, 8, 4, 8200, 100),  # 128 MiB are moved
])
@pytest.mark.parametrize("alias", [False, True])
def test_evict(hip, rng, lengths, page, heads, layers, budget, recent, alias):
    evict_case(hip, rng, lengths, page, heads, layers, budget, recent, use_kept=not alias,
               alias=alias and budget <= pages_of(max(lengths), page) * page)


@pytest.mark.parametrize("kind", ["zeros", "few_values", "signs", "not_finite", "denormal"])
@pytest.mark.parametrize("budget,recent", [(1000, 0), (1000, 100), (2900, 500)])
def test_evict_order_of_scores(hip, rng, kind, budget, recent):
    """Equal scores keep the first; the order is f32's total order (-NaN < -inf < ... -0 < +0 ... < NaN)."""
    n = 3003
    if kind == "zeros":
        s = np.zeros(n)
    elif kind == "few_values":
        s = rng.integers(0, 4, n)
    elif kind == "signs":
        s = np.where(rng.random(n) < 0.5, -0.0, rng.standard_normal(n))
    elif kind == "denormal":
        s = rng.integers(0, 50, n) * np.float64(np.finfo(np.float32).smallest_subnormal)
    else:
        s = rng.choice(np.array([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0]), n)
    s = np.resize(s.astype(np.float32), pages_of(n, 16) * 16)
    evict_case(hip, rng, [n, n - 1], 16, 2, 1, budget, recent, score=s)


def test_evict_leaves_shared_pages_alone(hip, rng):
    """Two rows over one prompt: the longer is evicted, the other's cache keeps its bytes (evict_case checks
    that of the whole source)."""
    src = Paged(hip, rng, [400, 200], 16, 2, scored=True)
    src.table[1, :12] = src.table[0, :12]
    src.upload()
    dst = Paged(hip, rng, [250, 0], 16, 2, scored=True)
    hip.kv_evict_paged(dst.handle(), src.handle(), None, 250, 50)
    assert np.array_equal(src.read("k").view(np.uint16), src.k.view(np.uint16))
    best = keep(src.score[0, 0, 1, :400], 250, 50)
    assert np.array_equal(dst.read("v")[0, dst.cells(0, 250), 1], src.v[0, src.cells(0, 400)[best], 1])
    assert list(dst.read("lengths")) == [250, 0]
    src.free()
    dst.free()


# ---- what the host cannot check ----

def test_bad_device_data_is_an_error_of_its_row(hip, rng):
    """A length beyond the table, a page beyond the pool, a position beyond max_pos: GH_E_RANGE at the submit,
    other rows as ever, and the next call works."""
    p = Paged(hip, rng, [100, 90, 300], 16, 2, scored=True)
    good_lengths, good_table = p.lengths.copy(), p.table.copy()
    q = rng.standard_normal((3, 8, D)).astype(np.float16)
    k = rng.standard_normal((3, 1, 2, D)).astype(np.float16)
    qb, ob, kb = hip.from_host(q), hip.alloc_buffer(q.nbytes), hip.from_host(k)
    pb = hip.from_host(np.array([3, 9, 5], np.uint32))
    dst = Paged(hip, rng, [50, 50, 50], 16, 2, scored=True)

    def calls():
        yield "write", lambda: hip.kv_write_paged(p.handle(), kb, kb, 1, 0)
        yield "attend", lambda: hip.attention_decode_paged(ob, qb, p.handle(), 8, 0, 0)
        yield "evict", lambda: hip.kv_evict_paged(dst.handle(), p.handle(), None, 50, 10)

    for bad in ("length", "page"):
        p.lengths, p.table = good_lengths.copy(), good_table.copy()
        if bad == "length":
            p.lengths[1] = p.width * 16 + 1
        else:
            p.table[1, :6] = p.slots // 16  # the first page beyond the pool
        p.upload()
        for name, call in calls():
            with pytest.raises(GhError) as e:
                call()
            assert e.value.code == -5, (bad, name)
            if name == "attend":
                out = hip.download(ob, np.float16, q.size).reshape(q.shape)
                now = p.read("k"), p.read("v")
                for r in (0, 2):
                    s = p.cells(r, int(good_lengths[r]))
                    want, _, bound, _ = attend(q[r, :4], now[0][0, s, 0], now[1][0, s, 0])
                    assert np.all(np.abs(out[r, :4] - want) <= bound)
            if name == "evict":
                assert dst.read("lengths")[0] == 50 and dst.read("lengths")[2] == 50
    p.lengths, p.table = good_lengths, good_table
    p.upload()
    with pytest.raises(GhError) as e:
        hip.rope_kv_write_paged(p.handle(), ob, qb, kb, kb, 8, pb, 1, 8, YARN, 0)
    assert e.value.code == -5
    hip.rope_kv_write_paged(p.handle(), ob, qb, kb, kb, 8, pb, 1, 9, YARN, 0)
    for _, call in calls():
        call()
    for b in (qb, ob, kb, pb):
        hip.free_buffer(b)
    p.free()
    dst.free()


def test_longer_rows_than_the_call_says(hip, rng):
    """A row past max_len is an error of that row; the others and what lies behind the last row are as ever."""
    p = Paged(hip, rng, [40, 300, 33], 16, 2, scored=True)
    q = rng.standard_normal((3, 8, D)).astype(np.float16)
    qb, ob = hip.from_host(q), hip.from_host(np.full((4, 8, D), 7, np.float16))
    before = p.read("score")
    with pytest.raises(GhError) as e:
        hip.attention_decode_paged(ob, qb, p.handle(), 8, 299, 0)
    assert e.value.code == -5
    out, after = hip.download(ob, np.float16, 4 * 8 * D).reshape(4, 8, D), p.read("score")
    for r in (0, 2):
        s = p.cells(r, int(p.lengths[r]))
        want, _, bound, _ = attend(q[r, 4:], p.k[0, s, 1], p.v[0, s, 1])
        assert np.all(np.abs(out[r, 4:] - want) <= bound)
    assert np.all(out[3] == 7) and np.array_equal(after[0, 1], before[0, 1])
    for b in (qb, ob):
        hip.free_buffer(b)
    p.free()


def test_what_lies_behind_the_last_row_stays(hip, rng):
    """Buffers with room for one more row: no operator writes there."""
    p, heads, group = Paged(hip, rng, [30, 0, 65], 16, 2, scored=True), 2, 4
    q = rng.standard_normal((4, heads * group, D)).astype(np.float16)
    k = rng.standard_normal((3, heads, D)).astype(np.float16)
    qb, kb, pb = hip.from_host(q), hip.from_host(k), hip.from_host(np.array([3, 4, 5], np.uint32))
    mark = np.full((4, heads * group, D), 7, np.float16)
    ob, rb = hip.from_host(mark), hip.from_host(mark)
    hip.rope_kv_write_paged(p.handle(), rb, qb, kb, kb, heads * group, pb, 1, 5, YARN, 0)
    hip.attention_decode_paged(ob, rb, p.handle(), heads * group, 0, 0)
    for b in (ob, rb):
        assert np.all(hip.download(b, np.float16, mark.size).reshape(mark.shape)[3] == 7)
    dst = Paged(hip, rng, [20, 0, 20], 16, 2, scored=True)
    kept = hip.from_host(np.full((4, 2, 20), 99, np.uint32))
    lengths = hip.from_host(np.full(4, 99, np.uint32))
    h = dst.handle()
    h.lengths = lengths
    hip.kv_evict_paged(h, p.handle(), kept, 20, 5)
    got = hip.download(kept, np.uint32, 160).reshape(4, 2, 20)
    assert np.all(got[[1, 3]] == 99) and not np.any(got[[0, 2]] == 99)
    assert list(hip.download(lengths, np.uint32, 4)) == [20, 99, 20, 99]
    for b in (qb, kb, pb, ob, rb, kept, lengths):
        hip.free_buffer(b)
    p.free()
    dst.free()


# ---- together ----

def test_two_backends_at_once(rng):
    """Two backends (a stream and scratch each) in two threads over one pool."""
    with HipBackend(0) as a, HipBackend(0) as b:
        p = Paged(a, rng, [5000, 0, 77, 3000], 16, 4)
        q = [rng.standard_normal((4, 16, D)).astype(np.float16) for _ in range(2)]
        got = [[], []]

        def work(i, hip):
            qb, ob = hip.from_host(q[i]), hip.alloc_buffer(q[i].nbytes)
            for _ in range(20):
                hip.attention_decode_paged(ob, qb, p.handle(), 16, 0, 0)
                got[i].append(hip.download(ob, np.float16, q[i].size).reshape(q[i].shape))
            hip.free_buffer(qb)
            hip.free_buffer(ob)

        threads = [threading.Thread(target=work, args=(i, hip)) for i, hip in enumerate((a, b))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for i in range(2):
            assert len(got[i]) == 20
            check_attention(p, 0, q[i], got[i][0])
            assert all(np.array_equal(x.view(np.uint16), got[i][0].view(np.uint16)) for x in got[i])
        p.free()


def test_recorded_decode_graphs_survive_the_scratch_of_paged_attention(rng):
    """Paged attention that moves the backend's workspace between two runs of a model's replayed decode."""
    shape = synth.SHAPES["tiny"]
    with HipBackend(0) as hip:
        m = HipModel(hip, synth.model_config(shape, 64, 16))
        for layer, tid, fmt, data in synth.model_tensors(shape, 1):
            m.load_tensor(layer, tid, fmt, data)
        m.prefill(np.arange(8), 0)
        first = m.decode_greedy(3, 8, 12)
        before = hip.scratch_info()[0]
        p = Paged(hip, rng, [9000] * 6, 64, 2, scored=True)
        old = p.read("score")
        q, out = run_attention(hip, p, 16, rng)
        check_attention(p, 0, q, out, old, p.read("score"))
        assert hip.scratch_info()[0] > before
        assert np.array_equal(m.decode_greedy(3, 8, 12), first)
        p.free()
        m.close()


def test_serving_run(hip, rng):
    """Prompts go into pages, then steps of append and attention over two layers in one encoder each, an
    eviction in between (rows go on in their new pages), against a restatement that holds every row's
    vectors in lists."""
    heads, group, page, layers, width, budget, recent = 2, 4, 16, 2, 12, 40, 8
    prompts = [50, 0, 17, 90]
    rows, q_heads, slots = len(prompts), heads * group, page * 64
    kc, vc = (hip.from_host(np.full((layers, slots, heads, D), np.nan, np.float16)) for _ in range(2))
    free = list(rng.permutation(slots // page))
    tables = [[free.pop() for _ in range(width)] for _ in range(rows)]
    table = hip.from_host(np.array(tables, np.uint32))
    lengths_b, pos_b = hip.alloc_buffer(4 * rows), hip.alloc_buffer(4 * rows)
    score = hip.from_host(np.zeros((layers, rows, heads, width * page), np.float32))
    pool = F.GhKv(kc, vc, F.KV_F16, layers, slots, heads, D, D)
    kv = GhKvPaged(pool, table, lengths_b, score, page, width, rows)
    lengths = np.array(prompts, np.uint32)
    position = lengths.copy()
    # per layer and row: K, V [n][heads][128] and scores [heads][n]
    state = [[(np.zeros((0, heads, D), np.float16),) * 2 + (np.zeros((heads, 0)),) for _ in range(rows)]
             for _ in range(layers)]

    def append(layer, r, k, v):
        a, b, s = state[layer][r]
        state[layer][r] = np.concatenate([a, k]), np.concatenate([b, v]), np.pad(s, ((0, 0), (0, len(k))))

    # the prompts: prefilled elsewhere (as random vectors), moved in by rows
    for r, n in enumerate(prompts):
        if n == 0:
            continue
        only = np.where(np.arange(rows) == r, lengths, 0).astype(np.uint32)
        hip.upload(lengths_b, only)
        for layer in range(layers):
            k, v = (rng.standard_normal((rows, n, heads, D)).astype(np.float16) for _ in range(2))
            kb, vb = hip.from_host(k), hip.from_host(v)
            hip.kv_write_paged(kv, kb, vb, n, layer)
            append(layer, r, k[r], v[r])
            hip.free_buffer(kb)
            hip.free_buffer(vb)

    def rope(x, pos, role):
        b = hip.from_host(x)
        hip.rope_yarn(b, len(x), D, int(pos), YARN, role)
        y = hip.download(b, np.float16, x.size).reshape(x.shape)
        hip.free_buffer(b)
        return y

    shape = (rows, q_heads, D)
    for step in range(12):
        if step == 4:
            lengths[1], position[1] = 0, 0  # a new sequence takes the free row
        live = np.array([r != 1 or step >= 4 for r in range(rows)])
        lengths[live] += 1
        hip.upload(lengths_b, np.where(live, lengths, 0).astype(np.uint32))
        hip.upload(pos_b, position)
        data = [(rng.standard_normal(shape).astype(np.float16), *(rng.standard_normal((rows, heads, D)).astype(np.float16)
                 for _ in range(2))) for _ in range(layers)]
        bufs = [[hip.from_host(x) for x in d] + [hip.alloc_buffer(2 * rows * q_heads * D) for _ in range(2)] for d in data]
        hip.begin()
        for layer, (qb, kb, vb, rb, ob) in enumerate(bufs):
            hip.rope_kv_write_paged(kv, rb, qb, kb, vb, q_heads, pos_b, 1, 300, YARN, layer)
            hip.attention_decode_paged(ob, rb, kv, q_heads, 0, layer)
        hip.submit()
        got_score = hip.download(score, np.float32, layers * rows * heads * width * page)
        got_score = got_score.reshape(layers, rows, heads, width * page)
        for layer, (q, k, v) in enumerate(data):
            out = hip.download(bufs[layer][4], np.float16, q.size).reshape(shape)
            for r in range(rows):
                if not live[r]:
                    assert not out[r].any()
                    continue
                append(layer, r, rope(k[r], position[r], F.ROPE_KEY)[None], v[r][None])
                a, b, s = state[layer][r]
                assert len(a) == lengths[r]
                turned = rope(q[r], position[r], F.ROPE_QUERY)
                for h in range(heads):
                    want, w, bound, wb = attend(turned[h * group:(h + 1) * group], a[:, h], b[:, h])
                    assert np.all(np.abs(out[r, h * group:(h + 1) * group] - want) <= bound), (step, layer, r, h)
                    got = got_score[layer, r, h, :len(a)].astype(np.float64)
                    s[h] += w.sum(0)
                    assert np.all(np.abs(got - s[h]) <= wb.sum(0) + 1e-6 * s[h] + 1e-7), (step, layer, r, h)
                    s[h] = got  # the operator's own sums decide an eviction
        for bs in bufs:
            for x in bs:
                hip.free_buffer(x)
        position[live] += 1
        if step in (5, 9):
            out_of = [r for r in range(rows) if live[r] and lengths[r] > budget]
            fresh = [list(t) for t in tables]
            for r in out_of:
                fresh[r] = [free.pop() for _ in range(pages_of(budget, page))]
            new_table = np.full((rows, width), 0xFFFFFFFF, np.uint32)
            for r in out_of:
                new_table[r, :len(fresh[r])] = fresh[r]
            tb = hip.from_host(new_table)
            hip.kv_evict_paged(GhKvPaged(pool, tb, lengths_b, score, page, width, rows), kv, None, budget, recent)
            now = hip.download(lengths_b, np.uint32, rows)
            for r in out_of:
                assert now[r] == budget
                lengths[r] = budget
                free.extend(tables[r])
                fresh[r] += [free.pop(0) for _ in range(width - len(fresh[r]))]
                tables[r] = fresh[r]
                for layer in range(layers):
                    a, b, s = state[layer][r]
                    best = [keep(s[h].astype(np.float32), budget, recent) for h in range(heads)]
                    state[layer][r] = (np.stack([a[best[h], h] for h in range(heads)], 1),
                                       np.stack([b[best[h], h] for h in range(heads)], 1),
                                       np.stack([s[h, best[h]] for h in range(heads)]))
            hip.upload(table, np.array(tables, np.uint32))
            hip.free_buffer(tb)
    for b in (kc, vc, table, lengths_b, pos_b, score):
        hip.free_buffer(b)


def test_prefill_into_a_run_of_pages(hip, rng):
    """A prompt whose pages lie in a row is written and prefilled by the contiguous operators through a view of
    the pool; decode goes on over the same pages."""
    heads, group, page, n, slots = 2, 4, 16, 75, 16 * 20
    q_heads, row = heads * group, heads * 256
    kc, vc = (hip.from_host(np.full((2, slots, heads, D), np.nan, np.float16)) for _ in range(2))
    layer, first, count = 1, 7, pages_of(n + 1, page)
    at = (layer * slots + first * page) * row
    part = F.GhKv(hip.view(kc, at, count * page * row), hip.view(vc, at, count * page * row), F.KV_F16, 1, count * page, heads, D, D)
    k, v = (rng.standard_normal((n + 1, heads, D)).astype(np.float16) for _ in range(2))
    q = rng.standard_normal((n + 1, q_heads, D)).astype(np.float16)
    kb, vb, qb = hip.from_host(k[:n]), hip.from_host(v[:n]), hip.from_host(q[:n])
    ob = hip.alloc_buffer(q.nbytes)
    hip.begin()
    hip.kv_write(part, kb, vb, 0, 0, n * heads)
    hip.attention_prefill(ob, qb, part, q_heads, 0, n, 0)
    hip.submit()
    table, lengths = hip.from_host(np.arange(first, first + count, dtype=np.uint32)), hip.from_host(np.array([n + 1], np.uint32))
    kv = GhKvPaged(F.GhKv(kc, vc, F.KV_F16, 2, slots, heads, D, D), table, lengths, F.GhBuf(), page, count, 1)
    k1, v1, q1 = hip.from_host(k[n:]), hip.from_host(v[n:]), hip.from_host(q[n:])
    hip.begin()
    hip.kv_write_paged(kv, k1, v1, 1, layer)
    hip.attention_decode_paged(ob, q1, kv, q_heads, 0, layer)
    hip.submit()
    out = hip.download(ob, np.float16, q_heads * D).reshape(q_heads, D)
    for h in range(heads):
        want, _, bound, _ = attend(q[n, h * group:(h + 1) * group], k[:, h], v[:, h])
        assert np.all(np.abs(out[h * group:(h + 1) * group] - want) <= bound)
    for b in (kc, vc, kb, vb, qb, ob, table, lengths, k1, v1, q1):
        hip.free_buffer(b)


@pytest.mark.parametrize("lengths", [[200, 90, 20], [7000, 20, 3000, 40]])  # both divisions of the work
def test_attention_of_scores_of_minus_infinity(hip, rng, lengths):
    """Such a position has weight 0: times an infinite V that is NaN, in its dim alone, and a row of nothing else is
    0 / 0, whether one wave or many have it."""
    p = Paged(hip, rng, lengths, 16, 8)
    cells = [p.cells(r, n) for r, n in enumerate(lengths)]
    p.k[0, cells[0][[7, 60]], 0, 0] = np.inf  # head 0 of row 0: two positions
    p.v[0, cells[0][7], 0, 5] = np.inf
    p.v[0, cells[0][60], 0, 6] = -np.inf
    p.v[0, cells[0][8], 0, 7] = np.inf  # a weight like any other
    for r in range(len(lengths)):  # head 1 of all rows: every position
        p.k[0, cells[r], 1, 0] = np.inf
    p.upload()
    q = np.abs(rng.standard_normal((len(lengths), 32, D))).astype(np.float16)
    q[:, :, 0] = -1
    q, out = run_attention(hip, p, 32, rng, q=q)
    assert np.isnan(out[0, :4, 5]).all() and np.isnan(out[0, :4, 6]).all() and np.all(out[0, :4, 7] == np.inf)
    seen = np.delete(cells[0], [7, 60])
    v = p.v[0, seen, 0].copy()
    v[7, 7] = 0
    want, _, bound, _ = attend(q[0, :4], p.k[0, seen, 0], v)
    dims = np.r_[:5, 8:D]
    assert np.all(np.abs(out[0, :4] - want)[:, dims] <= bound[:, dims])
    assert np.isnan(out[:, 4:8]).all()
    for r in range(len(lengths)):
        want, _, bound, _ = attend(q[r, 8:12], p.k[0, cells[r], 2], p.v[0, cells[r], 2])
        assert np.all(np.abs(out[r, 8:12] - want) <= bound)
    p.free()


def test_attention_without_memory_does_not_ask_each_time(rng):
    """Calls after the first keep the scratch that it found; with memory again the rows go together."""
    with HipBackend(0) as hip:
        p = Paged(hip, rng, [3000, 100, 2000, 1, 700], 16, 8, scored=True)
        hip.set_scratch_limit(20 << 20)  # all rows: 25 MB
        q = None
        for call in range(4):
            before = p.read("score")
            q, out = run_attention(hip, p, 128, rng, q=q)
            check_attention(p, 0, q, out, before, p.read("score"))
            info = hip.scratch_info()
            assert call == 0 or info == last
            last = info
        hip.set_scratch_limit(0)
        before = p.read("score")
        q, out = run_attention(hip, p, 128, rng, q=q)
        check_attention(p, 0, q, out, before, p.read("score"))
        assert hip.scratch_info()[0] > last[0]
        p.free()


def test_attention_of_growing_rows_seldom_moves_its_scratch(rng):
    """The call's longest row from 600 to 3000 in steps of 16: five times half as much again."""
    with HipBackend(0) as hip:
        p = Paged(hip, rng, [3000] * 8, 16, 8, scored=True)
        qb = hip.from_host(rng.standard_normal((8, 128, D)).astype(np.float16))
        ob, lengths = hip.alloc_buffer(qb.bytes), p.bufs["lengths"]
        sizes = []
        for n in range(600, 3001, 16):
            hip.upload(lengths, np.full(8, n, np.uint32))
            hip.attention_decode_paged(ob, qb, p.handle(), 128, n, 0)
            sizes.append(hip.scratch_info()[0])
        assert len(set(sizes)) <= 6
        hip.free_buffer(qb)
        hip.free_buffer(ob)
        p.free()


# ---- batches of many rows, chunks of many tiles ----

def many_lengths(rng, rows, most):
    """Rows up to `most`, some free, one of them at the front, the last one whole."""
    lengths = [int(n) for n in rng.integers(1, most + 1, rows)]
    for r in rng.choice(rows, rows // 10, replace=False):
        lengths[r] = 0
    lengths[0], lengths[-1] = 0, most
    return lengths


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("rows,heads,most,width", [
    (64, 4, 700, 64), (65, 4, 700, 64),   # chunks, up to 64 rows and past them
    (130, 2, 300, 64), (300, 2, 150, 64), (512, 1, 100, 40), (600, 1, 120, 40),  # chunks, 600 in two groups
    (100, 1, 300, 19),                    # spans, five a row
    (600, 2, 90, 6),                      # spans, one a row, two groups of rows
])
def test_attention_of_many_rows(hip, rng, rows, heads, most, width, scored):
    p = Paged(hip, rng, many_lengths(rng, rows, most), 16, heads, width=width, scored=scored)
    before = p.read("score") if scored else None
    q, out = run_attention(hip, p, 4 * heads, rng)
    check_attention(p, 0, q, out, before, p.read("score") if scored else None)
    p.free()


@pytest.mark.parametrize("scored", [False, True])
def test_attention_of_many_tiles_a_wave(hip, rng, scored):
    """64 kv heads: 32 chunks of 79 tiles, more than a wave looks up at once, with rows that begin at tiles 65, 66 and 69 of
    a chunk. Rows go over the same pages again and again."""
    heads, lengths = 64, [20000, 5, 1300, 19003]
    p = Paged(hip, rng, [256] * 4, 16, heads, width=1250, scored=scored)
    used = p.table[:, :16].ravel()
    p.table = rng.choice(used, (4, 1250)).astype(np.uint32)
    p.lengths = np.array(lengths, np.uint32)
    hip.upload(p.bufs["table"], p.table)
    hip.upload(p.bufs["lengths"], p.lengths)
    before = p.read("score") if scored else None
    q, out = run_attention(hip, p, 2 * heads, rng)
    after = p.read("score") if scored else None
    for r, n in enumerate(lengths):
        s = p.cells(r, n)
        for h in (0, 3, 31, 62, 63):
            want, w, bound, wb = attend(q[r, 2 * h:2 * h + 2], p.k[0, s, h], p.v[0, s, h])
            assert np.all(np.abs(out[r, 2 * h:2 * h + 2] - want) <= bound), (r, h)
            if scored:
                total = before[0, r, h, :n].astype(np.float64) + w.sum(0)
                assert np.all(np.abs(after[0, r, h, :n] - total) <= wb.sum(0) + 3 * 2.0 ** -24 * total), (r, h)
                assert np.array_equal(after[0, r, h, n:], before[0, r, h, n:])
    p.free()


# ---- what the host cannot check, in every division of the work ----

@pytest.mark.parametrize("bad", ["length", "max_len", "page", "last_page"])
@pytest.mark.parametrize("rows,heads,most,width", [
    (24, 8, 700, 100), (80, 2, 700, 64),  # chunks
    (3, 2, 300, 19), (100, 1, 300, 19),   # spans
])
def test_attention_of_bad_rows_leaves_the_others_alone(hip, rng, rows, heads, most, width, bad):
    """GH_E_RANGE at the submit; other rows' outputs and scores are as ever, and so are all scores past the rows. The
    next call works."""
    p = Paged(hip, rng, many_lengths(rng, rows, most), 16, heads, width=width, scored=True)
    odd = rows // 2
    if p.lengths[odd] < 40:  # of the length before it
        p.lengths[odd], p.table[odd] = p.lengths[-1], p.table[-1]
    good_lengths, good_table = p.lengths.copy(), p.table.copy()
    n = int(good_lengths[odd])
    max_len = 0
    if bad == "length":
        p.lengths[odd] = 16 * width + 1
    elif bad == "max_len":
        max_len = most
        p.lengths[odd] = most + 1
        if most + 1 <= 16 * width:
            p.table[odd] = p.table[-1, 0]
    else:
        p.table[odd, 1 if bad == "page" else (n - 1) // 16] = p.slots // 16 if bad == "page" else 0xFFFFFFFF
    p.upload()
    before = p.read("score")
    q = rng.standard_normal((rows, 4 * heads, D)).astype(np.float16)
    qb, ob = hip.from_host(q), hip.from_host(np.full((rows + 1, 4 * heads, D), 7, np.float16))
    with pytest.raises(GhError) as e:
        hip.attention_decode_paged(ob, qb, p.handle(), 4 * heads, max_len, 0)
    assert e.value.code == -5
    out, after = hip.download(ob, np.float16, (rows + 1) * 4 * heads * D).reshape(rows + 1, 4 * heads, D), p.read("score")
    assert np.all(out[rows] == 7)
    others = np.arange(rows) != odd
    p.lengths = np.where(others, good_lengths, 0)
    out[odd] = 0
    after[:, odd] = before[:, odd]
    check_attention(p, 0, q, out[:rows], before, after)
    p.lengths, p.table = good_lengths, good_table
    p.upload()
    hip.attention_decode_paged(ob, qb, p.handle(), 4 * heads, max_len, 0)
    got = hip.download(ob, np.float16, rows * 4 * heads * D).reshape(rows, 4 * heads, D)
    check_attention(p, 0, q, got)
    for b in (qb, ob):
        hip.free_buffer(b)
    p.free()


@pytest.mark.parametrize("bad", ["length", "page"])
@pytest.mark.parametrize("tokens", [1, 5])
def test_writes_of_bad_rows_leave_everything_else_alone(hip, rng, bad, tokens):
    """The whole pool and the scores: rows 0 and 2 have their vectors, nothing else changed."""
    p = Paged(hip, rng, [100, 96, 300], 16, 2, layers=2, scored=True)
    good = p.lengths.copy()
    at = [p.cells(r, int(good[r]))[-tokens:] for r in range(3)]
    if bad == "length":
        p.lengths[1] = 16 * p.width + 1
    else:
        p.table[1, 5] = p.slots // 16  # the page of all its new positions
    p.upload()
    k, v = (rng.standard_normal((3, tokens, 2, D)).astype(np.float16) for _ in range(2))
    kb, vb = hip.from_host(k), hip.from_host(v)
    with pytest.raises(GhError) as e:
        hip.kv_write_paged(p.handle(), kb, vb, tokens, 1)
    assert e.value.code == -5
    for r in (0, 2):
        p.k[1, at[r]], p.v[1, at[r]] = k[r], v[r]
        p.score[1, r, :, int(good[r]) - tokens:int(good[r])] = 0
    for name in ("k", "v", "score", "table", "lengths"):
        assert np.array_equal(p.read(name).view(np.uint8), getattr(p, name).view(np.uint8)), name
    hip.free_buffer(kb)
    hip.free_buffer(vb)
    p.free()


@pytest.mark.parametrize("tokens", [1, 5])
@pytest.mark.parametrize("over", [1, 3])
def test_positions_past_max_pos_touch_no_memory(hip, rng, tokens, over):
    """Of a row whose last `over` tokens lie past max_pos those are skipped, in the queries, the pool and the scores."""
    heads, group, max_pos = 2, 4, 500
    lengths, q_heads = [100, 96, 300], heads * group
    p = Paged(hip, rng, lengths, 16, heads, scored=True)
    positions = np.array([7, max_pos - tokens + 1 + over, 450], np.uint32)
    q = rng.standard_normal((3, tokens, q_heads, D)).astype(np.float16)
    k, v = (rng.standard_normal((3, tokens, heads, D)).astype(np.float16) for _ in range(2))
    qb, kb, vb, pb, ob = (hip.from_host(x) for x in (q, k, v, positions, np.full_like(q, 7)))
    with pytest.raises(GhError) as e:
        hip.rope_kv_write_paged(p.handle(), ob, qb, kb, vb, q_heads, pb, tokens, max_pos, YARN, 0)
    assert e.value.code == -5
    got = hip.download(ob, np.float16, q.size).reshape(q.shape)
    skipped = np.zeros((3, tokens), bool)
    skipped[1, max(0, tokens - over):] = True
    for r in range(3):
        for t in range(tokens):
            at = p.cells(r, lengths[r])[lengths[r] - tokens + t]
            if skipped[r, t]:
                assert np.all(got[r, t] == 7)
                continue
            for name, x, role in (("q", q[r, t], F.ROPE_QUERY), ("k", k[r, t], F.ROPE_KEY)):
                b = hip.from_host(x)
                hip.rope_yarn(b, len(x), D, int(positions[r]) + t, YARN, role)
                y = hip.download(b, np.float16, x.size).reshape(x.shape)
                hip.free_buffer(b)
                if name == "q":
                    assert np.array_equal(got[r, t].view(np.uint16), y.view(np.uint16))
                else:
                    p.k[0, at] = y
            p.v[0, at] = v[r, t]
            p.score[0, r, :, lengths[r] - tokens + t] = 0
    for name in ("k", "v", "score"):
        assert np.array_equal(p.read(name).view(np.uint8), getattr(p, name).view(np.uint8)), name
    for b in (qb, kb, vb, pb, ob):
        hip.free_buffer(b)
    p.free()


def test_rope_write_at_far_positions_has_the_bits_of_the_single_operations(hip, rng):
    """Past the original context, where queries have a temperature, and up to the last position of the table."""
    positions = np.array([16383, 16384, 100001, 262142], np.uint32)
    p = Paged(hip, rng, [20, 30, 2, 33], 16, 2)
    q = rng.standard_normal((4, 2, 8, D)).astype(np.float16)
    k, v = (rng.standard_normal((4, 2, 2, D)).astype(np.float16) for _ in range(2))
    qb, kb, vb, pb, ob = (hip.from_host(x) for x in (q, k, v, positions, q))
    hip.rope_kv_write_paged(p.handle(), ob, qb, kb, vb, 8, pb, 2, 262143, YARN, 0)
    got, pool = hip.download(ob, np.float16, q.size).reshape(q.shape), p.read("k")
    for r in range(4):
        for t in range(2):
            at = p.cells(r, int(p.lengths[r]))[int(p.lengths[r]) - 2 + t]
            for x, y, role in ((q[r, t], got[r, t], F.ROPE_QUERY), (k[r, t], pool[0, at], F.ROPE_KEY)):
                b = hip.from_host(x)
                hip.rope_yarn(b, len(x), D, int(positions[r]) + t, YARN, role)
                assert np.array_equal(hip.download(b, np.float16, x.size).view(np.uint16), y.ravel().view(np.uint16))
                hip.free_buffer(b)
    for b in (qb, kb, vb, pb, ob):
        hip.free_buffer(b)
    p.free()


@pytest.mark.parametrize("bad", ["length", "page", "dst_page"])
@pytest.mark.parametrize("in_place", [False, True])
def test_eviction_of_bad_rows_leaves_the_others_alone(hip, rng, bad, in_place):
    """Row 1 has a length or a page that does not fit: rows 0 and 2 move as ever, row 3 stays, no page of another row is
    written, and of a row whose length is bad nothing is."""
    lengths, budget, recent, heads = [100, 90, 300, 40], 50, 10, 2
    src = Paged(hip, rng, lengths, 16, heads, 2, scored=True)
    dst = Paged(hip, rng, [budget] * 3 + [0], 16, heads, 2, scored=True, width=src.width if in_place else None, garbage=np.float16(3))
    dst.k[:], dst.v[:], dst.score[:] = 3, 4, -1
    dst.lengths = np.arange(90, 94, dtype=np.uint32)
    mine = dst.cells(1, 64)
    if bad == "length":
        src.lengths[1] = 16 * src.width + 1
    elif bad == "page":
        src.table[1, :6] = src.slots // 16
    else:
        dst.table[1, :4] = dst.slots // 16
    src.upload()
    dst.upload()
    if in_place:
        dst.score, dst.lengths = src.score.copy(), src.lengths.copy()
        for name in ("score", "lengths"):
            hip.free_buffer(dst.bufs[name])
            dst.bufs[name] = src.bufs[name]
    kept = hip.from_host(np.full((2, 4, heads, budget), 99999, np.uint32))
    with pytest.raises(GhError) as e:
        hip.kv_evict_paged(dst.handle(), src.handle(), kept, budget, recent)
    assert e.value.code == -5
    got = hip.download(kept, np.uint32, 8 * heads * budget).reshape(2, 4, heads, budget)
    want_kept = np.full_like(got, 99999)
    for r in (0, 2):
        dst.lengths[r] = budget
        old, new = src.cells(r, lengths[r]), dst.cells(r, budget)
        for layer in range(2):
            for h in range(heads):
                best = keep(src.score[layer, r, h, :lengths[r]], budget, recent)
                want_kept[layer, r, h] = best
                dst.score[layer, r, h, :budget] = src.score[layer, r, h, best]
                dst.k[layer, new, h], dst.v[layer, new, h] = src.k[layer, old[best], h], src.v[layer, old[best], h]
    now = {name: dst.read(name) for name in ("k", "v", "score", "lengths")}
    if bad != "length":  # its results are unspecified, within its own pages, scores, list and length
        got[:, 1] = want_kept[:, 1]
        now["score"][:, 1] = dst.score[:, 1]
        now["lengths"][1] = dst.lengths[1]
        now["k"][:, mine], now["v"][:, mine] = dst.k[:, mine], dst.v[:, mine]
    assert np.array_equal(got, want_kept)
    for name, x in now.items():
        assert np.array_equal(x.view(np.uint8), getattr(dst, name).view(np.uint8)), name
    for name in ("k", "v", "table") + (() if in_place else ("lengths", "score")):
        assert np.array_equal(src.read(name).view(np.uint8), getattr(src, name).view(np.uint8)), "source " + name
    hip.free_buffer(kept)
    if in_place:
        dst.bufs.pop("score"), dst.bufs.pop("lengths")
    src.free()
    dst.free()
