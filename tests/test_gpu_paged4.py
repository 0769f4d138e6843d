"""The operators over paged caches in 4 bits, and those over both schemes that came with them (the append with norms,
the read-back), against 64-bit definitions over the values that the pool's bytes stand for (tests/paged4.py)."""
import numpy as np
import pytest

from graph_horizon_amd import GhError, Yarn
from graph_horizon_amd import _ffi as F
from paged import D, Paged, keep, pages_of
from paged4 import VECTOR, Paged4, check_attention4, pack, parts, unpack

pytestmark = pytest.mark.gpu
YARN = Yarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
HALF = 2.0 ** -24  # FP32's half step


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
    "tile_edges": [15, 16, 17, 0, 31, 32, 33, 127, 128, 129, 1],
    "empty": [0, 0],
    "ragged": [1000, 3, 0, 257, 640, 129, 1],
    "long": [9001, 100],
}


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("name", list(LENGTHS))
@pytest.mark.parametrize("page,heads,group", [(16, 8, 4), (64, 2, 8), (32, 1, 1), (128, 5, 3), (16, 3, 16), (256, 1, 7)])
def test_attention(hip, rng, name, page, heads, group, scored):
    p = Paged4(hip, rng, LENGTHS[name], page, heads, layers=2, scored=scored)
    before = None if not scored else p.read("score")
    q, out = run_attention(hip, p, heads * group, rng, layer=1)
    check_attention4(p, 1, q, out, before, p.read("score") if scored else None)
    assert np.array_equal(p.read("k"), p.kb) and np.array_equal(p.read("v"), p.vb)
    for name in ("table", "lengths"):
        assert np.array_equal(p.read(name), getattr(p, name)), name
    p.free()


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("lengths,page,heads,width", [
    ([700] * 70 + [0, 3000, 5], 16, 8, 200),   # chunks over more than 64 rows
    ([4000, 0, 3100, 2999, 17, 1024] * 3, 32, 8, 130),  # chunks over few
    ([12345, 5000], 64, 8, 200),
    ([12345, 5000, 20], 64, 8, 2000),
    ([0] * 70, 16, 8, 300),                    # nothing in them
    ([0] * 20 + [1] + [0] * 30, 16, 8, 300),
    ([1, 33, 0, 64, 32] * 14, 16, 3, 300),     # as many chunks as tiles allow
])
def test_attention_in_chunks(hip, rng, lengths, page, heads, width, scored):
    p = Paged4(hip, rng, lengths, page, heads, width=width, scored=scored)
    before = p.read("score") if scored else None
    q, out = run_attention(hip, p, 2 * heads, rng)
    check_attention4(p, 0, q, out, before, p.read("score") if scored else None)
    p.free()


@pytest.mark.parametrize("heads,group", [(1, 4), (2, 3), (3, 2), (4, 1), (5, 2), (9, 1), (12, 4)])
def test_attention_in_chunks_of_any_number_of_heads(hip, rng, heads, group):
    """Teams of one to four waves, with and without waves over; a pool whose rows of all heads end off 128 bytes."""
    lengths = [int(n) for n in rng.integers(0, 400, 30)] + [2000, 0, 33]
    p = Paged4(hip, rng, lengths, 16, heads, width=16 * 1024 // 16, scored=heads % 2 == 1)
    before = p.read("score") if p.score is not None else None
    q, out = run_attention(hip, p, heads * group, rng)
    check_attention4(p, 0, q, out, before, None if before is None else p.read("score"))
    p.free()


def test_attention_past_the_cache(hip, rng):
    """128 MiB of vectors, from which they are read with another cache policy."""
    p = Paged4(hip, rng, [60000, 45000, 17], 64, 8, width=1000)
    q, out = run_attention(hip, p, 32, rng)
    check_attention4(p, 0, q, out)
    p.free()


@pytest.mark.parametrize("max_len", [300, 320, 1000, 4096])
@pytest.mark.parametrize("group", [2, 4])
def test_attention_launch_longer_than_rows(hip, rng, max_len, group):
    p = Paged4(hip, rng, [300, 0, 17], 16, 4, width=256, scored=True)
    before = p.read("score")
    q, out = run_attention(hip, p, 4 * group, rng, max_len=max_len)
    check_attention4(p, 0, q, out, before, p.read("score"))
    p.free()


def test_attention_row_groups(hip, rng):
    """More rows than one launch lays out."""
    lengths = [int(n) for n in rng.integers(0, 700, 600)]
    p = Paged4(hip, rng, lengths, 16, 1, scored=True)
    before = p.read("score")
    q, out = run_attention(hip, p, 2, rng)
    check_attention4(p, 0, q, out, before, p.read("score"))
    p.free()


@pytest.mark.parametrize("lengths,width", [([3000, 40, 1111], 188), ([2500, 0, 40, 700] * 8, 157)])
def test_attention_repeats_bit_for_bit_and_into_its_queries(hip, rng, lengths, width):
    p = Paged4(hip, rng, lengths, 16, 8, width=width)
    q, first = run_attention(hip, p, 32, rng)
    for _ in range(3):
        assert np.array_equal(run_attention(hip, p, 32, rng, q=q)[1].view(np.uint16), first.view(np.uint16))
    buf = hip.from_host(q)
    hip.attention_decode_paged(buf, buf, p.handle(), 32, 0, 0)
    assert np.array_equal(hip.download(buf, np.uint16, q.size).reshape(q.shape), first.view(np.uint16))
    hip.free_buffer(buf)
    p.free()


def test_attention_shared_and_repeated_pages(hip, rng):
    p = Paged4(hip, rng, [200, 200, 64], 16, 2)
    p.table[1, :8] = p.table[0, :8]
    p.table[2, :4] = p.table[2, [0, 1, 0, 1]]
    p.upload()
    q, out = run_attention(hip, p, 8, rng)
    check_attention4(p, 0, q, out)
    p.free()


@pytest.mark.parametrize("heads", [8, 1])
def test_attention_pool_past_4_gib(hip, rng, heads):
    """Pages whose byte offsets pass 32 bits (a pool of 4.5 GiB each for K and V)."""
    page, slots = 64, (9 << 29) // (VECTOR * heads) // 64 * 64
    lengths = [130, 70]
    small = Paged4(hip, rng, lengths, page, heads)
    kv = [hip.alloc_buffer(slots * heads * VECTOR) for _ in range(2)]
    last = slots // page - 1
    table = small.table.copy()
    for r in range(2):
        for i in range(pages_of(lengths[r], page)):
            table[r, i] = last
            for b, x in zip(kv, (small.kb, small.vb)):
                at = int(small.table[r, i]) * page
                hip.upload(b, x[0, at:at + page], last * page * heads * VECTOR)
            last -= 3 if i else slots // page // 2
            last %= slots // page
    tb, q = hip.from_host(table), rng.standard_normal((2, 4 * heads, D)).astype(np.float16)
    h = small.handle()
    h.kv = F.GhKv(kv[0], kv[1], F.KV_Q4, 1, slots, heads, D, D)
    h.table = tb
    qb, ob = hip.from_host(q), hip.alloc_buffer(q.nbytes)
    hip.attention_decode_paged(ob, qb, h, 4 * heads, 0, 0)
    check_attention4(small, 0, q, hip.download(ob, np.float16, q.size).reshape(q.shape))
    # and what the read-back finds there
    n = 130 * 2 * heads * D
    kb, vb = hip.alloc_buffer(2 * n), hip.alloc_buffer(2 * n)
    hip.kv_read_paged(kb, vb, h, 130, 0)
    got = hip.download(kb, np.float16, n).reshape(2, 130, heads, D)
    assert np.array_equal(got[0], small.k[0, small.cells(0, 130)])
    assert np.array_equal(got[1, 60:], small.k[0, small.cells(1, 70)])
    for b in (*kv, tb, qb, ob, kb, vb):
        hip.free_buffer(b)
    small.free()


def test_attention_peaked_and_flat_weights(hip, rng):
    """One key far above all others; 30000 keys of 2^-26 of the largest each, which together are 2^-11 of it."""
    n = 30000
    p = Paged4(hip, rng, [n, n], 64, 1)
    q = np.zeros((2, 1, D), np.float16)
    q[:, 0, 0] = 8
    k, v = np.zeros_like(p.k), np.where(np.isnan(p.v), 0, p.v).astype(np.float16)
    a, b = p.cells(0, n), p.cells(1, n)
    k[0, a[1234], 0, 0] = 60
    k[0, b, 0, 0] = -25.5  # 8 * 25.5 / sqrt(128) = 18.03 = 26.01 ln 2
    k[0, b[77], 0, 0] = 0
    v[0, b, 0, 1] = 1000
    v[0, b[77], 0] = 0
    p.kb, p.vb = pack(k), pack(v)
    p.upload()
    q, out = run_attention(hip, p, 1, rng, q=q)
    check_attention4(p, 0, q, out)
    assert 0.2 < out[1, 0, 1] < 0.7  # 30000 * 2^-26 * 1000
    p.free()


def test_attention_nan_stays_where_it_is_seen(hip, rng):
    """A NaN group in V and in K: NaN in its dims, and in its head, of its row alone. The pool is NaN elsewhere."""
    p = Paged4(hip, rng, [100, 100, 100], 16, 2)
    k, v = p.k.copy(), p.v.copy()
    v[0, p.cells(0, 100)[40], 1, 5] = np.inf
    k[0, p.cells(1, 100)[50], 0, 127] = np.nan
    p.kb, p.vb = pack(k), pack(v)
    p.upload()
    q, out = run_attention(hip, p, 8, rng)
    bad = np.isnan(out)
    want = np.zeros_like(bad)
    want[0, 4:, :32] = True
    want[1, :4] = True
    assert np.array_equal(bad, want)
    p.free()


def test_attention_largest_values(hip, rng):
    """Values at FP16's ends stay finite, scores beyond FP32's exponent of weights too."""
    p = Paged4(hip, rng, [40], 16, 1)
    v = np.where(np.isnan(p.v), 0, p.v).astype(np.float16)
    at = p.cells(0, 40)
    v[0, at, 0, :32] = np.where(rng.random((40, 32)) < 0.5, -65504, 65504)
    p.vb = pack(v)
    p.upload()
    assert np.isfinite(unpack(p.vb)[0, at]).all()
    q, out = run_attention(hip, p, 4, rng)
    check_attention4(p, 0, q, out)
    p.free()


@pytest.mark.parametrize("what", ["length", "page", "page_in_half", "max_len"])
@pytest.mark.parametrize("rows", [2, 80])
def test_attention_reports_what_does_not_fit(hip, rng, what, rows):
    """Only the row at fault is lost. 80 rows are laid out together."""
    p = Paged4(hip, rng, [100] + [600] * (rows - 1), 16, 8, width=40)
    if what == "length":
        p.lengths[0] = 16 * p.width + 1
    elif what == "page":
        p.table[0, 2] = p.slots // p.page
    elif what == "page_in_half":
        p.table[0, 1] = 0xFFFFFFFF
    p.upload()
    q = rng.standard_normal((rows, 16, D)).astype(np.float16)
    qb, ob = hip.from_host(q), hip.from_host(np.zeros_like(q))
    max_len = 0
    if what == "max_len":
        p.lengths[0], max_len = 601, 600
        p.upload()
    with pytest.raises(GhError) as e:
        hip.attention_decode_paged(ob, qb, p.handle(), 16, max_len, 0)
    assert e.value.code == -5
    out = hip.download(ob, np.float16, q.size).reshape(q.shape)
    p.lengths[0] = 0
    out[0] = 0
    check_attention4(p, 0, q, out)
    for b in (qb, ob):
        hip.free_buffer(b)
    p.free()


# ---- append and read-back ----

def vectors(rng, p, tokens):
    return [rng.standard_normal((p.rows, tokens, p.heads, D)).astype(np.float16) for _ in range(2)]


def read_back(hip, p, tokens, layer):
    n = p.rows * tokens * p.heads * D
    kb, vb = (hip.from_host(np.full(n, 7, np.float16)) for _ in range(2))
    hip.kv_read_paged(kb, vb, p.handle(), tokens, layer)
    got = [hip.download(b, np.float16, n).reshape(p.rows, tokens, p.heads, D) for b in (kb, vb)]
    for b in (kb, vb):
        hip.free_buffer(b)
    return got


@pytest.mark.parametrize("tokens", [1, 3, 40])
@pytest.mark.parametrize("page,heads,scored", [(16, 8, True), (32, 3, False), (256, 1, True)])
def test_write_and_read_back(hip, rng, tokens, page, heads, scored):
    """The definition's bytes in the rows' last positions, and nothing else changed; read back, what they stand for."""
    lengths = [tokens, 100, 0, max(1, tokens - 1), 257]
    p = Paged4(hip, rng, lengths, page, heads, layers=2, scored=scored)
    k, v = vectors(rng, p, tokens)
    k[1, 0, 0, :32] = 0.3125                       # no range
    k[1, 0, 0, 32:64] = 6e-8 * rng.integers(0, 30, 32)  # a step below FP16's least
    v[1, 0, 0, :64] = rng.integers(0, 2, 64) * 131008.0 - 65504
    v[1, 0, 0, 70], v[4, 0, 0, 100] = np.nan, np.inf
    kb, vb = hip.from_host(k), hip.from_host(v)
    hip.kv_write_paged(p.handle(), kb, vb, tokens, 1)
    score = None if p.score is None else p.score.copy()
    for r, n in enumerate(lengths):
        for t in range(tokens):
            at = n - tokens + t
            if at < 0:
                continue
            p.kb[1, p.cells(r, n)[at]], p.vb[1, p.cells(r, n)[at]] = pack(k[r, t]), pack(v[r, t])
            if scored:
                score[1, r, :, at] = 0
    assert np.array_equal(p.read("k"), p.kb) and np.array_equal(p.read("v"), p.vb)
    if scored:
        assert np.array_equal(p.read("score"), score)
    for got, x in zip(read_back(hip, p, tokens, 1), (k, v)):
        for r, n in enumerate(lengths):
            for t in range(tokens):
                want = unpack(pack(x[r, t])) if n - tokens + t >= 0 else np.float16(7)
                assert np.array_equal(got[r, t], np.broadcast_to(want, got[r, t].shape), equal_nan=True), (r, t)
    for b in (kb, vb):
        hip.free_buffer(b)
    p.free()


def test_read_back_of_fp16(hip, rng):
    p = Paged(hip, rng, [70, 0, 5], 16, 3, layers=2)
    k, v = read_back(hip, p, 60, 1)
    for r, n in enumerate([70, 0, 5]):
        have = min(n, 60)
        at = p.cells(r, n)[n - have:]
        assert np.array_equal(k[r, 60 - have:].view(np.uint16), p.k[1, at].view(np.uint16))
        assert np.array_equal(v[r, 60 - have:].view(np.uint16), p.v[1, at].view(np.uint16))
        assert (k[r, :60 - have] == 7).all()
    p.free()


def angles(yarn, pos):
    """The FP32 angles [positions][pairs] of the definition (gh_rope_yarn's), in 64 bits."""
    f = np.float32
    pair = np.arange(yarn.rope_dim // 2)

    def corr(beta):
        return yarn.rope_dim * np.log(yarn.original_context / (beta * 2 * np.pi)) / (2 * np.log(yarn.freq_base))

    lo = max(np.floor(corr(yarn.beta_fast)), 0)
    hi = min(np.ceil(corr(yarn.beta_slow)), yarn.rope_dim - 1)
    # the exponent is an FP32 number too: its rounding, times ln(freq_base) = 13.8, is more than the power's own
    freq = np.power(float(yarn.freq_base), (f(-2) * pair.astype(f) / f(yarn.rope_dim)).astype(np.float64)).astype(f)
    ramp = f(1) - np.clip((pair.astype(f) - f(lo)) / f(max(hi - lo, 0.001)), f(0), f(1))
    far = np.asarray(pos, f)[:, None] * freq
    return ((f(1) / f(yarn.factor) * far) * (f(1) - ramp) + far * ramp).astype(np.float64)


def normed(x, w, eps):
    """x [...][dim] in 64 bits over the root of its mean square, times w."""
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)


def turned(x, yarn, pos, query):
    """x [n][heads][dim] in 64 bits at n positions, and a bound of what FP32 does to it: the angle's frequency is off by
    an FP32 step or so, which the position multiplies, and the norm and the rotation by 32 half steps."""
    pos = np.asarray(pos)
    t = angles(yarn, pos)[:, None]
    y = x.copy()
    n = yarn.rope_dim
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    y[..., 0:n:2], y[..., 1:n:2] = a * np.cos(t) - b * np.sin(t), a * np.sin(t) + b * np.cos(t)
    scale = np.ones(len(pos))
    if query:
        scale = 1 + yarn.q_temperature_scale * np.log1p(pos // yarn.original_context)
    size = np.repeat(np.sqrt((x[..., 0::2] ** 2 + x[..., 1::2] ** 2)), 2, -1)
    slip = np.zeros(x.shape)
    slip[..., :n] = np.repeat(4 * HALF * np.abs(t), 2, -1)
    up = np.ones(x.shape)
    up[..., :n] = scale[:, None, None]  # gh_rope_yarn scales what it turns
    return y * up, size * (slip + 32 * HALF) * up


def check_fp16(got, want, bound):
    err = np.abs(got.astype(np.float64) - want)
    limit = bound + 2.0 ** -11 * (np.abs(want) + bound) + 2.0 ** -25
    assert np.all(err <= limit), float((err / limit).max())


def check_codes(b, want, bound):
    """Bytes against values known up to `bound`: minimum and step of each 32, then half a step for each value. The
    step's cut-off leaves less than half a step at the top code."""
    c, d, m = parts(b)
    w, e = want.reshape(c.shape), bound.reshape(c.shape).max(-1)
    low, high = w.min(-1), w.max(-1)
    assert np.all(np.abs(m - low) <= e + 2.0 ** -11 * np.abs(low) + 2.0 ** -25)
    step = (high - low + 2 * e) / 15 * (1 + 4 * HALF)
    least = (high - low - 2 * e) / 15 * (1 - 4 * HALF)
    assert np.all(d <= step) and np.all(d >= least * (1 - 2.0 ** -10) - 2.0 ** -24)
    err = np.abs(m[..., None] + d[..., None] * c - w)
    limit = (d / 2 + e + 2.0 ** -11 * np.abs(low) + 2.0 ** -20)[..., None]
    assert np.all(err <= limit), float((err / limit).max())


@pytest.mark.parametrize("bits,form", [(4, "rope"), (4, "norm"), (16, "norm")])
@pytest.mark.parametrize("tokens", [1, 7])
@pytest.mark.parametrize("heads,group,rope_dim", [(8, 4, 128), (1, 1, 64), (2, 7, 90)])
def test_rope_and_norm_write(hip, rng, bits, form, tokens, heads, group, rope_dim):
    lengths = [tokens, 300, 0, 77, max(1, tokens - 2)]
    p = (Paged4 if bits == 4 else Paged)(hip, rng, lengths, 32, heads, layers=2, scored=True)
    yarn = Yarn(rope_dim, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    k, v = vectors(rng, p, tokens)
    q = (3 * rng.standard_normal((p.rows, tokens, heads * group, D))).astype(np.float16)
    q[1, 0, 0], k[1, 0, 0] = 0, 0  # a head of zeros: eps alone under the root
    wq, wk = ((1 + 0.3 * rng.standard_normal(D)).astype(np.float16) for _ in range(2))
    pos = np.array([0, 290, 5, 40000, 16384], np.uint32)
    qb, kb, vb, pb, wqb, wkb = (hip.from_host(x) for x in (q, k, v, pos, wq, wk))
    ob = hip.from_host(np.full_like(q, 9))
    args = (kb, vb, heads * group) + ((wqb, wkb, 1e-5) if form == "norm" else ()) + (pb, tokens, 40010, yarn, 1)
    before = p.read("k")
    (hip.norm_rope_kv_write_paged if form == "norm" else hip.rope_kv_write_paged)(p.handle(), ob, qb, *args)
    out = hip.download(ob, np.float16, q.size).reshape(q.shape)
    kc, vc, score = p.read("k"), p.read("v"), p.read("score")
    written = np.zeros(kc.shape[:2], bool)
    for r, n in enumerate(lengths):
        for t in range(tokens):
            at = n - tokens + t
            if at < 0:
                assert (out[r, t] == 9).all()
                continue
            x, y = q[r, t].astype(np.float64), k[r, t].astype(np.float64)
            if form == "norm":
                x, y = normed(x, wq, 1e-5), normed(y, wk, 1e-5)
            check_fp16(out[r, t], *(z[0] for z in turned(x[None], yarn, [int(pos[r]) + t], True)))
            want, bound = (z[0] for z in turned(y[None], yarn, [int(pos[r]) + t], False))
            slot = p.cells(r, n)[at]
            written[1, slot] = True
            if bits == 4:
                check_codes(kc[1, slot], want, bound)
                assert np.array_equal(vc[1, slot], pack(v[r, t]))
            else:
                check_fp16(kc[1, slot], want, bound)
                assert np.array_equal(vc[1, slot].view(np.uint16), v[r, t].view(np.uint16))
            assert not score[1, r, :, at].any()
            p.score[1, r, :, at] = 0
    assert np.array_equal(kc[~written].view(np.uint8), before[~written].view(np.uint8))
    assert np.array_equal(score, p.score)
    hip.upload(ob, q)  # in place, the same bits
    (hip.norm_rope_kv_write_paged if form == "norm" else hip.rope_kv_write_paged)(p.handle(), ob, ob, *args)
    again = hip.download(ob, np.float16, q.size).reshape(q.shape)
    same = np.array([[n - tokens + t >= 0 for t in range(tokens)] for n in lengths])
    assert np.array_equal(again[same].view(np.uint16), out[same].view(np.uint16))
    for b in (qb, kb, vb, pb, wqb, wkb, ob):
        hip.free_buffer(b)
    p.free()


def test_rope_write_rounds_as_its_fp16_form(hip, rng):
    """The queries of a 4-bit append have the bits of the FP16 append's."""
    tokens, heads = 3, 2
    q = rng.standard_normal((2, tokens, 8, D)).astype(np.float16)
    pos = hip.from_host(np.array([5, 1000], np.uint32))
    outs = []
    for cls in (Paged, Paged4):
        p = cls(hip, np.random.default_rng(3), [10, 20], 16, heads)
        k, v = vectors(np.random.default_rng(4), p, tokens)
        qb, kb, vb = hip.from_host(q), hip.from_host(k), hip.from_host(v)
        hip.rope_kv_write_paged(p.handle(), qb, qb, kb, vb, 8, pos, tokens, 2000, YARN, 0)
        outs.append(hip.download(qb, np.uint16, q.size))
        for b in (qb, kb, vb):
            hip.free_buffer(b)
        p.free()
    hip.free_buffer(pos)
    assert np.array_equal(*outs)


def test_append_reports_what_does_not_fit(hip, rng):
    p = Paged4(hip, rng, [40, 40, 40], 16, 2, extra_pages=0)
    kb0 = p.kb.copy()
    k, v = vectors(rng, p, 1)
    q = np.zeros((3, 1, 2, D), np.float16)
    kb, vb, qb, w = hip.from_host(k), hip.from_host(v), hip.from_host(q), hip.from_host(np.ones(D, np.float16))
    pos = hip.from_host(np.array([39, 101, 0xFFFFFFFF], np.uint32))
    p.table[1, 2] = 1000
    p.upload()
    with pytest.raises(GhError) as e:
        hip.norm_rope_kv_write_paged(p.handle(), qb, qb, kb, vb, 2, w, w, 1e-5, pos, 1, 100, YARN, 0)
    assert e.value.code == -5
    with pytest.raises(GhError):
        hip.kv_write_paged(p.handle(), kb, vb, 1, 0)
    with pytest.raises(GhError):
        hip.kv_read_paged(kb, vb, p.handle(), 1, 0)
    got = p.read("k")
    slots = [p.cells(r, 40)[39] for r in (0, 2)]
    others = np.setdiff1d(np.arange(p.slots), slots)
    assert np.array_equal(got[0, others], kb0[0, others])
    for b in (kb, vb, qb, w, pos):
        hip.free_buffer(b)
    p.free()


# ---- eviction ----

@pytest.mark.parametrize("kept_list", [True, False])
@pytest.mark.parametrize("page,heads,budget,recent", [(16, 3, 50, 10), (64, 8, 129, 129), (32, 1, 1, 0)])
def test_evict(hip, rng, page, heads, budget, recent, kept_list):
    lengths = [200, budget, 131, 0]
    p = Paged4(hip, rng, lengths, page, heads, layers=2, scored=True)
    p.score[:] = rng.integers(0, 20, p.score.shape)
    p.upload()
    d = Paged4(hip, rng, [budget if n > budget else 0 for n in lengths], page, heads, layers=2, scored=True)
    d.lengths[:] = 7
    d.upload()
    kept = hip.alloc_buffer(2 * 4 * heads * budget * 4) if kept_list else None
    hip.kv_evict_paged(d.handle(), p.handle(), kept, budget, recent)
    kc, vc, score, new = d.read("k"), d.read("v"), d.read("score"), d.read("lengths")
    got = hip.download(kept, np.uint32, 2 * 4 * heads * budget).reshape(2, 4, heads, budget) if kept_list else None
    kb, vb = d.kb.copy(), d.vb.copy()
    for r, n in enumerate(lengths):
        assert new[r] == (budget if n > budget else 7)
        if n <= budget:
            continue
        for layer in range(2):
            for h in range(heads):
                best = keep(p.score[layer, r, h, :n], budget, recent)
                if kept_list:
                    assert np.array_equal(got[layer, r, h], best)
                to, at = d.cells(r, budget), p.cells(r, n)[best]
                kb[layer, to, h], vb[layer, to, h] = p.kb[layer, at, h], p.vb[layer, at, h]
                assert np.array_equal(score[layer, r, h, :budget], p.score[layer, r, h, best])
    assert np.array_equal(kc, kb) and np.array_equal(vc, vb)
    if kept_list:
        hip.free_buffer(kept)
    p.free()
    d.free()


# ---- norms and RoPE of a prefill's rows ----

@pytest.mark.parametrize("heads,kv_heads,dim,rope_dim", [(32, 8, 128, 128), (3, 1, 64, 64), (2, 2, 256, 128), (1, 0, 8, 8), (0, 5, 16, 10),
                                                          (7, 1, 96, 96), (4, 2, 512, 512), (2, 1, 40, 24)])
@pytest.mark.parametrize("rows,base", [(1, 0), (5, 16380), (131, 33000)])
def test_norm_rope_batched(hip, rng, heads, kv_heads, dim, rope_dim, rows, base):
    yarn = Yarn(rope_dim, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    q = (3 * rng.standard_normal((rows, heads, dim))).astype(np.float16)
    k = (0.01 * rng.standard_normal((rows, kv_heads, dim))).astype(np.float16)
    wq, wk = ((1 + 0.3 * rng.standard_normal(dim)).astype(np.float16) for _ in range(2))
    for x in (q, k):
        if x.size:
            x[0, 0] = 0
            x[rows - 1, -1] = 60000  # squares beyond FP16
    guard = np.full(64, 5, np.float16)
    qb, kb = (hip.from_host(np.concatenate([x.ravel(), guard])) for x in (q, k))
    wqb, wkb = hip.from_host(wq), hip.from_host(wk)
    hip.norm_rope_batched(qb, kb, heads, kv_heads, dim, base, rows, wqb, wkb, 1e-5, yarn)
    for b, x, w, query in ((qb, q, wq, True), (kb, k, wk, False)):
        got = hip.download(b, np.float16, x.size + 64)
        assert (got[x.size:] == 5).all()
        if x.size:
            check_fp16(got[:x.size].reshape(x.shape), *turned(normed(x, w, 1e-5), yarn, np.arange(base, base + rows), query))
    for b in (qb, kb, wqb, wkb):
        hip.free_buffer(b)


def test_norm_rope_keeps_what_is_not_finite_in_its_head(hip, rng):
    q = rng.standard_normal((2, 4, D)).astype(np.float16)
    k = rng.standard_normal((2, 1, D)).astype(np.float16)
    q[0, 1, 3], q[1, 2, 77] = np.nan, np.inf
    w = hip.from_host(np.ones(D, np.float16))
    qb, kb = hip.from_host(q), hip.from_host(k)
    hip.norm_rope_batched(qb, kb, 4, 1, D, 0, 2, w, w, 1e-5, YARN)
    got = hip.download(qb, np.float16, q.size).reshape(q.shape)
    bad = ~np.isfinite(got).all(-1)
    assert bad[0, 1] and bad[1, 2] and bad.sum() == 2
    for b in (qb, kb, w):
        hip.free_buffer(b)
