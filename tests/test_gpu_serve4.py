"""The operators of a batch over 4-bit caches together, as a server runs them, and calls at the ends of what they allow."""
import threading

import numpy as np
import pytest

from graph_horizon_amd import GhError, GhKvPaged, HipBackend, HipModel, Yarn, synth
from graph_horizon_amd import _ffi as F
from paged import D, keep
from paged4 import Paged4, check_attention4, pack, unpack
from sampled import sample
from test_gpu_paged4 import check_codes, check_fp16, normed, run_attention, turned
from test_gpu_sample import PARAMS, SETTINGS, check, run

pytestmark = pytest.mark.gpu
YARN = Yarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)


def test_serving_run(hip, rng):
    """Prompts: norms with RoPE, prefill over a contiguous cache, append. Then steps of one encoder each: append with norms, attention,
    logits and the next tokens' draw, from which the next step's vectors follow; an eviction in between and a read-back at the end."""
    heads, group, page, vocab, stride, budget, recent, eps = 2, 4, 16, 2999, 3000, 40, 8, 1e-5
    q_heads, width = heads * group, 8
    prompts = [50, 0, 17, 90]
    rows = len(prompts)
    p = Paged4(hip, rng, [width * page] * rows, page, heads, scored=True, score=0.0, extra_pages=40)
    before = p.kb.copy(), p.vb.copy()
    wq, wk = ((1 + 0.3 * rng.standard_normal(D)).astype(np.float16) for _ in range(2))
    wqb, wkb = hip.from_host(wq), hip.from_host(wk)
    p.lengths[:] = 0
    for r, n in enumerate(prompts):
        if not n:
            continue
        q, k, v = (rng.standard_normal((n, h, D)).astype(np.float16) for h in (q_heads, heads, heads))
        contiguous = np.zeros((2, n, heads, D), np.float16)
        qb, ob, cb = hip.from_host(q), hip.alloc_buffer(q.nbytes), hip.from_host(contiguous)
        half = contiguous[0].nbytes
        cache = F.GhKv(hip.view(cb, 0, half), hip.view(cb, half, half), F.KV_F16, 1, n, heads, D, D)
        # the other rows' share of the append lies before their first position
        wide = np.zeros((2, rows, n, heads, D), np.float16)
        wide[0, r], wide[1, r] = k, v
        kb, vb = hip.from_host(wide[0]), hip.from_host(wide[1])
        row = k.nbytes
        kr, vr = hip.view(kb, r * row, row), hip.view(vb, r * row, row)
        p.lengths[:] = np.where(np.arange(rows) == r, n, 0)
        hip.upload(p.bufs["lengths"], p.lengths)
        hip.begin()
        hip.norm_rope_batched(qb, kr, q_heads, heads, D, 0, n, wqb, wkb, eps, YARN)
        hip.kv_write(cache, kr, vr, 0, 0, n * heads)
        hip.attention_prefill(ob, qb, cache, q_heads, 0, n, 0)
        hip.kv_write_paged(p.handle(), kb, vb, n, 0)
        hip.submit()
        at = p.cells(r, n)
        keys = hip.download(kb, np.float16, wide[0].size).reshape(wide[0].shape)[r]
        check_fp16(keys, *turned(normed(k, wk, eps), YARN, np.arange(n), False))
        assert np.array_equal(p.read("k")[0, at], pack(keys))
        assert np.array_equal(p.read("v")[0, at], pack(v))
        for b in (qb, ob, cb, kb, vb):
            hip.free_buffer(b)
    p.lengths = np.array(prompts, np.uint32)
    now = p.read("k")
    held = np.zeros(p.slots, bool)
    for r, n in enumerate(prompts):
        held[p.cells(r, n)] = True
    assert np.array_equal(now[0, ~held], before[0][0, ~held])

    weight = hip.load_weight(F.FMT_Q4_K, synth.quant_blocks(rng, F.FMT_Q4_K, vocab, q_heads * D, 0.02), q_heads * D, vocab)
    table = rng.standard_normal((vocab, q_heads + 2 * heads, D)).astype(np.float16)  # a token's vectors
    params = np.array([(0.8, 0.95, 40, 0.0), (0.0, 1.0, 0, 0.0), (1.2, 0.9, 0, 0.02), (1.0, 1.0, 0, 0.0)], PARAMS)
    params_b, uniform_b = hip.from_host(params), hip.alloc_buffer(4 * rows)
    logits_b, tokens_b, probs_b = hip.alloc_buffer(rows * stride * 4), hip.alloc_buffer(4 * rows), hip.alloc_buffer(4 * rows)
    pos_b, ob = hip.alloc_buffer(4 * rows), hip.alloc_buffer(rows * q_heads * 256)
    position, tokens = np.array(prompts, np.uint32), np.array([5, 6, 7, 8])
    for step in range(14):
        live = np.array([r != 1 or step >= 4 for r in range(rows)])  # a new sequence takes the free row
        p.lengths[live] += 1
        hip.upload(p.bufs["lengths"], p.lengths)
        hip.upload(pos_b, position)
        u = rng.random(rows).astype(np.float32)
        hip.upload(uniform_b, u)
        x = table[tokens]
        q, k, v = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
        qb, kb, vb = hip.from_host(q), hip.from_host(k), hip.from_host(v)
        score = p.read("score")
        hip.begin()
        hip.norm_rope_kv_write_paged(p.handle(), qb, qb, kb, vb, q_heads, wqb, wkb, eps, pos_b, 1, 400, YARN, 0)
        hip.attention_decode_paged(ob, qb, p.handle(), q_heads, 0, 0)
        for r in range(rows):
            hip.logits(hip.view(logits_b, r * stride * 4, vocab * 4), hip.view(ob, r * q_heads * 256, q_heads * 256), weight, q_heads * D, vocab)
        hip.sample_rows(tokens_b, probs_b, logits_b, rows, vocab, stride, params_b, uniform_b)
        hip.submit()
        got_q, out = (hip.download(b, np.float16, q.size).reshape(q.shape) for b in (qb, ob))
        p.kb, p.vb = p.read("k"), p.read("v")
        for r in np.nonzero(live)[0]:
            slot = p.cells(r, int(p.lengths[r]))[-1]
            check_fp16(got_q[r], *(z[0] for z in turned(normed(q[r], wq, eps)[None], YARN, [int(position[r])], True)))
            check_codes(p.kb[0, slot], *(z[0] for z in turned(normed(k[r], wk, eps)[None], YARN, [int(position[r])], False)))
            assert np.array_equal(p.vb[0, slot], pack(v[r]))
            score[0, r, :, p.lengths[r] - 1] = 0
        check_attention4(p, 0, got_q, out, score, p.read("score"))
        logits = hip.download(logits_b, np.float32, rows * stride).reshape(rows, stride)[:, :vocab]
        drawn, probs = hip.download(tokens_b, np.uint32, rows), hip.download(probs_b, np.float32, rows)
        for r in range(rows):
            want, prob, near = sample(logits[r], *params[r], u[r])
            assert drawn[r] == want or near < 1e-11
            assert drawn[r] != want or abs(probs[r] - prob) <= 2.0 ** -24 * prob + 2.0 ** -36
        tokens = np.where(live, drawn, tokens)
        position[live] += 1
        for b in (qb, kb, vb):
            hip.free_buffer(b)
        if step == 6:  # long rows go on in new pages
            old, score = p.lengths.copy(), p.read("score")
            fresh = p.table.copy()
            spare = np.setdiff1d(np.arange(p.slots // page), p.table.ravel())
            for i, r in enumerate(np.nonzero(old > budget)[0]):
                fresh[r] = spare[i * width:(i + 1) * width]
            was = p.table
            src, new_b = p.handle(), hip.from_host(fresh)
            dst = p.handle()
            dst.table = new_b
            hip.kv_evict_paged(dst, src, None, budget, recent)
            kb1, vb1, score1 = p.read("k"), p.read("v"), p.read("score")
            for r in range(rows):
                if old[r] <= budget:
                    continue
                from_cells = p.cells(r, int(old[r]))
                p.table = fresh
                to_cells = p.cells(r, budget)
                p.table = was
                for h in range(heads):
                    best = keep(score[0, r, h, :old[r]], budget, recent)
                    assert np.array_equal(kb1[0, to_cells, h], p.kb[0, from_cells[best], h])
                    assert np.array_equal(vb1[0, to_cells, h], p.vb[0, from_cells[best], h])
                    assert np.array_equal(score1[0, r, h, :budget], score[0, r, h, best])
            p.lengths = np.minimum(old, budget)
            assert np.array_equal(p.read("lengths"), p.lengths)
            p.table = fresh
            hip.upload(p.bufs["table"], fresh)
            hip.free_buffer(new_b)
    most = int(p.lengths.max())
    kb, vb = (hip.from_host(np.full((rows, most, heads, D), 3, np.float16)) for _ in range(2))
    hip.kv_read_paged(kb, vb, p.handle(), most, 0)
    for b, pool in ((kb, p.kb), (vb, p.vb)):
        got = hip.download(b, np.float16, rows * most * heads * D).reshape(rows, most, heads, D)
        for r, n in enumerate(p.lengths):
            assert (got[r, :most - n] == 3).all()
            assert np.array_equal(got[r, most - n:], unpack(pool[0, p.cells(r, int(n))]))
    for b in (kb, vb, wqb, wkb, weight, params_b, uniform_b, logits_b, tokens_b, probs_b, pos_b, ob):
        hip.free_buffer(b)
    p.free()


def test_two_backends_at_once(rng):
    """Two backends (a stream and scratch each) in two threads, over one pool and the same logits."""
    with HipBackend(0) as a, HipBackend(0) as b:
        p = Paged4(a, rng, [5000, 0, 77, 3000], 16, 4, width=700)
        q = [rng.standard_normal((4, 16, D)).astype(np.float16) for _ in range(2)]
        logits = (3 * rng.standard_normal((4, 50001))).astype(np.float32)
        params = np.array([(0.9, 0.9, 0, 0.0), (1.0, 1.0, 300, 0.0), (1.5, 0.99, 0, 0.01), (0.0, 1.0, 0, 0.0)], PARAMS)
        u = rng.random((2, 4)).astype(np.float32)
        got, failed = [[], []], []

        def work(i, hip):
            try:
                qb, ob, lb, pb, ub = hip.from_host(q[i]), hip.alloc_buffer(q[i].nbytes), hip.from_host(logits), hip.from_host(params), hip.from_host(u[i])
                tb = hip.alloc_buffer(16)
                for _ in range(20):
                    hip.begin()
                    hip.attention_decode_paged(ob, qb, p.handle(), 16, 0, 0)
                    hip.sample_rows(tb, None, lb, 4, 50001, 50001, pb, ub)
                    hip.submit()
                    got[i].append((hip.download(ob, np.float16, q[i].size).reshape(q[i].shape), hip.download(tb, np.uint32, 4)))
                for x in (qb, ob, lb, pb, ub, tb):
                    hip.free_buffer(x)
            except Exception as e:  # noqa: BLE001
                failed.append(e)

        threads = [threading.Thread(target=work, args=(i, hip)) for i, hip in enumerate((a, b))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not failed
        for i in range(2):
            out, tokens = got[i][0]
            check_attention4(p, 0, q[i], out)
            for r in range(4):
                assert tokens[r] == sample(logits[r], *params[r], u[i, r])[0]
            assert len(got[i]) == 20
            for x, t in got[i]:
                assert np.array_equal(x.view(np.uint16), out.view(np.uint16)) and np.array_equal(t, tokens)
        p.free()


def test_recorded_decode_graphs_survive_the_scratch(rng):
    """Attention over 4-bit caches and sampling that move the backend's workspace between runs of a model's replayed decode."""
    shape = synth.SHAPES["tiny"]
    with HipBackend(0) as hip:
        m = HipModel(hip, synth.model_config(shape, 64, 16))
        for layer, tid, fmt, data in synth.model_tensors(shape, 1):
            m.load_tensor(layer, tid, fmt, data)
        m.prefill(np.arange(8), 0)
        first = m.decode_greedy(3, 8, 12)
        before = hip.scratch_info()[0]
        p = Paged4(hip, rng, [9000] * 6, 64, 2, scored=True)
        old = p.read("score")
        q, out = run_attention(hip, p, 32, rng)
        check_attention4(p, 0, q, out, old, p.read("score"))
        between = hip.scratch_info()[0]
        assert between > before
        assert np.array_equal(m.decode_greedy(3, 8, 12), first)
        logits = (3 * rng.standard_normal((400, 500))).astype(np.float32)
        check(hip, logits, [SETTINGS[3]] * 400, rng.random(400).astype(np.float32))
        assert hip.scratch_info()[0] > between
        assert np.array_equal(m.decode_greedy(3, 8, 12), first)
        check(hip, logits, [SETTINGS[5]] * 400, rng.random(400).astype(np.float32))
        p.free()
        m.close()


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("lengths,limit", [([3000, 100, 2000, 1, 700], 12 << 20), ([700] * 70, 8 << 20), ([700] * 70, 14 << 20)])
def test_attention_with_scratch_for_some_rows(rng, scored, lengths, limit):
    with HipBackend(0) as hip:
        hip.set_scratch_limit(limit)
        p = Paged4(hip, rng, lengths, 16, 8, scored=scored, width=200)
        for _ in range(2):
            before = p.read("score") if scored else None
            if limit == 8 << 20:  # the chunks' partials alone are 385 of 33 KB
                with pytest.raises(GhError) as e:
                    run_attention(hip, p, 64, rng)
                assert e.value.code == -4
                continue
            q, out = run_attention(hip, p, 64, rng)
            check_attention4(p, 0, q, out, before, p.read("score") if scored else None)
        p.free()


def test_what_lies_behind_the_last_row_stays(hip, rng):
    """Buffers with room for one more row: no operator writes there."""
    heads, group = 3, 5
    p = Paged4(hip, rng, [30, 0, 65], 16, heads, scored=True)
    q = rng.standard_normal((4, heads * group, D)).astype(np.float16)
    k = rng.standard_normal((3, heads, D)).astype(np.float16)
    qb, kb, pb, w = hip.from_host(q), hip.from_host(k), hip.from_host(np.array([3, 4, 5], np.uint32)), hip.from_host(np.ones(D, np.float16))
    mark = np.full((4, heads * group, D), 7, np.float16)
    ob, rb, kr, vr = (hip.from_host(mark) for _ in range(4))
    hip.norm_rope_kv_write_paged(p.handle(), rb, qb, kb, kb, heads * group, w, w, 1e-6, pb, 1, 5, YARN, 0)
    hip.attention_decode_paged(ob, rb, p.handle(), heads * group, 0, 0)
    hip.kv_read_paged(kr, vr, p.handle(), 1, 0)
    for b, n in ((ob, heads * group * D), (rb, heads * group * D), (kr, heads * D), (vr, heads * D)):
        assert np.all(hip.download(b, np.float16, mark.size)[3 * n:] == 7)
    for b in (qb, kb, pb, w, ob, rb, kr, vr):
        hip.free_buffer(b)
    p.free()


@pytest.mark.parametrize("bad", ["length", "page"])
@pytest.mark.parametrize("tokens", [1, 5])
def test_bad_rows_leave_everything_else_alone(hip, rng, bad, tokens):
    """An append and a read-back of three rows, the second with a length or a page that does not fit."""
    p = Paged4(hip, rng, [100, 96, 300], 16, 2, layers=2, scored=True)
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
        p.kb[1, at[r]], p.vb[1, at[r]] = pack(k[r]), pack(v[r])
        p.score[1, r, :, int(good[r]) - tokens:int(good[r])] = 0
    assert np.array_equal(p.read("k"), p.kb) and np.array_equal(p.read("v"), p.vb) and np.array_equal(p.read("score"), p.score)
    mark = np.full(k.shape, 7, np.float16)
    hip.upload(kb, mark)
    hip.upload(vb, mark)
    with pytest.raises(GhError) as e:
        hip.kv_read_paged(kb, vb, p.handle(), tokens, 1)
    assert e.value.code == -5
    for b, pool in ((kb, p.kb), (vb, p.vb)):
        got = hip.download(b, np.float16, k.size).reshape(k.shape)
        for r in (0, 2):
            assert np.array_equal(got[r], unpack(pool[1, at[r]]))
        assert (got[1] == 7).all()
    hip.free_buffer(kb)
    hip.free_buffer(vb)
    p.free()


@pytest.mark.parametrize("bad", ["length", "page", "dst_page"])
def test_eviction_within_one_pool_and_of_bad_rows(hip, rng, bad):
    """dst is src's pool with other pages, its lengths and scores src's own. Row 1 does not fit: rows 0 and 2 move as ever, row 3 is
    short and stays, and no page of another row is written."""
    heads, budget, recent = 3, 50, 10
    p = Paged4(hip, rng, [100, 90, 300, 40], 16, heads, 2, scored=True, extra_pages=30)
    good = p.lengths.copy()
    cells = [p.cells(r, int(good[r])) for r in range(4)]
    spare = np.setdiff1d(np.arange(p.slots // 16), p.table[p.table < p.slots // 16])
    to = np.full_like(p.table, 0xFFFFFFFF)
    to[:3, :4] = spare[:12].reshape(3, 4)
    own = to[1, :4].copy()
    if bad == "length":
        p.lengths[1] = 16 * p.width + 1
    elif bad == "page":
        p.table[1, :6] = p.slots // 16
    else:
        to[1, :4] = p.slots // 16
    p.upload()
    new = hip.from_host(to)
    dst = p.handle()
    dst.table = new
    with pytest.raises(GhError) as e:
        hip.kv_evict_paged(dst, p.handle(), None, budget, recent)
    assert e.value.code == -5
    kb, vb, score = p.kb.copy(), p.vb.copy(), p.score.copy()
    j = np.arange(budget)
    for r in (0, 2):
        there = to[r, j // 16].astype(np.int64) * 16 + j % 16
        for layer in range(2):
            for h in range(heads):
                best = keep(p.score[layer, r, h, :good[r]], budget, recent)
                kb[layer, there, h], vb[layer, there, h] = p.kb[layer, cells[r][best], h], p.vb[layer, cells[r][best], h]
                score[layer, r, h, :budget] = p.score[layer, r, h, best]
    same = np.ones(p.slots, bool)
    for page in own:  # row 1's results are its own
        same[int(page) * 16:int(page) * 16 + 16] = False
    assert np.array_equal(p.read("k")[:, same], kb[:, same]) and np.array_equal(p.read("v")[:, same], vb[:, same])
    rows = [0, 2, 3]
    assert np.array_equal(p.read("score")[:, rows], score[:, rows])
    assert list(p.read("lengths")[rows]) == [budget, budget, 40]
    hip.free_buffer(new)
    p.free()


def test_norm_write_beyond_fp16(hip, rng):
    """Normed keys past FP16's range: an infinity in an FP16 pool, NaN for their 32 in 4 bits."""
    w = np.ones(D, np.float16)
    w[40] = 60000
    k = rng.standard_normal((1, 1, D)).astype(np.float16)
    k[0, 0, 40] = 4  # a norm of 3 or so
    p = Paged4(hip, rng, [1], 16, 1)
    wb, kb, pb, qb = hip.from_host(w), hip.from_host(k), hip.from_host(np.zeros(1, np.uint32)), hip.from_host(np.zeros((1, 1, D), np.float16))
    hip.norm_rope_kv_write_paged(p.handle(), qb, qb, kb, kb, 1, wb, wb, 1e-6, pb, 1, 0, YARN, 0)
    got = unpack(p.read("k")[0, p.cells(0, 1)[0], 0])
    assert np.isnan(got[32:64]).all() and np.isfinite(np.delete(got, np.s_[32:64])).all()
    for b in (wb, kb, pb, qb):
        hip.free_buffer(b)
    p.free()


@pytest.mark.parametrize("lengths,width", [([40, 300, 77], None), ([5000, 40, 3000, 17], 1200)])  # spans, chunks
def test_a_query_that_is_not_finite_is_its_own(hip, rng, lengths, width):
    heads, group = 4, 3
    p = Paged4(hip, rng, lengths, 16, heads, width=width)
    q = rng.standard_normal((len(lengths), heads * group, D)).astype(np.float16)
    plain = run_attention(hip, p, heads * group, rng, q=q)[1]
    q[0, 1, 5], q[1, 7, 100], q[2, 11, 64] = np.nan, np.inf, -np.inf
    out = run_attention(hip, p, heads * group, rng, q=q)[1]
    bad = np.zeros(q.shape[:2], bool)
    bad[0, 1] = bad[1, 7] = bad[2, 11] = True
    assert np.array_equal(np.isnan(out).any(-1), bad)
    assert np.array_equal(out[~bad].view(np.uint16), plain[~bad].view(np.uint16))
    p.free()


def test_append_and_read_back_past_4_gib(hip, rng):
    """Pages whose byte offsets pass 32 bits (a pool of 4.5 GiB each for K and V); evicted from one to another of these."""
    page, heads = 64, 8
    slots = (9 << 29) // (80 * heads) // page * page
    kc, vc = (hip.alloc_buffer(slots * heads * 80) for _ in range(2))
    last = slots // page - 1
    table, other = hip.from_host(np.array([[last, last - 1]], np.uint32)), hip.from_host(np.array([[last - 7, last - 5]], np.uint32))
    lengths, score = hip.from_host(np.array([100], np.uint32)), hip.from_host(rng.random((1, 1, heads, 2 * page)).astype(np.float32))
    kv = F.GhKv(kc, vc, F.KV_Q4, 1, slots, heads, D, D)
    k, v = (rng.standard_normal((1, 100, heads, D)).astype(np.float16) for _ in range(2))
    kb, vb = hip.from_host(k), hip.from_host(v)
    rows = [GhKvPaged(kv, t, lengths, score, page, 2, 1) for t in (table, other)]
    hip.kv_write_paged(rows[0], kb, vb, 100, 0)
    weight = rng.random((1, 1, heads, 2 * page)).astype(np.float32)
    hip.upload(score, weight)
    hip.kv_read_paged(kb, vb, rows[0], 100, 0)
    for b, x in ((kb, k), (vb, v)):
        assert np.array_equal(hip.download(b, np.float16, x.size).reshape(x.shape), unpack(pack(x)))
    hip.kv_evict_paged(rows[1], rows[0], None, 70, 20)
    hip.kv_read_paged(kb, vb, rows[1], 70, 0)
    for b, x in ((kb, k), (vb, v)):
        got = hip.download(b, np.float16, 70 * heads * D).reshape(70, heads, D)
        for h in range(heads):
            assert np.array_equal(got[:, h], unpack(pack(x[0, keep(weight[0, 0, h, :100], 70, 20), h])))
    for b in (kc, vc, table, other, lengths, score, kb, vb):
        hip.free_buffer(b)


# ---- sampling ----

@pytest.mark.parametrize("temperature", [1e13, 1e20, 3e38, float("inf")])
def test_min_p_at_high_temperatures(hip, rng, temperature):
    """Weights that round to 1 far from the largest logit pass a min_p of 1."""
    for vocab in (50, 20000):
        logits = (3 * rng.standard_normal((4, vocab))).astype(np.float32)
        logits[2] *= 1e5
        params = [(temperature, 1.0, 0, 1.0), (temperature, 0.9, 0, 1.0), (temperature, 1.0, 30, 1.0), (temperature, 1.0, 0, 0.5)]
        for u in (0.1, 0.6, 0.97):
            check(hip, logits, params, [u] * 4)


@pytest.mark.parametrize("vocab", [700, 5003, 40001])
def test_any_settings(hip, rng, vocab):
    """Rows of all spreads, with ties and masked tokens, each with settings of its own."""
    rows = 120
    logits = (10 ** rng.uniform(-3, 2, (rows, 1)) * rng.standard_normal((rows, vocab)) + rng.uniform(-50, 50, (rows, 1))).astype(np.float32)
    logits[::5] = np.round(logits[::5])
    logits[1::7, rng.integers(0, vocab, vocab // 2)] = -np.inf
    params = [(float(10 ** rng.uniform(-2, 1.5)), float(rng.choice([1.0, rng.random(), 0.999, 1e-4])),
               int(rng.choice([0, rng.integers(1, vocab + 5), rng.integers(1, 60)])), float(rng.choice([0.0, rng.random(), 1e-5])))
              for _ in range(rows)]
    check(hip, logits, params, rng.random(rows).astype(np.float32), stride=vocab + 3)


def test_largest_vocabulary(hip, rng):
    vocab = 1 << 24
    logits = (2 * rng.standard_normal((2, vocab))).astype(np.float32)
    check(hip, logits, [(0.9, 0.9, 0, 0.0), (1.0, 1.0, 100000, 1e-3)], rng.random(2).astype(np.float32))


def test_logits_past_4_gib(hip, rng):
    """Rows whose byte offsets pass 32 bits."""
    rows, stride, vocab = 70, 1 << 24, 5001
    assert rows * stride * 4 > 1 << 32
    lb = hip.alloc_buffer(((rows - 1) * stride + vocab) * 4)
    logits = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    for r in range(rows):
        hip.upload(hip.view(lb, r * stride * 4, vocab * 4), logits[r])
    params, u = np.array([SETTINGS[3 + r % 12] for r in range(rows)], PARAMS), rng.random(rows).astype(np.float32)
    pb, ub, tb = hip.from_host(params), hip.from_host(u), hip.alloc_buffer(4 * rows)
    hip.sample_rows(tb, None, lb, rows, vocab, stride, pb, ub)
    got = hip.download(tb, np.uint32, rows)
    for r in range(rows):
        want, _, near = sample(logits[r], *params[r], u[r])
        assert got[r] == want or near < 1e-11
    for b in (lb, pb, ub, tb):
        hip.free_buffer(b)


def test_rows_at_any_address(hip, rng):
    """Logits, tokens, probs and numbers at odd multiples of 4 bytes; the same tokens as at 16."""
    rows, vocab = 5, 4097
    logits = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    params, u = [SETTINGS[3 + r] for r in range(rows)], rng.random(rows).astype(np.float32)
    want, shares = run(hip, logits, params, u, stride=4100)
    pb = hip.from_host(np.array(params, PARAMS))
    for off in (4, 8, 12):
        big = hip.alloc_buffer(16 + logits.nbytes)
        ub, tb, qb = (hip.alloc_buffer(16 + 4 * rows) for _ in range(3))
        lv, uv, tv, qv = (F.GhBuf(b.addr + off, n) for b, n in ((big, logits.nbytes), (ub, 4 * rows), (tb, 4 * rows), (qb, 4 * rows)))
        hip.upload(big, logits, off)
        hip.upload(ub, u, off)
        hip.sample_rows(tv, qv, lv, rows, vocab, vocab, pb, uv)
        assert np.array_equal(hip.download(tb, np.uint32, rows, off), want)
        assert np.array_equal(hip.download(qb, np.float32, rows, off), shares)
        for b in (big, ub, tb, qb):
            hip.free_buffer(b)
    hip.free_buffer(pb)
