"""gh_sample_rows against its definition in 64 bits (tests/sampled.py) and the host's gh_sample."""
import ctypes as C

import numpy as np
import pytest

from graph_horizon_amd import GhSampling
from graph_horizon_amd import _ffi as F
from sampled import sample

pytestmark = pytest.mark.gpu
PARAMS = np.dtype([("temperature", "<f4"), ("top_p", "<f4"), ("top_k", "<u4"), ("min_p", "<f4")])


def run(hip, logits, params, u, stride=None, probs=True):
    rows, vocab = logits.shape
    stride = stride or vocab
    wide = np.full((rows, stride), 1e30, np.float32)  # what lies behind a row's tokens does not count
    wide[:, :vocab] = logits
    lb, pb, ub = hip.from_host(wide), hip.from_host(np.array(params, PARAMS)), hip.from_host(np.asarray(u, np.float32))
    tb, qb = hip.from_host(np.full(rows + 1, 77, np.uint32)), hip.from_host(np.full(rows + 1, 77, np.float32))
    hip.sample_rows(tb, qb if probs else None, lb, rows, vocab, stride, pb, ub)
    tokens, got = hip.download(tb, np.uint32, rows + 1), hip.download(qb, np.float32, rows + 1)
    assert tokens[rows] == 77 and got[rows] == 77
    for b in (lb, pb, ub, tb, qb):
        hip.free_buffer(b)
    return tokens[:rows], got[:rows]


def check(hip, logits, params, u, **kw):
    tokens, probs = run(hip, logits, params, u, **kw)
    for r in range(len(logits)):
        t, p, k, m = params[r]
        want, prob, near = sample(logits[r], t, p, k, m, u[r])
        if near > 1e-11:  # else rounding in 64 bits may decide
            assert tokens[r] == want, (r, params[r], u[r], near)
        # weights are held to 2^-45 of the largest (2^-38 at 2^24 tokens), the share to FP32
        if tokens[r] == want:
            assert abs(probs[r] - prob) <= 2.0 ** -24 * prob + 2.0 ** -36, (r, params[r])
    return tokens


SETTINGS = [(0.0, 1.0, 0, 0.0), (-1.0, 0.5, 3, 0.1), (1.0, 1.0, 0, 0.0), (0.8, 0.9, 50, 0.0), (1.0, 1.0, 1, 0.0), (0.7, 0.95, 0, 0.0),
            (1.0, 1.0, 0, 0.05), (1.3, 0.99, 1000, 0.01), (0.05, 0.9, 40, 0.0), (5.0, 1.0, 7, 0.0), (1.0, 0.0, 0, 0.0),
            (1.0, 1e-30, 5, 0.0), (1.0, 1.0, 0, 1.0), (1.0, 1.0, 0, 2.0), (100.0, 0.5, 0, 0.0), (1e-30, 0.9, 0, 0.1), (float("nan"), 0.9, 0, 0.0),
            (1.0, float("nan"), 0, float("nan")), (float("inf"), 0.3, 0, 0.0), (1.0, 0.99999994, 0, 0.0), (0.5, 0.7, 0xFFFFFFFF, 0.3)]


@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 2049, 32000])
@pytest.mark.parametrize("spread", [3.0, 0.01])
def test_settings(hip, rng, vocab, spread):
    params = [s for s in SETTINGS for _ in range(3)]
    logits = (spread * rng.standard_normal((len(params), vocab))).astype(np.float32)
    check(hip, logits, params, rng.random(len(params)).astype(np.float32), stride=vocab + int(vocab) % 3)


@pytest.mark.parametrize("rows", [1, 7, 70])
def test_large_vocabulary(hip, rng, rows):
    vocab = 131072
    logits = (2.2 * rng.standard_normal((rows, vocab))).astype(np.float32)
    for r in range(rows):
        logits[r, rng.integers(0, vocab, 50)] += 12 * rng.random(50).astype(np.float32) ** 2
    params = [SETTINGS[(3 + r) % len(SETTINGS)] for r in range(rows)]
    check(hip, logits, params, rng.random(rows).astype(np.float32))


@pytest.mark.parametrize("u", [0.0, 1e-30, 0.25, 0.5, 0.75, 0.99999994, 1.0, 5.0, -1.0, float("nan"), float("inf")])
def test_draws_at_the_ends(hip, rng, u):
    logits = np.array([[0, 0, 0, 0], [-1, 2, 2, 5], [3, 3, -np.inf, 3], [0, -200, -200, 0]], np.float32)
    tokens, probs = run(hip, logits, [(1.0, 1.0, 0, 0.0)] * 4, [u] * 4)
    # four equal tokens: u in quarters
    want = 3 if u >= 1 else 0 if not u > 0 else int(u * 4)
    assert tokens[0] == want and probs[0] == 0.25
    for r in range(4):
        assert tokens[r] == sample(logits[r], 1.0, 1.0, 0, 0.0, u)[0]


def test_ties_go_by_index(hip):
    """Equal logits at every cut: top-k, top-p, min-p and the draw, in the list and, of 20000, in the row itself."""
    for vocab in (40, 20000):
        logits = np.zeros((6, vocab), np.float32)
        logits[:, 5] = 1
        logits[1, ::2] = -0.0  # ranks below 0, with its weight
        n = vocab // 4
        params = [(1.0, 1.0, n, 0.0), (1.0, 1.0, n, 0.0), (1.0, 0.5, 0, 0.0), (1.0, 1.0, 0, 0.36), (1.0, 1.0, 0, 0.37), (0.5, 0.25, n, 0.1)]
        for u in (0.0, 0.31, 0.77, 0.999999):
            check(hip, logits, params, [u] * 6)


def test_not_finite(hip, rng):
    """-inf and NaN are no candidates, nor is +inf but for a greedy row; a row of nothing else takes the argmax."""
    logits = rng.standard_normal((7, 3000)).astype(np.float32)
    logits[0, ::2] = -np.inf
    logits[1, 1::2] = np.nan
    logits[2, 2000], logits[2, 100] = np.inf, np.inf
    logits[3] = -np.inf
    logits[4] = np.nan
    logits[5] = np.nan
    logits[5, 2222] = np.inf
    logits[6, :-1] = -3.4e38
    params = [(1.0, 0.95, 400, 0.0)] * 7
    tokens = check(hip, logits, params, rng.random(7).astype(np.float32))
    assert list(tokens[3:6]) == [0, 0, 2222] and tokens[6] == 2999
    greedy = check(hip, logits, [(0.0, 1.0, 0, 0.0)] * 7, [0.5] * 7)
    assert greedy[2] == 100
    assert not np.isnan(run(hip, logits, params, [0.3] * 7)[1]).any()


@pytest.mark.parametrize("vocab", [8192, 8193, 12000])
def test_one_bin_holds_all(hip, rng, vocab):
    """Logits within 2^-10 of each other, just as many as the list takes and more."""
    logits = (7 + 0.0005 * rng.random((8, vocab))).astype(np.float32)
    params = [(1.0, 1.0, 0, 0.0), (1.0, 0.4, 0, 0.0), (1e-4, 0.9, 0, 0.0), (1.0, 1.0, 777, 0.0), (1e-4, 1.0, 0, 0.3), (1e-4, 0.9, 6000, 0.001),
              (1e-5, 1.0, 0, 0.0), (1.0, 0.9, 5000, 0.9999)]
    check(hip, logits, params, rng.random(8).astype(np.float32))


def test_agrees_with_the_host_sampler(hip, rng):
    """The same uniform number gives gh_sample's token where FP32 sums do not decide."""
    vocab, rows = 4000, 60
    logits = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    params = [SETTINGS[2 + r % 6] for r in range(rows)]
    lib, u, want = hip.lib, [], []
    for r in range(rows):
        state = C.c_uint64(lib.gh_rng_seed(100 + r))
        p = GhSampling(params[r][0], params[r][1], params[r][2], params[r][3], 1.0, 0)
        row, token, copy = logits[r].copy(), C.c_uint32(), C.c_uint64(state.value)
        u.append(lib.gh_rng_next_f32(C.byref(copy)))
        assert lib.gh_sample(row.ctypes.data, vocab, C.byref(p), None, 0, C.byref(state), C.byref(token)) == 0
        want.append(token.value)
    tokens, _ = run(hip, logits, params, u)
    sure = 0
    for r in range(rows):
        if sample(logits[r], *params[r], u[r])[2] > 1e-4:
            assert tokens[r] == want[r], r
            sure += 1
    assert sure > rows // 2


def test_repeats_and_needs_no_probs(hip, rng):
    logits = (2 * rng.standard_normal((20, 50000))).astype(np.float32)
    params, u = [SETTINGS[2 + i % 8] for i in range(20)], rng.random(20).astype(np.float32)
    first = run(hip, logits, params, u)
    for _ in range(3):
        again = run(hip, logits, params, u)
        assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
    tokens, probs = run(hip, logits, params, u, probs=False)
    assert np.array_equal(tokens, first[0]) and (probs == 77).all()


def test_rows_in_turns(hip, rng):
    """More rows than the scratch takes at once, and almost no memory for it."""
    rows, vocab = 2000, 257
    logits = rng.standard_normal((rows, vocab)).astype(np.float32)
    params, u = [SETTINGS[r % len(SETTINGS)] for r in range(rows)], rng.random(rows).astype(np.float32)
    check(hip, logits, params, u)
    from graph_horizon_amd import HipBackend
    with HipBackend(0) as other:
        other.set_scratch_limit(1 << 20)
        check(other, logits[:40], params[:40], u[:40])


def test_frequencies(hip, rng):
    """Drawn as often as the weights say: 4000 draws of eight tokens, each within five standard deviations."""
    logits = np.tile(np.log(np.array([1, 2, 3, 4, 5, 6, 7, 8], np.float32)), (4000, 1))
    tokens, _ = run(hip, logits, [(1.0, 1.0, 0, 0.0)] * 4000, rng.random(4000).astype(np.float32))
    n = np.bincount(tokens, minlength=8)
    p = np.arange(1, 9) / 36
    assert np.all(np.abs(n - 4000 * p) <= 5 * np.sqrt(4000 * p * (1 - p)))
