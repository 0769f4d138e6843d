"""The checks and launch plans of the operators over 4-bit pools, of norms with RoPE and of sampling, without a device
(tests/rows_host.cpp). Every refused call launches nothing and is latched; every accepted one stays within its scratch."""
import ctypes as C
import os
import random
import subprocess

import pytest

from graph_horizon_amd import _ffi as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SCRATCH = 1 << 50
INVALID, OOM, RANGE, STATE, UNSUPPORTED = -1, -4, -5, -7, -8
NAN, INF = float("nan"), float("inf")
YARN = F.GhYarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)


class Launch(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in ("kernel", "gx", "gy", "gz", "block")] + [("args", C.c_ubyte * 512)]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("rows") / "rows_host.so")
    host = os.path.join(ROOT, "graph_horizon_amd", "csrc", "host")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-Wall", "-Werror", "-o", out, os.path.join(ROOT, "tests", "rows_host.cpp"),
                    os.path.join(host, "paged.cpp"), os.path.join(host, "rows.cpp")], check=True)
    h = C.CDLL(out)
    for name in ("gh_kv_write_paged", "gh_rope_kv_write_paged", "gh_norm_rope_kv_write_paged", "gh_kv_read_paged",
                 "gh_attention_decode_paged", "gh_kv_evict_paged", "gh_norm_rope_batched", "gh_sample_rows"):
        getattr(h, name).argtypes = F.SIGNATURES[name][1]
    h.host_backend.restype = h.host_encoder.restype = h.host_launch.restype = C.c_void_p
    h.host_encoder.argtypes = h.host_latched.argtypes = h.host_error.argtypes = [C.c_void_p]
    h.host_reset.argtypes = [C.c_void_p, C.c_uint64]
    h.host_scratch.restype = C.c_uint64
    h.host_error.restype = h.host_kernel.restype = C.c_char_p
    return h


class Host:
    def __init__(self, lib, cus=256):
        self.lib, self.b = lib, lib.host_backend(cus)
        self.enc = lib.host_encoder(self.b)
        self.at = 1 << 40

    def buf(self, nbytes, off=0):
        b = F.GhBuf(self.at + off, nbytes, 0, F.BUF_ALLOC, 0, 0)
        self.at += (nbytes + 4095 + off) // 4096 * 4096
        return b

    def kv(self, layers=2, slots=1024, heads=2, page=16, width=8, rows=3, scored=False, scheme=F.KV_Q4):
        cache = layers * slots * heads * (80 if scheme == F.KV_Q4 else 256)
        pool = F.GhKv(self.buf(cache), self.buf(cache), scheme, layers, slots, heads, 128, 128)
        score = self.buf(layers * rows * heads * width * page * 4) if scored else F.GhBuf()
        return F.GhKvPaged(pool, self.buf(rows * width * 4), self.buf(rows * 4), score, page, width, rows)

    def call(self, name, *args, limit=0):
        """(status, launches as (kernel, launch)) of a call; a refused one has launched nothing and is latched."""
        self.lib.host_reset(self.b, limit)
        args = [C.byref(a) if isinstance(a, C.Structure) else a for a in args]
        rc = getattr(self.lib, name)(self.b, self.enc, *args)
        got = [Launch.from_buffer_copy(C.string_at(self.lib.host_launch(i), C.sizeof(Launch)))
               for i in range(self.lib.host_launches())]
        assert rc == self.lib.host_latched(self.b)
        if rc:
            assert not got and self.lib.host_error(self.b)
        return rc, [(self.lib.host_kernel(g.kernel).decode(), g) for g in got]

    def field(self, launch, name, ctype=C.c_uint64):
        at = self.lib.host_offset(name.encode())
        assert at != 0xFFFFFFFF
        return ctype.from_buffer_copy(bytes(launch.args)[at:at + C.sizeof(ctype)]).value


@pytest.fixture
def host(lib):
    return Host(lib)


def part(b, off, nbytes=None):
    return F.GhBuf(b.addr + off, b.bytes if nbytes is None else nbytes, 0, F.BUF_VIEW, 0, 0)


def shorter(b, by=1):
    return F.GhBuf(b.addr, b.bytes - by, b.format, b.kind, 0, 0)


# ---- 4-bit pools ----

def test_a_q4_pool_is_a_third_of_an_fp16_one(host):
    kv = host.kv()
    k = host.buf(3 * 2 * 256)
    assert host.call("gh_kv_write_paged", kv, k, k, 1, 1)[1][0][0] == "write4"
    kv.kv.k = shorter(kv.kv.k)
    assert host.call("gh_kv_write_paged", kv, k, k, 1, 1)[0] == RANGE
    kv = host.kv()
    kv.kv.scheme = F.KV_F16
    assert host.call("gh_kv_write_paged", kv, k, k, 1, 1)[0] == RANGE
    for scheme in (F.KV_INT8, 3, 0xFFFFFFFF):
        kv.kv.scheme = scheme
        assert host.call("gh_kv_write_paged", kv, k, k, 1, 1)[0] == UNSUPPORTED


def test_layers_of_a_q4_pool(host):
    """A layer's caches start layer · slots · heads · 80 bytes on."""
    kv, k = host.kv(layers=3, slots=64, heads=5), host.buf(3 * 5 * 256)
    _, got = host.call("gh_kv_write_paged", kv, k, k, 1, 2)
    assert C.c_uint64.from_buffer_copy(bytes(got[0][1].args)[:8]).value == kv.kv.k.addr + 2 * 64 * 5 * 80


def test_read_refusals(host):
    for scheme, kernel in ((F.KV_Q4, "read4"), (F.KV_F16, "read")):
        kv, n = host.kv(scored=True, scheme=scheme), 3 * 5 * 2 * 256
        k, v = host.buf(n), host.buf(n)
        rc, got = host.call("gh_kv_read_paged", k, v, kv, 5, 1)
        assert rc == 0 and [g[0] for g in got] == [kernel] and got[0][1].gx == 15
        both = host.buf(2 * n)
        assert host.call("gh_kv_read_paged", both, part(both, n, n), kv, 5, 1)[0] == 0
        for args, status in (((k, v, kv, 0, 0), INVALID), ((k, v, kv, 6, 0), RANGE), ((shorter(k), v, kv, 5, 0), RANGE),
                             ((k, part(v, 8), kv, 5, 0), RANGE), ((k, None, kv, 5, 0), RANGE), ((k, v, kv, 5, 2), RANGE),
                             ((k, v, kv, 0xFFFFFFFF, 0), INVALID), ((k, v, None, 5, 0), INVALID), ((k, k, kv, 5, 0), INVALID),
                             ((both, part(both, n - 16, n), kv, 5, 0), INVALID), ((part(kv.kv.k, 0), v, kv, 5, 0), INVALID),
                             ((k, part(kv.score, 0, n), kv, 5, 0), INVALID), ((k, part(kv.table, 0, n), kv, 5, 0), INVALID),
                             ((part(kv.lengths, 0, n), v, kv, 5, 0), INVALID)):
            assert host.call("gh_kv_read_paged", *args)[0] == status, args


def test_norm_write_refusals(host):
    name = "gh_norm_rope_kv_write_paged"
    for scheme, kernel in ((F.KV_Q4, "norm_write4"), (F.KV_F16, "norm_write")):
        kv = host.kv(scored=True, scheme=scheme)
        q, o, k, v = host.buf(3 * 8 * 256), host.buf(3 * 8 * 256), host.buf(3 * 2 * 256), host.buf(3 * 2 * 256)
        wq, wk, pos = host.buf(256), host.buf(256), host.buf(12)

        def call(kv=kv, o=o, q=q, k=k, v=v, heads=8, wq=wq, wk=wk, eps=1e-5, pos=pos, tokens=1, most=9, yarn=YARN, layer=0):
            return host.call(name, kv, o, q, k, v, heads, wq, wk, eps, pos, tokens, most, yarn, layer)

        rc, got = call()
        assert rc == 0 and [g[0] for g in got] == [kernel]
        assert call(o=q)[0] == 0 and call(wk=wq)[0] == 0 and call(eps=0.0)[0] == 0
        for status, change in (
                (INVALID, dict(eps=-1e-9)), (INVALID, dict(eps=NAN)), (INVALID, dict(eps=INF)), (RANGE, dict(wq=None)), (RANGE, dict(wk=shorter(wk))),
                (RANGE, dict(wq=part(host.buf(512), 8, 256))), (INVALID, dict(wq=part(o, 256, 256))), (INVALID, dict(wk=part(kv.kv.k, 80 * 16, 256))),
                (INVALID, dict(wk=part(kv.kv.v, 0, 256))), (INVALID, dict(wk=part(kv.score, 16, 256))), (INVALID, dict(o=q, wq=part(q, 0, 256))),
                (RANGE, dict(most=262144)), (INVALID, dict(yarn=None)), (INVALID, dict(heads=0)), (RANGE, dict(heads=9)), (RANGE, dict(pos=None)),
                (INVALID, dict(tokens=0)), (RANGE, dict(tokens=2)), (RANGE, dict(layer=2)), (INVALID, dict(kv=None)), (RANGE, dict(o=None)),
                (INVALID, dict(o=part(q, 256, q.bytes)))):
            assert call(**change)[0] == status, change


@pytest.mark.parametrize("seed", range(60))
def test_attention_plans_stay_within_their_scratch(host, seed):
    """The spans or chunks cover the rows; the partials, their (m, l), the scores and the layout lie in the scratch and
    apart; the groups of rows cover all rows once; spans are whole numbers of tiles for each of four waves."""
    rng = random.Random(seed)
    heads, group = rng.choice((1, 2, 3, 8, 64)), rng.randint(1, 16)
    page, rows = rng.choice((16, 64, 1024)), int(2 ** rng.uniform(0, 11))
    width, scored = max(1, int(2 ** rng.uniform(4, 18)) // page), rng.random() < 0.5
    kv = host.kv(layers=1, slots=page * 4, heads=heads, page=page, width=width, rows=rows, scored=scored)
    q = host.buf(rows * heads * group * 256)
    max_len = rng.choice((0, rng.randint(1, width * page)))
    rc, got = host.call("gh_attention_decode_paged", q, q, kv, heads * group, max_len, 0)
    assert rc == 0
    want, size, at = max_len or width * page, host.lib.host_scratch(), 0
    for kernel, g in got:
        f = lambda name, t=C.c_uint64: host.field(g, "GhPagedAttnArgs." + name, t)  # noqa: E731
        u = lambda name: f(name, C.c_uint32)  # noqa: E731
        split = f("layout") == 0
        assert u("max_len") == want and u("raw_len") >= want and u("raw_len") % 32 == 0 and u("rows") <= 512
        assert g.gy <= 65535 and g.gz <= 65535 and g.gx * g.gy * g.gz < 2 ** 32 and g.block == 256
        row = (f("q") - q.addr) // (heads * group * 256)
        if kernel in ("attn4", "split4"):
            assert row == at
            at += u("rows")
        if split:
            parts = u("chunks") * u("rows")
            assert u("least") % 8 == 0 and u("least") <= 512 and 16 * u("least") * u("chunks") >= want
            assert kernel != "split4" or (g.gx == 8 * heads and 8 * g.gy >= parts > 8 * (g.gy - 1) and g.gz == 1)
            assert kernel != "attn4"
        else:
            parts = u("chunks") + u("rows")
            assert kernel != "split4" and f("layout") + 4 * (u("rows") + 2) <= f("part_acc")
        spans = [(f("part_acc"), parts * heads * group * 512), (f("part_ml"), parts * heads * group * 8)]
        if scored:
            spans.append((f("raw"), u("rows") * heads * group * u("raw_len") * 4))
        spans.sort()
        assert spans[0][0] >= SCRATCH and spans[-1][0] + spans[-1][1] <= SCRATCH + size
        assert all(a + n <= b for (a, n), (b, _) in zip(spans, spans[1:]))
    assert at == rows


def test_evict_takes_pools_of_one_scheme(host):
    name = "gh_kv_evict_paged"
    src, dst = host.kv(scored=True), host.kv(scored=True, width=3)
    rc, got = host.call(name, dst, src, None, 40, 4)
    assert rc == 0 and [g[0] for g in got] == ["select", "move4"]
    assert host.field(got[1][1], "GhPagedEvictArgs.src_layer") == 1024 * 2 * 80
    assert host.call(name, host.kv(scored=True, width=3, scheme=F.KV_F16), src, None, 40, 4)[0] == INVALID


# ---- norms and RoPE ----

def test_norm_rope_refusals(host):
    q, k, wq, wk = host.buf(5 * 8 * 256), host.buf(5 * 2 * 256), host.buf(256), host.buf(256)

    def call(q=q, k=k, heads=8, kv_heads=2, dim=128, base=0, rows=5, wq=wq, wk=wk, eps=1e-5, yarn=YARN):
        return host.call("gh_norm_rope_batched", q, k, heads, kv_heads, dim, base, rows, wq, wk, eps, yarn)

    rc, got = call()
    assert rc == 0 and [g[0] for g in got] == ["norm_rope"] and got[0][1].gx == 5
    assert call(wk=wq)[0] == 0 and call(base=262139)[0] == 0 and call(heads=0, kv_heads=0) == (0, [])
    wide = F.GhYarn(130, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    for status, change in (
            (INVALID, dict(rows=0)), (UNSUPPORTED, dict(dim=0)), (UNSUPPORTED, dict(dim=124)), (UNSUPPORTED, dict(dim=520)), (INVALID, dict(yarn=wide)),
            (INVALID, dict(yarn=None)), (INVALID, dict(eps=NAN)), (INVALID, dict(eps=-1.0)), (INVALID, dict(eps=INF)), (RANGE, dict(base=262140)),
            (RANGE, dict(base=0xFFFFFFFE)), (RANGE, dict(rows=6)), (RANGE, dict(rows=0xFFFFFFFF)), (RANGE, dict(q=None)), (RANGE, dict(k=None)),
            (RANGE, dict(wq=None)), (RANGE, dict(wk=shorter(wk))), (RANGE, dict(heads=9)), (UNSUPPORTED, dict(heads=65536)), (RANGE, dict(q=part(host.buf(5 * 8 * 256 + 16), 2))),
            (RANGE, dict(wq=part(host.buf(512), 8, 256))), (INVALID, dict(k=part(q, 256, 5 * 2 * 256))), (INVALID, dict(wq=part(q, 0, 256))),
            (INVALID, dict(wk=part(k, 16, 256)))):
        assert call(**change)[0] == status, change


@pytest.mark.parametrize("dim,lanes", [(8, 1), (16, 2), (24, 4), (40, 8), (64, 8), (96, 16), (128, 16), (256, 32), (264, 64), (512, 64)])
def test_norm_rope_grids_hold_whole_heads(host, dim, lanes):
    yarn = F.GhYarn(8, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    for heads, kv_heads in ((1, 0), (32, 8), (0, 3), (100, 100)):
        q, k, w = host.buf(max(1, 7 * heads * dim * 2)), host.buf(max(1, 7 * kv_heads * dim * 2)), host.buf(dim * 2)
        _, got = host.call("gh_norm_rope_batched", q, k, heads, kv_heads, dim, 3, 7, w, w, 0.0, yarn)
        assert got[0][1].gx == 7 * -(-(heads + kv_heads) * lanes // 256)


# ---- sampling ----

def sample_args(host, rows=3, vocab=1000, stride=1000):
    return dict(tokens=host.buf(rows * 4), probs=host.buf(rows * 4), logits=host.buf(((rows - 1) * stride + vocab) * 4), rows=rows, vocab=vocab,
                stride=stride, params=host.buf(rows * 16), uniform=host.buf(rows * 4))


def call_sample(host, limit=0, **a):
    return host.call("gh_sample_rows", a["tokens"], a["probs"], a["logits"], a["rows"], a["vocab"], a["stride"], a["params"], a["uniform"], limit=limit)


def test_sample_refusals(host):
    good = sample_args(host)
    rc, got = call_sample(host, **good)
    assert rc == 0 and [g[0] for g in got] == ["sample_max", "sample_bins", "sample_collect", "sample_pick"]
    assert call_sample(host, **dict(good, probs=None))[0] == 0
    g = good
    for status, change in (
            (INVALID, dict(rows=0)), (INVALID, dict(rows=65536)), (INVALID, dict(vocab=0)), (INVALID, dict(stride=999)), (UNSUPPORTED, dict(vocab=(1 << 24) + 1, stride=1 << 25)),
            (RANGE, dict(rows=4)), (RANGE, dict(tokens=None)), (RANGE, dict(logits=None)), (RANGE, dict(params=None)), (RANGE, dict(uniform=None)),
            (RANGE, dict(tokens=shorter(g["tokens"]))), (RANGE, dict(probs=shorter(g["probs"]))), (RANGE, dict(logits=shorter(g["logits"]))),
            (RANGE, dict(params=shorter(g["params"]))), (RANGE, dict(uniform=shorter(g["uniform"]))), (RANGE, dict(stride=1001)),
            (RANGE, dict(params=part(host.buf(100), 8, 48))), (RANGE, dict(tokens=part(host.buf(100), 2, 12))), (RANGE, dict(logits=part(host.buf(13000), 2, 12000))),
            (INVALID, dict(tokens=part(g["logits"], 400, 12))), (INVALID, dict(probs=part(g["params"], 0, 12))), (INVALID, dict(tokens=g["uniform"])),
            (INVALID, dict(probs=g["tokens"])), (INVALID, dict(probs=part(g["uniform"], 8, 12)))):
        assert call_sample(host, **dict(g, **change))[0] == status, change
    assert call_sample(host, limit=1000, **good)[0] == OOM
    assert host.lib.gh_sample_rows(host.b, None, None, None, None, 1, 1, 1, None, None) == STATE


@pytest.mark.parametrize("seed", range(40))
def test_sample_plans(host, seed):
    """Chunks cover the row in at most 64 parts; each row of a group has its scratch, apart and within; the groups cover all
    rows once, with little memory too; weights of all tokens sum up to at most 2^62."""
    rng = random.Random(seed)
    rows, vocab = int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 24))
    stride = vocab + rng.choice((0, 1, 4))
    a = sample_args(host, rows, vocab, stride)
    limit = rng.choice((0, 0, 500000, 79000))
    rc, got = call_sample(host, limit=limit, **a)
    assert rc == 0
    row_bytes, bin_bytes, list_bytes = (host.lib.host_sample_bytes(i) for i in range(3))
    at = 0
    for kernel, g in got:
        f = lambda name, t=C.c_uint64: host.field(g, "GhSampleArgs." + name, t)  # noqa: E731
        chunks, per = f("chunks", C.c_uint32), f("per", C.c_uint32)
        assert 1 <= chunks <= 64 and per % 4 == 0 and (chunks - 1) * per < vocab <= chunks * per
        n = g.gx if kernel == "sample_pick" else g.gy
        assert kernel == "sample_pick" or g.gx == chunks
        if kernel == "sample_max":
            assert f("logits") == a["logits"].addr + at * stride * 4 and f("tokens") == a["tokens"].addr + 4 * at
            assert f("params") == a["params"].addr + 16 * at and f("uniform") == a["uniform"].addr + 4 * at and f("probs") == a["probs"].addr + 4 * at
            at += n
        spans = sorted([(f("part"), n * 1024), (f("bins"), n * bin_bytes), (f("list"), n * list_bytes)])
        assert spans[0][0] >= SCRATCH and spans[-1][0] + spans[-1][1] <= SCRATCH + host.lib.host_scratch()
        assert all(x + y <= z for (x, y), (z, _) in zip(spans, spans[1:])) and f("bins") % 8 == 0 and f("part") % 16 == 0
        scale = f("scale", C.c_double)
        assert scale <= 2.0 ** 51 and scale * vocab <= 2.0 ** 62 and (scale == 2.0 ** 51 or 2.0 ** 61 < scale * vocab)
        assert scale == 2.0 ** f("shift", C.c_int32)
        assert not f("wide", C.c_uint32) or stride % 4 == 0
    assert at == rows
