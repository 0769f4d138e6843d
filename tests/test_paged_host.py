"""The checks and launch plans of the operators over paged caches, without a device: host/paged.cpp built
with recorded launches (tests/paged_host.cpp). Every refused call launches nothing and is latched; every
accepted one stays within its buffers and scratch."""
import ctypes as C
import os
import random
import subprocess

import pytest

from graph_horizon_amd import _ffi as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SCRATCH = 1 << 50
INVALID, OOM, RANGE, STATE, UNSUPPORTED = -1, -4, -5, -7, -8


class Pages(C.Structure):
    _fields_ = [(n, C.c_uint64) for n in ("kc", "vc", "table", "lengths", "score", "fault")] + \
               [(n, C.c_uint32) for n in ("width", "shift", "pages", "kv_heads")]


class AttnArgs(C.Structure):
    _fields_ = [("p", Pages)] + [(n, C.c_uint64) for n in ("q", "out", "part_acc", "part_ml", "raw", "stream", "layout")] + \
               [(n, C.c_uint32) for n in ("q_heads", "group", "rows", "max_len", "chunks", "least", "solo", "raw_len")] + \
               [("scale", C.c_float), ("blocks", C.c_uint32)]


class Launch(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in ("kernel", "gx", "gy", "gz", "block")] + [("args", C.c_ubyte * 512)]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("paged") / "paged_host.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    "-Wall", "-Werror", "-o", out, os.path.join(ROOT, "tests", "paged_host.cpp"),
                    os.path.join(ROOT, "graph_horizon_amd", "csrc", "host", "paged.cpp")], check=True)
    h = C.CDLL(out)
    for name in ("gh_kv_write_paged", "gh_rope_kv_write_paged", "gh_attention_decode_paged", "gh_kv_evict_paged"):
        getattr(h, name).argtypes = F.SIGNATURES[name][1]
    h.host_backend.restype = h.host_encoder.restype = h.host_launch.restype = C.c_void_p
    h.host_encoder.argtypes = h.host_latched.argtypes = h.host_error.argtypes = [C.c_void_p]
    h.host_reset.argtypes = [C.c_void_p, C.c_uint64]
    h.host_scratch.restype = C.c_uint64
    h.host_error.restype = C.c_char_p
    return h


class Host:
    def __init__(self, lib, cus=256):
        self.lib, self.b = lib, lib.host_backend(cus)
        self.enc = lib.host_encoder(self.b)
        self.at = 1 << 40
        ids = (C.c_uint32 * 6)()
        lib.host_kernels(ids)
        self.ids = dict(zip(("write", "attn", "join", "select", "move", "join2"), ids))

    def buf(self, nbytes, off=0):
        b = F.GhBuf(self.at + off, nbytes, 0, F.BUF_ALLOC, 0, 0)
        self.at += (nbytes + 4095 + off) // 4096 * 4096
        return b

    def kv(self, layers=2, slots=1024, heads=2, page=16, width=8, rows=3, scored=False):
        cache = layers * slots * heads * 256
        pool = F.GhKv(self.buf(cache), self.buf(cache), F.KV_F16, layers, slots, heads, 128, 128)
        score = self.buf(layers * rows * heads * width * page * 4) if scored else F.GhBuf()
        return F.GhKvPaged(pool, self.buf(rows * width * 4), self.buf(rows * 4), score, page, width, rows)

    def call(self, name, *args, limit=0):
        """(status, launches) of a call; a refused one has launched nothing and is latched."""
        self.lib.host_reset(self.b, limit)
        args = [C.byref(a) if isinstance(a, C.Structure) else a for a in args]
        rc = getattr(self.lib, name)(self.b, self.enc, *args)
        got = [Launch.from_buffer_copy(C.string_at(self.lib.host_launch(i), C.sizeof(Launch)))
               for i in range(self.lib.host_launches())]
        assert rc == self.lib.host_latched(self.b)
        if rc:
            assert not got and self.lib.host_error(self.b)
        return rc, got


@pytest.fixture
def host(lib):
    return Host(lib)


def shift_buf(b, off):
    return F.GhBuf(b.addr + off, b.bytes, b.format, b.kind, 0, 0)


def shorter(b, by=1):
    return F.GhBuf(b.addr, b.bytes - by, b.format, b.kind, 0, 0)


def handles(host):
    """(what is wrong, status, handle): the handle checks that every entry point makes."""
    def change(status, what, **fields):
        kv = host.kv(scored=True)
        for k, v in fields.items():
            target = kv.kv if k in ("scheme", "head_dim", "value_dim", "kv_heads", "context", "k", "v") else kv
            setattr(target, k, v(getattr(target, k)) if callable(v) else v)
        return what, status, kv

    yield change(UNSUPPORTED, "scheme", scheme=1)
    yield change(UNSUPPORTED, "head_dim", head_dim=64)
    yield change(UNSUPPORTED, "value_dim", value_dim=256)
    yield change(INVALID, "no kv heads", kv_heads=0)
    for page in (0, 1, 8, 24, 48, 65536):
        yield change(INVALID, "page_size %d" % page, page_size=page)
    yield change(INVALID, "no slots", context=0)
    yield change(INVALID, "part of a page", context=1023)
    yield change(RANGE, "more slots than memory", context=2048)
    yield change(RANGE, "context overflows", context=0xFFFFFFF0)
    yield change(INVALID, "no rows", rows=0)
    yield change(INVALID, "too many rows", rows=65536)
    yield change(INVALID, "no table", table_width=0)
    yield change(INVALID, "positions past 31 bits", table_width=1 << 27)
    for name in ("k", "v", "table", "lengths", "score"):
        yield change(RANGE, name + " too small", **{name: shorter})
        yield change(RANGE, name + " not aligned", **{name: lambda b: shift_buf(b, 2)})
    for name in ("k", "v", "table", "lengths"):
        yield change(RANGE, name + " missing", **{name: F.GhBuf()})


def test_handles_are_checked_by_every_entry_point(host):
    big = host.buf(1 << 30)
    yarn = F.GhYarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    count = 0
    for what, status, kv in handles(host):
        good = host.kv(scored=True)
        for name, args in (("gh_kv_write_paged", (kv, big, big, 1, 0)),
                           ("gh_rope_kv_write_paged", (kv, big, big, big, big, 8, big, 1, 100, yarn, 0)),
                           ("gh_attention_decode_paged", (big, big, kv, 8, 0, 0)),
                           ("gh_kv_evict_paged", (good, kv, None, 8, 1)), ("gh_kv_evict_paged", (kv, good, None, 8, 1))):
            assert host.call(name, *args)[0] == status, (what, name)
            count += 1
    assert count > 150
    assert host.lib.gh_kv_write_paged(host.b, None, None, None, None, 1, 0) == STATE
    assert host.call("gh_kv_write_paged", None, big, big, 1, 0)[0] == INVALID


def test_write_refusals(host):
    kv = host.kv()
    n = 3 * 5 * 2 * 256
    k, v = host.buf(n), host.buf(n)
    assert host.call("gh_kv_write_paged", kv, k, v, 5, 1)[0] == 0
    for args, status in (((kv, k, v, 0, 0), INVALID), ((kv, k, v, 6, 0), RANGE), ((kv, shorter(k), v, 5, 0), RANGE),
                         ((kv, k, shorter(v), 5, 0), RANGE), ((kv, shift_buf(k, 8), v, 5, 0), RANGE),
                         ((kv, k, None, 5, 0), RANGE), ((kv, k, v, 5, 2), RANGE), ((kv, k, v, 0xFFFFFFFF, 0), INVALID)):
        assert host.call("gh_kv_write_paged", *args)[0] == status


def test_rope_write_refusals(host):
    kv = host.kv()
    q, o, k, v = host.buf(3 * 8 * 256), host.buf(3 * 8 * 256), host.buf(3 * 2 * 256), host.buf(3 * 2 * 256)
    pos, yarn = host.buf(12), F.GhYarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    name = "gh_rope_kv_write_paged"
    assert host.call(name, kv, o, q, k, v, 8, pos, 1, 262143, yarn, 0)[0] == 0
    assert host.lib.host_rope_positions(C.c_void_p(host.b)) == 262144
    assert host.call(name, kv, q, q, k, v, 8, pos, 1, 0, yarn, 0)[0] == 0  # in place
    wide = F.GhYarn(130, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    for args, status in (((kv, o, q, k, v, 8, pos, 1, 262144, yarn, 0), RANGE), ((kv, o, q, k, v, 8, pos, 1, 9, None, 0), INVALID),
                         ((kv, o, q, k, v, 8, pos, 1, 9, wide, 0), INVALID), ((kv, o, q, k, v, 0, pos, 1, 9, yarn, 0), INVALID),
                         ((kv, o, q, k, v, 9, pos, 1, 9, yarn, 0), RANGE), ((kv, shorter(o), q, k, v, 8, pos, 1, 9, yarn, 0), RANGE),
                         ((kv, o, q, k, v, 8, shorter(pos), 1, 9, yarn, 0), RANGE), ((kv, o, q, k, v, 8, None, 1, 9, yarn, 0), RANGE),
                         ((kv, o, None, k, v, 8, pos, 1, 9, yarn, 0), RANGE), ((kv, o, q, k, v, 8, pos, 0, 9, yarn, 0), INVALID),
                         ((kv, F.GhBuf(q.addr + 256, 3 * 8 * 256, 0, 1, 0, 0), q, k, v, 8, pos, 1, 9, yarn, 0), INVALID)):
        assert host.call(name, *args)[0] == status, args


def test_attention_refusals(host):
    kv = host.kv(scored=True)
    q, o = host.buf(3 * 8 * 256), host.buf(3 * 8 * 256)
    name = "gh_attention_decode_paged"
    assert host.call(name, o, q, kv, 8, 128, 1)[0] == 0
    for args, status in (((o, q, kv, 0, 0, 0), INVALID), ((o, q, kv, 7, 0, 0), INVALID), ((o, q, kv, 34, 0, 0), UNSUPPORTED),
                         ((o, q, kv, 8, 129, 0), RANGE), ((o, q, kv, 8, 0, 2), RANGE), ((o, q, kv, 10, 0, 0), RANGE),
                         ((shorter(o), q, kv, 8, 0, 0), RANGE), ((o, shift_buf(q, 4), kv, 8, 0, 0), RANGE),
                         ((None, q, kv, 8, 0, 0), RANGE)):
        assert host.call(name, *args)[0] == status, args
    wide = host.kv(heads=9000, slots=16, layers=1, rows=1)
    assert host.call(name, q, q, wide, 72000, 0, 0)[0] == UNSUPPORTED
    assert host.call(name, o, q, kv, 8, 0, 0, limit=1000)[0] == OOM
    # with room for some of the rows, as many launches as it takes
    many = host.kv(rows=40, width=64, slots=1024, scored=True)
    q = host.buf(40 * 8 * 256)
    rc, whole = host.call(name, q, q, many, 8, 0, 0)
    rc2, parts = host.call(name, q, q, many, 8, 0, 0, limit=host.lib.host_scratch() // 3)
    assert rc == rc2 == 0 and len(whole) == 2 and len(parts) > 4
    args = [AttnArgs.from_buffer_copy(bytes(g.args)) for g in parts if g.kernel not in (host.ids["join"], host.ids["join2"])]
    assert sum(a.rows for a in args) == 40
    assert [(a.q - q.addr) // 2048 for a in args] == [sum(b.rows for b in args[:i]) for i in range(len(args))]


def test_outputs_are_an_input_itself_or_apart(host):
    kv, part = host.kv(), 3 * 8 * 256
    q, k, v, pos = host.buf(3 * part), host.buf(part), host.buf(part), host.buf(12)
    yarn = F.GhYarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)

    def at(b, off):
        return F.GhBuf(b.addr + off, part, 0, F.BUF_ALLOC, 0, 0)

    # views of one buffer: q itself, next to it, and half a vector on
    for off, status in ((0, 0), (part, 0), (2 * part, 0), (part - 16, INVALID), (128, INVALID)):
        assert host.call("gh_attention_decode_paged", at(q, off), q, kv, 8, 0, 0)[0] == status, off
        assert host.call("gh_attention_decode_paged", q, at(q, off), kv, 8, 0, 0)[0] == status, off
        assert host.call("gh_rope_kv_write_paged", kv, at(q, off), q, k, v, 8, pos, 1, 9, yarn, 0)[0] == status, off
    kv_bytes = 3 * 2 * 256
    for off, status in ((0, INVALID), (kv_bytes - 16, INVALID), (kv_bytes, 0)):
        assert host.call("gh_rope_kv_write_paged", kv, at(k, off), q, k, v, 8, pos, 1, 9, yarn, 0)[0] == status, off
        assert host.call("gh_rope_kv_write_paged", kv, at(v, off), q, k, v, 8, pos, 1, 9, yarn, 0)[0] == status, off


def test_evict_refusals(host):
    name = "gh_kv_evict_paged"
    src, dst = host.kv(scored=True), host.kv(scored=True, width=3)
    kept = host.buf(2 * 3 * 2 * 40 * 4)
    rc, got = host.call(name, dst, src, kept, 40, 40)
    assert rc == 0 and [g.kernel for g in got] == [host.ids["select"], host.ids["move"]]
    same = F.GhKvPaged.from_buffer_copy(src)  # scores and lengths in place, another table
    same.table = host.buf(src.table.bytes)
    assert host.call(name, same, src, None, 40, 0)[0] == 0
    narrow = F.GhKvPaged.from_buffer_copy(dst)
    narrow.score = src.score
    part = F.GhKvPaged.from_buffer_copy(dst)
    part.score = F.GhBuf(src.score.addr + 64, dst.score.bytes, 0, 1, 0, 0)
    lengths = F.GhKvPaged.from_buffer_copy(dst)
    lengths.lengths = F.GhBuf(src.lengths.addr + 4, 12, 0, 1, 0, 0)
    for d, s, k, budget, recent, status in (
            (dst, src, kept, 0, 0, INVALID), (dst, src, kept, 40, 41, INVALID), (dst, src, kept, 49, 1, RANGE),
            (dst, src, shorter(kept), 40, 1, RANGE), (dst, src, shift_buf(kept, 2), 40, 1, RANGE),
            (host.kv(width=3), src, kept, 40, 1, INVALID), (dst, host.kv(), kept, 40, 1, INVALID),
            (host.kv(scored=True, rows=2), src, None, 8, 1, INVALID), (host.kv(scored=True, page=32), src, None, 8, 1, INVALID),
            (host.kv(scored=True, layers=3), src, None, 8, 1, INVALID), (host.kv(scored=True, heads=1), src, None, 8, 1, INVALID),
            (narrow, src, None, 8, 1, INVALID), (part, src, None, 8, 1, INVALID), (lengths, src, None, 8, 1, INVALID)):
        assert host.call(name, d, s, k, budget, recent)[0] == status, (budget, recent, status)
    assert host.call(name, dst, src, None, 40, 1, limit=100)[0] == OOM


@pytest.mark.parametrize("seed", range(60))
def test_attention_plans_stay_within_their_scratch(host, seed):
    """The spans or chunks cover the rows; the regions of the partials, their (m, l), the scores and the layout
    lie in the scratch and apart; the groups of rows cover all rows once; the grid is one that the device takes."""
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
    for g in got:
        a = AttnArgs.from_buffer_copy(bytes(g.args))
        split = a.layout == 0
        assert a.max_len == want and a.raw_len >= want and a.raw_len % 16 == 0 and a.rows <= 512
        assert g.gy <= 65535 and g.gz <= 65535 and g.gx * g.gy * g.gz < 2 ** 32 and g.block == 256
        row = (a.q - q.addr) // (heads * group * 256)
        assert a.out - q.addr == a.q - q.addr and a.p.table - kv.table.addr == row * width * 4
        assert a.p.lengths - kv.lengths.addr == row * 4
        if scored:
            assert a.p.score - kv.score.addr == row * heads * width * page * 4
        if g.kernel in (host.ids["join"], host.ids["join2"]):
            assert row + a.rows == at
            assert (g.gx, g.gy, g.gz) == (heads * group + heads * a.blocks, a.rows, 1 + (g.kernel == host.ids["join2"]))
        else:
            assert row == at
            at += a.rows
            if split:
                assert 4 <= a.least <= 32 and a.chunks * a.least * 16 >= want > (a.chunks - 1) * a.least * 16
                assert g.kernel - host.ids["attn"] == 2 + scored and (g.gx, g.gy, g.gz) == (heads, a.chunks, a.rows)
            else:
                most = a.rows * -(-want // 16)
                assert g.kernel - host.ids["attn"] == scored and most < 2 ** 30
                # enough waves for every chunk that the rows can fill, whatever their lengths
                for total in (1, most // 3 + 1, most):
                    half = -(-2 * total // a.chunks)
                    per = max(a.least, half if half <= a.solo else -(-total // a.chunks))
                    assert -(-total // per) * heads <= 4 * g.gx and -(-total // per) <= a.chunks
        parts = a.chunks * a.rows if split else a.chunks + a.rows
        regions = [(a.part_acc, parts * heads * group * 512), (a.part_ml, parts * heads * group * 8)]
        regions += [(a.raw, a.rows * heads * group * a.raw_len * 4)] if scored else []
        regions += [] if split else [(a.layout, (a.rows + 2) * 4)]
        regions.sort()
        assert all(x % 16 == 0 or x == a.part_ml and x % 8 == 0 for x, _ in regions)
        assert regions[0][0] >= SCRATCH and regions[-1][0] + regions[-1][1] <= SCRATCH + size
        assert all(x + nx <= y for (x, nx), (y, _) in zip(regions, regions[1:]))
    assert at == rows


def at_end(b, size):
    """A buffer of `size` bytes that begins with the last 16 bytes of b."""
    return F.GhBuf(b.addr + (b.bytes - 16) // 16 * 16, size, 0, F.BUF_ALLOC, 0, 0)


def with_(kv, **bufs):
    kv = F.GhKvPaged.from_buffer_copy(kv)
    for name, b in bufs.items():
        setattr(kv.kv if name in ("k", "v") else kv, name, b)
    return kv


def test_what_an_eviction_writes_lies_apart_from_what_it_reads(host):
    """The kept list is read again as positions while scores, lengths and vectors are written: it meets none of the
    handles' buffers; dst's scores, lengths and vectors meet nothing of src's but their own counterparts."""
    name = "gh_kv_evict_paged"
    src, dst = host.kv(scored=True), host.kv(scored=True, width=3)
    kept_bytes = 2 * 3 * 2 * 16 * 4
    for kv in (src, dst):
        for b in (kv.kv.k, kv.kv.v, kv.table, kv.lengths, kv.score):
            for kept in (F.GhBuf(b.addr, kept_bytes, 0, F.BUF_ALLOC, 0, 0), at_end(b, kept_bytes),
                         F.GhBuf(b.addr - kept_bytes + 4, kept_bytes, 0, F.BUF_ALLOC, 0, 0)):
                assert host.call(name, dst, src, kept, 16, 1)[0] == INVALID
        for b in (kv.table, kv.lengths, kv.score):
            behind = F.GhBuf(b.addr + b.bytes, kept_bytes, 0, F.BUF_ALLOC, 0, 0)
            assert host.call(name, dst, src, behind, 16, 1)[0] == 0
    for written in ("score", "lengths", "k", "v"):
        size = getattr(dst.kv if written in "kv" else dst, written).bytes
        for read in ("k", "v", "table", "lengths", "score"):
            if read == written:
                continue
            b = getattr(src.kv if read in "kv" else src, read)
            assert host.call(name, with_(dst, **{written: at_end(b, size)}), src, None, 16, 1)[0] == INVALID, (written, read)
    same = with_(src, table=host.buf(src.table.bytes))  # in place: scores, lengths and pool are src's own
    assert host.call(name, same, src, None, 16, 1)[0] == 0
    assert host.call(name, with_(same, lengths=host.buf(12)), src, None, 16, 1)[0] == 0
    assert host.call(name, src, src, None, 16, 1)[0] == INVALID  # the same pages


def test_eviction_buffers_may_be_parts_of_longer_ones(host):
    """Only the bytes that a call uses count, not what its buffers hold behind them."""
    name = "gh_kv_evict_paged"
    src, dst = host.kv(scored=True), host.kv(scored=True, width=3)
    for field in ("score", "lengths"):
        n, m = getattr(src, field).bytes, getattr(dst, field).bytes
        whole = host.buf(n + m)
        lo = with_(src, **{field: whole})
        hi = with_(dst, **{field: F.GhBuf(whole.addr + n, m, 0, F.BUF_ALLOC, 0, 0)})
        assert host.call(name, hi, lo, None, 40, 1)[0] == 0, field


def test_a_handles_buffers_lie_apart(host):
    big, yarn = host.buf(1 << 30), F.GhYarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    good = host.kv(scored=True)
    names = ("k", "v", "table", "lengths", "score")
    for one in names:
        for other in names:
            if one == other:
                continue
            kv = host.kv(scored=True)
            b, size = (getattr(kv.kv if n in "kv" else kv, n) for n in (one, other))
            kv = with_(kv, **{other: at_end(b, size.bytes)})
            for name, args in (("gh_kv_write_paged", (kv, big, big, 1, 0)),
                               ("gh_rope_kv_write_paged", (kv, big, host.buf(1 << 20), big, big, 8, big, 1, 100, yarn, 0)),
                               ("gh_attention_decode_paged", (big, big, kv, 8, 0, 0)),
                               ("gh_kv_evict_paged", (good, kv, None, 8, 1)), ("gh_kv_evict_paged", (kv, good, None, 8, 1))):
                assert host.call(name, *args)[0] == INVALID, (one, other, name)
    # one allocation, cut up
    kv = host.kv(scored=True)
    whole, at = host.buf(1 << 23), 0
    for n in names:
        size = getattr(kv.kv if n in "kv" else kv, n).bytes
        kv = with_(kv, **{n: F.GhBuf(whole.addr + at, whole.bytes - at, 0, F.BUF_ALLOC, 0, 0)})
        at += (size + 15) // 16 * 16
    assert host.call("gh_attention_decode_paged", big, big, kv, 8, 0, 0)[0] == 0


def test_outputs_lie_apart_from_the_handle(host):
    """Attention's out and the append's q_out meet no buffer of the handle, nor positions; no input lies in the scores that
    the call writes, and positions in nothing that it writes."""
    kv = host.kv(scored=True)
    yarn = F.GhYarn(128, 16384, 1e6, 16.0, 32.0, 1.0, 1.0, 0.1)
    n = 3 * 8 * 256
    q, o, k, v, pos = host.buf(n), host.buf(n), host.buf(3 * 2 * 256), host.buf(3 * 2 * 256), host.buf(12)

    def rope(o=o, q=q, k=k, v=v, pos=pos):
        return host.call("gh_rope_kv_write_paged", kv, o, q, k, v, 8, pos, 1, 9, yarn, 0)[0]

    def attend(o=o, q=q):
        return host.call("gh_attention_decode_paged", o, q, kv, 8, 0, 0)[0]

    assert rope() == attend() == 0
    for b in (kv.kv.k, kv.kv.v, kv.table, kv.lengths, kv.score):
        for off in (-(n - 16), 0, (b.bytes - 1) // 16 * 16):
            bad = F.GhBuf(b.addr + off, n, 0, F.BUF_ALLOC, 0, 0)
            assert rope(o=bad) == attend(o=bad) == INVALID
            assert rope(o=bad, q=bad) == attend(o=bad, q=bad) == INVALID  # in place
    s = kv.score
    for off in (0, (s.bytes - 1) // 16 * 16):
        bad = F.GhBuf(s.addr + off, n, 0, F.BUF_ALLOC, 0, 0)
        assert rope(q=bad) == rope(k=bad) == rope(v=bad) == rope(pos=bad) == attend(q=bad) == INVALID
        assert host.call("gh_kv_write_paged", kv, bad, v, 1, 0)[0] == host.call("gh_kv_write_paged", kv, k, bad, 1, 0)[0] == INVALID
    for b in (kv.kv.k, kv.kv.v, o):
        assert rope(pos=F.GhBuf(b.addr + b.bytes - 4, 12, 0, F.BUF_ALLOC, 0, 0)) == INVALID
    assert rope(pos=kv.lengths) == 0
    # vectors may come from slots of the pool that the call does not write
    part = F.GhBuf(kv.kv.k.addr, n, 0, F.BUF_ALLOC, 0, 0)
    assert rope(q=part) == rope(k=part) == rope(v=part) == attend(q=part) == 0


@pytest.fixture
def scratch(host):
    """A host whose scratch stays from call to call: requests() are the sizes that it had to ask for."""
    lib = host.lib
    lib.host_drop_scratch.argtypes = [C.c_void_p]
    lib.host_asked.restype = C.c_uint64
    lib.host_keep_scratch()
    host.requests = lambda: [lib.host_asked(i) for i in range(lib.host_keep_scratch())]
    yield host
    lib.host_drop_scratch(host.b)


@pytest.mark.parametrize("scored", [False, True])
def test_a_growing_length_seldom_asks_for_scratch(scratch, scored):
    """A decode loop that passes its longest length: scratch grows with room to spare, by half."""
    kv = scratch.kv(layers=1, slots=64, heads=8, page=64, width=64, rows=16, scored=scored)
    q = scratch.buf(16 * 64 * 256)
    for length in range(500, 4000):
        assert scratch.call("gh_attention_decode_paged", q, q, kv, 64, length, 0)[0] == 0
    assert len(scratch.requests()) <= 6  # 1.5^6 > 8
    lists = scratch.kv(layers=4, slots=64, heads=8, page=64, width=64, rows=16, scored=True)
    to = with_(lists, table=scratch.buf(lists.table.bytes))
    before = len(scratch.requests())
    for budget in range(2000, 4000, 10):
        assert scratch.call("gh_kv_evict_paged", to, lists, None, budget, 1)[0] == 0
    assert len(scratch.requests()) - before <= 3


def test_scratch_without_room_to_spare_is_what_the_call_needs(scratch):
    kv = scratch.kv(layers=1, slots=64, heads=8, page=64, width=64, rows=4, scored=True)
    q = scratch.buf(4 * 64 * 256)
    assert scratch.call("gh_attention_decode_paged", q, q, kv, 64, 4000, 0)[0] == 0
    with_room = scratch.requests()[0]
    scratch.lib.host_drop_scratch(scratch.b)
    scratch.lib.host_keep_scratch()
    rc, got = scratch.call("gh_attention_decode_paged", q, q, kv, 64, 4000, 0, limit=with_room - 1)
    first, second = scratch.requests()
    assert rc == 0 and len(got) == 2 and first == with_room and second < with_room <= 3 * second // 2 + 1


def rows_of(host, got):
    """Rows of each attention launch."""
    return [AttnArgs.from_buffer_copy(bytes(g.args)).rows for g in got if g.kernel not in (host.ids["join"], host.ids["join2"])]


@pytest.mark.parametrize("scored,heads", [(True, 8), (False, 8), (False, 64)])
def test_scratch_that_could_not_be_had_is_not_asked_for_again(scratch, scored, heads):
    """With memory for some of the rows only the first call looks for how many; later ones take turns in what there
    is, also where a row's share grows, and now and then one looks again."""
    rows = 64
    kv = scratch.kv(layers=1, slots=64, heads=heads, page=64, width=64, rows=rows, scored=scored)
    q = scratch.buf(rows * 8 * heads * 256)

    def call(max_len, limit):
        return scratch.call("gh_attention_decode_paged", q, q, kv, 8 * heads, max_len, 0, limit=limit)

    rc, got = call(500, 0)
    need = scratch.requests()[0] * 2 // 3  # without the room to spare
    scratch.lib.host_drop_scratch(scratch.b)
    scratch.lib.host_keep_scratch()
    limit = need // 3
    rc, got = call(500, limit)
    taken = rows_of(scratch, got)
    assert rc == 0 and sum(taken) == rows and len(taken) > 2
    found = len(scratch.requests())
    assert found > 2
    for length in [500] * 40 + list(range(500, 512)):
        rc, got = call(length, limit)
        assert rc == 0 and sum(rows_of(scratch, got)) == rows and len(rows_of(scratch, got)) <= len(taken)
    assert len(scratch.requests()) == found
    calls = 0
    while len(rows_of(scratch, call(500, 0)[1])) > 1:
        calls += 1
        assert calls < 300
    assert len(scratch.requests()) == found + 1


def test_scratch_for_longer_rows_under_a_limit(scratch):
    kv = scratch.kv(layers=1, slots=64, heads=8, page=64, width=64, rows=16, scored=True)
    q = scratch.buf(16 * 64 * 256)
    limit = 12 << 20  # the chunks take 8.1 MiB of it
    for length in range(600, 2600, 10):
        rc, got = scratch.call("gh_attention_decode_paged", q, q, kv, 64, length, 0, limit=limit)
        assert rc == 0 and sum(rows_of(scratch, got)) == 16
    assert len(scratch.requests()) <= 8
    # a row that fits nowhere is an error each time, and shorter ones go on
    for _ in range(3):
        assert scratch.call("gh_attention_decode_paged", q, q, kv, 64, 4096, 0, limit=1 << 20)[0] in (0, OOM)
        assert scratch.call("gh_attention_decode_paged", q, q, kv, 64, 2600, 0, limit=limit)[0] == 0


class Field(C.Structure):
    _fields_ = [("name", C.c_char_p), ("offset", C.c_uint32), ("size", C.c_uint32)]


@pytest.mark.parametrize("which,mine", [("host_pages_fields", Pages), ("host_attn_fields", AttnArgs)])
def test_argument_structures_are_the_kernels(lib, which, mine):
    """Pages and AttnArgs above have the fields, offsets and sizes of the ones in gh_kargs.h."""
    call = getattr(lib, which)
    call.restype = C.POINTER(Field)
    fields, i = call(), 0
    while fields[i].name:
        name, kind = mine._fields_[i]
        assert fields[i].name.decode() == name
        assert (fields[i].offset, fields[i].size) == (getattr(mine, name).offset, C.sizeof(kind)), name
        i += 1
    assert i == len(mine._fields_) and fields[i].offset == C.sizeof(mine)
