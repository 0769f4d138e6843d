"""gh_sample_rows and its kernels, compiled for the CPU (tests/wave_host), against the definition in 64 bits: with the waves of a
workgroup in any order between its barriers."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import flat_tail
from graph_horizon_amd import _ffi as F
from sampled import sample

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PARAMS = np.dtype([("temperature", "<f4"), ("top_p", "<f4"), ("top_k", "<u4"), ("min_p", "<f4")])


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = tmp_path_factory.mktemp("sample")
    here = os.path.join(ROOT, "tests", "wave_host")
    clang = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "clang++")
    subprocess.run([clang, "-x", "c++", "-O1", "-std=c++17", "-fPIC", "-Wall", "-Werror", "-I", here, "-c", os.path.join(here, "sample_kernels.cpp"),
                    "-o", str(out / "kernels.o")], check=True)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-Wall", "-Werror",
                    "-o", str(out / "sample.so"), os.path.join(here, "sample_plan.cpp"),
                    os.path.join(ROOT, "graph_horizon_amd", "csrc", "host", "rows.cpp"), str(out / "kernels.o")], check=True)
    h = C.CDLL(str(out / "sample.so"))
    h.gh_sample_rows.argtypes = F.SIGNATURES["gh_sample_rows"][1]
    h.wave_backend.restype = h.wave_encoder.restype = C.c_void_p
    h.wave_encoder.argtypes = h.wave_error.argtypes = [C.c_void_p]
    h.wave_limit.argtypes = [C.c_uint64]
    h.wave_error.restype = C.c_char_p
    h.backend = h.wave_backend(256)
    return h


def run(lib, logits, params, u, order=0, backend=None):
    rows, vocab = logits.shape
    logits = np.ascontiguousarray(logits)
    params, u = np.array(params, PARAMS), np.asarray(u, np.float32)
    room = np.zeros(4 * rows + 4, np.float32)  # the parameters lie on 16 bytes
    off = -room.ctypes.data % 16 // 4
    room[off:off + 4 * rows].view(PARAMS)[:] = params
    tokens, probs = np.full(rows, 77, np.uint32), np.full(rows, 77, np.float32)
    bufs = [F.GhBuf(x.ctypes.data, x.nbytes) for x in (tokens, probs, logits, room[off:off + 4 * rows], u)]
    lib.wave_order(order)
    backend = backend or lib.backend
    rc = lib.gh_sample_rows(backend, lib.wave_encoder(backend), C.byref(bufs[0]), C.byref(bufs[1]), C.byref(bufs[2]), rows, vocab,
                            vocab, C.byref(bufs[3]), C.byref(bufs[4]))
    assert rc == 0, lib.wave_error(backend)
    return tokens, probs


def check(lib, logits, params, u, order=0):
    tokens, probs = run(lib, logits, params, u, order)
    for r in range(len(logits)):
        t, p, k, m = params[r]
        want, prob, near = sample(logits[r], t, p, k, m, u[r])
        assert near > 1e-11 and tokens[r] == want, (r, params[r], u[r], near)
        assert abs(probs[r] - prob) <= 2.0 ** -24 * prob + 2.0 ** -36, (r, params[r])


@pytest.mark.parametrize("order", range(6))
@pytest.mark.parametrize("params", [(1.0, 1.0, 0, 0.0), (1.0, 0.6, 0, 0.0), (0.8, 0.9, 700, 0.0), (1.0, 1.0, 0, 0.2), (0.9, 0.8, 900, 0.05)])
def test_waves_in_any_order(lib, order, params):
    """Rows whose searches end in bins of more than 64 tokens, in the list and in the row itself."""
    rng = np.random.default_rng(5)
    for vocab, spread in ((3000, 2.0), (3000, 0.0005), (9000, 0.0005)):
        logits = (7 + spread * rng.standard_normal((2, vocab))).astype(np.float32)
        check(lib, logits, [params] * 2, rng.random(2).astype(np.float32), order)


@pytest.mark.parametrize("vocab,distance", [(50000, 24.0), ((1 << 17) + 1, 23.5)])
def test_a_flat_far_tail_keeps_its_mass(lib, vocab, distance):
    """What many tiny weights sum up to, next to one of 1: the tail's share is 1e-5 or less and drawn from as such."""
    def by_row(logits, want, us):
        got = [run(lib, logits[i % len(us)][None], [c[0]], [c[1]], order=1) for i, c in enumerate(want)]
        return [int(t[0]) for t, _ in got], [float(p[0]) for _, p in got]
    flat_tail.check(by_row, vocab, distance)


def test_short_of_memory_it_is_not_asked_for_at_every_call(lib):
    """Scratch for three rows of ten, and no more to be had: later calls take turns in it at once."""
    rng = np.random.default_rng(6)
    logits, params, u = rng.standard_normal((10, 50)).astype(np.float32), [(1.0, 0.9, 0, 0.0)] * 10, rng.random(10).astype(np.float32)
    want = run(lib, logits, params, u)
    backend = lib.wave_backend(256)
    lib.wave_limit(3 * 79000)
    asked = []
    for _ in range(4):
        got = run(lib, logits, params, u, backend=backend)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        asked.append(lib.wave_limit(3 * 79000))
    assert asked[0] > 1 and asked[1:] == [0, 0, 0], asked
    lib.wave_limit(0)  # memory is there again: asked for in the 256th call that did with less at the latest
    for _ in range(260):
        run(lib, logits, params, u, order=0xFFFFFFFF, backend=backend)
    assert lib.wave_limit(0) >= 1
