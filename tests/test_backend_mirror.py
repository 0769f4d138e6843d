"""The Python mirror's encoders, without a device: a stand-in library with the entry points' argument types."""
import ctypes as C

import pytest

from graph_horizon_amd import GhKvPaged, HipBackend
from graph_horizon_amd import _ffi as F


class Library:
    """Encoders as the native library keeps them, and what was called."""

    def __init__(self):
        self.open, self.calls = False, []

        def begin(h, slot):
            if self.open:
                return -7
            self.open = True
            slot[0] = 42
            return 0

        def submit(h, enc):
            if not self.open:
                return -7
            self.open = False
            return 0

        self.keep = []
        self.bind("gh_begin", begin)
        self.bind("gh_submit", submit)
        for name in ("gh_attention_decode_paged", "gh_kv_write_paged", "gh_rope_kv_write_paged", "gh_kv_evict_paged",
                     "gh_attention_prefill"):
            self.bind(name, lambda *a: 0 if self.open else -7)
        self.gh_last_error = lambda h: b""

    def bind(self, name, body):
        res, args = F.SIGNATURES[name]

        def called(*a):
            self.calls.append(name)
            return body(*a)

        self.keep.append(C.CFUNCTYPE(res, *args)(called))
        setattr(self, name, self.keep[-1])


@pytest.fixture
def hip():
    b = HipBackend.__new__(HipBackend)
    b.lib, b.h, b.enc = Library(), C.c_void_p(1), None
    b._slot = C.c_void_p()
    b._slot_ref = C.pointer(b._slot)
    yield b
    b.h = None


def wrong_calls(hip):
    buf, kv = F.GhBuf(), GhKvPaged()
    yield lambda: hip.attention_decode_paged(buf, buf, F.GhKv(), 8, 0, 0)
    yield lambda: hip.attention_decode_paged(buf, buf, kv, 8, None, 0)
    yield lambda: hip.kv_write_paged(kv, buf, "k", 1, 0)
    yield lambda: hip.kv_evict_paged(kv, kv, None, 1.5, 0)
    yield lambda: hip.attention_prefill(buf, buf, F.GhKv(), 8, "0", 4, 0)


def test_arguments_of_a_wrong_type_leave_no_encoder_open(hip):
    for call in wrong_calls(hip):
        with pytest.raises(C.ArgumentError):
            call()
        assert hip.enc is None and not hip.lib.open
        hip.attention_decode_paged(F.GhBuf(), F.GhBuf(), GhKvPaged(), 8, 0, 0)
        assert hip.lib.calls[-1] == "gh_submit"


def test_arguments_of_a_wrong_type_leave_the_callers_encoder_alone(hip):
    hip.begin()
    for call in wrong_calls(hip):
        with pytest.raises(C.ArgumentError):
            call()
        assert hip.enc is not None and hip.lib.open
    hip.submit()
    assert hip.lib.calls == ["gh_begin", "gh_submit"]
