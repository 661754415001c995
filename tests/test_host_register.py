"""aud_host_register where the runtime fails (emulator build): only the refusal to register memory that exists already is a range
that is noted; every other failure is the caller's to know."""
import ctypes as C
import mmap
import os
import sys

import numpy as np
import pytest

from auditory_amd import capi, runtime

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emul"))

INVALID_VALUE, OUT_OF_MEMORY, ALREADY_REGISTERED = 1, 2, 712


@pytest.fixture
def emu():
    import backend
    with backend.emulated("plain") as lib:
        status = C.c_int.in_dll(lib, "aud_emul_host_register_status")
        yield lib, status
        status.value = 0


def test_a_runtime_that_refuses_existing_memory(emu):
    lib, status = emu
    ctx = runtime.get_ctx(0)
    a = np.zeros(3000)
    status.value = INVALID_VALUE
    ctx.register_host(a)
    with pytest.raises(capi.AuditoryError):
        ctx.register_host(a[5:])                 # it is noted: the overlap is found
    ctx.unregister_host(a)
    with pytest.raises(capi.AuditoryError):
        ctx.unregister_host(a)


@pytest.mark.parametrize("code", [OUT_OF_MEMORY, ALREADY_REGISTERED])
def test_other_failures_are_errors(emu, code):
    lib, status = emu
    ctx = runtime.get_ctx(0)
    a = np.zeros(3000)
    status.value = code
    with pytest.raises(capi.AuditoryError) as e:
        ctx.register_host(a)
    assert e.value.status == capi.AUD_EHIP
    with pytest.raises(capi.AuditoryError):
        ctx.unregister_host(a)                   # nothing was noted
    status.value = 0
    ctx.register_host(a)
    ctx.unregister_host(a)


def test_ranges_that_are_not_there_or_not_writable(emu):
    lib, status = emu
    ctx = runtime.get_ctx(0)
    status.value = INVALID_VALUE
    page = mmap.PAGESIZE
    register = lambda p, n: lib.aud_host_register(ctx.handle, C.c_void_p(p), n)  # noqa: E731
    assert register(page, page) == capi.AUD_EHIP                 # nothing is mapped at so low an address
    two = mmap.mmap(-1, 2 * page)
    at = C.addressof(C.c_char.from_buffer(two))
    libc = C.CDLL(None, use_errno=True)
    assert libc.mprotect(C.c_void_p(at + page), C.c_size_t(page), mmap.PROT_READ) == 0
    assert register(at, 2 * page) == capi.AUD_EHIP               # its second half cannot be written
    assert register(at + page, page) == capi.AUD_EHIP
    assert register(at, page) == capi.AUD_OK
    assert lib.aud_host_unregister(ctx.handle, C.c_void_p(at)) == capi.AUD_OK
    assert libc.mprotect(C.c_void_p(at + page), C.c_size_t(page), mmap.PROT_READ | mmap.PROT_WRITE) == 0
    assert register(at, 2 * page) == capi.AUD_OK
    assert lib.aud_host_unregister(ctx.handle, C.c_void_p(at)) == capi.AUD_OK
