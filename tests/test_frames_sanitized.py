"""The feature-map and frame-sequence operators on the sanitizer builds of the CPU thread emulator: accesses past a buffer or past
the LDS that a launch asked for, arithmetic without meaning, threads that race."""
from test_emul_parity import _sanitizer_run


def test_emul_frames_under_asan_ubsan():
    _sanitizer_run("asan", "frames")


def test_emul_frames_under_tsan():
    _sanitizer_run("tsan", "frames")
