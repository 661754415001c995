"""Group norm with an activation, the causal convolution and the selective scan (auditory_amd.norm, auditory_amd.scan) against
their definitions in 64 bits: on the CPU thread emulator (kernel sources compiled unchanged) and on the GPU."""
import ctypes as C
import os
import sys

import pytest
import torch

import frame_cases as F
from auditory_amd import capi, frames, norm, runtime, scan

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emul"))

gpu = pytest.mark.gpu


def ids(cases):
    return ["-".join(str(v) for v in c) for c in cases]


@pytest.fixture(scope="module")
def emu_lib():
    import backend
    with backend.emulated("plain") as lib:
        yield lib


@pytest.fixture
def emu(emu_lib, monkeypatch):
    """the operators on CPU tensors, their kernels run by the thread emulator"""
    monkeypatch.setattr(frames, "context", lambda x, name: runtime.get_ctx(0))
    monkeypatch.setattr(frames, "current_stream", lambda index: None)
    yield emu_lib
    for plans in (norm._PLANS, scan._CONV_PLANS, scan._SCAN_PLANS):  # (they hold the emulator's context)
        plans.clear()


# ---- values and gradients ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("case", F.NORM, ids=ids(F.NORM))
def test_emul_norm(emu, case):
    F.norm_case("cpu", *case)


@pytest.mark.parametrize("case", F.CONV, ids=ids(F.CONV))
def test_emul_conv(emu, case):
    F.conv_case("cpu", *case)


@pytest.mark.parametrize("case", F.SCAN, ids=ids(F.SCAN))
def test_emul_scan(emu, case):
    F.scan_case("cpu", *case)


@gpu
@pytest.mark.parametrize("case", F.NORM, ids=ids(F.NORM))
def test_gpu_norm(case):
    F.norm_case("cuda:0", *case)


@gpu
@pytest.mark.parametrize("case", F.CONV, ids=ids(F.CONV))
def test_gpu_conv(case):
    F.conv_case("cuda:0", *case)


@gpu
@pytest.mark.parametrize("case", F.SCAN, ids=ids(F.SCAN))
def test_gpu_scan(case):
    F.scan_case("cuda:0", *case)
