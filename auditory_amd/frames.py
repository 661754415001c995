"""What the feature-map and frame-sequence operators (norm.py, scan.py) share on the host: the native module that checks their
tensors and calls the library (csrc/frames_torch.cpp), and the library's context of the GPU a tensor lives on."""
import ctypes as C

import torch

from . import capi, runtime

ACTS = {"none": capi.AUD_ACT_NONE, "relu": capi.AUD_ACT_RELU, "silu": capi.AUD_ACT_SILU, "gelu": capi.AUD_ACT_GELU}
_NATIVE = None


def bad(msg):
    return capi.AuditoryError(capi.AUD_EINVAL, msg)


def bind(module, lib, on_gpu):
    """point the native module at a loaded library's entry points (on_gpu False: the CPU thread emulator of the tests)"""
    module.bind({name: C.cast(getattr(lib, name), C.c_void_p).value for name in capi.SYMBOLS}, on_gpu)


def native():
    """the native module, bound to libauditory_hip.so; raises if it is not built (there is no other path)"""
    global _NATIVE
    if _NATIVE is None:
        try:
            from . import _frames
        except ImportError as e:
            raise ImportError("auditory_amd._frames is not built or does not load (%s): run `python -m auditory_amd.build`" % e)
        bind(_frames, capi.load(), True)
        _NATIVE = _frames
    return _NATIVE


def context(x, name):
    """the address of the library's context of a tensor's GPU; made on the first call there (not inside a stream capture)"""
    ctx = runtime._CTX.get(x.get_device())
    if ctx is None or not ctx.handle:
        if not x.is_cuda:
            raise bad("%s must be a tensor on a GPU, it is on %s" % (name, x.device))
        with torch.cuda.device(x.device):  # (making a context makes its device current)
            runtime._CTX.pop(x.get_device(), None)
            ctx = runtime.get_ctx(x.get_device())
    return ctx.handle.value


def act_of(name, allowed):
    if name not in allowed:
        raise bad("act must be one of %s" % ", ".join(allowed))
    return ACTS[name]
