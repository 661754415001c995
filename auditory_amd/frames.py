"""What the feature-map and frame-sequence operators (norm.py, scan.py) share on the host: checks of their tensors, and plans.

A plan is what a call works out from the LAYOUT of its arguments alone -- types, shapes, strides, options: the parameter block
of the C ABI, checked, and the size of the workspace.  Plans are kept per layout, so a call of a kind that was made before goes
straight to the library; addresses and values are never kept."""
import ctypes as C

import torch

from . import capi, runtime

F32, I32 = torch.float32, torch.int32
DTYPES = {torch.float32: capi.AUD_F32, torch.bfloat16: capi.AUD_BF16, torch.float16: capi.AUD_F16}
ACTS = {"none": capi.AUD_ACT_NONE, "relu": capi.AUD_ACT_RELU, "silu": capi.AUD_ACT_SILU, "gelu": capi.AUD_ACT_GELU}
MAX_PLANS = 512


def bad(msg):
    return capi.AuditoryError(capi.AUD_EINVAL, msg)


def context(x, name):
    """the library's context of the GPU a tensor lives on (there is no CPU path)"""
    index = x.get_device()
    if index < 0:
        raise bad("%s must be a tensor on a GPU, it is on %s" % (name, x.device))
    if index not in runtime._CTX:
        with torch.cuda.device(index):  # (making a context makes its device current)
            return runtime.get_ctx(index)
    return runtime._CTX[index]


def current_stream(index):
    """torch's current stream of a GPU: the operators queue their kernels there"""
    return torch.cuda.current_stream(index).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):  # the same without a Stream object around it
    current_stream = torch._C._cuda_getCurrentRawStream  # noqa: F811


class Plans(dict):
    """plans by layout"""

    def keep(self, key, plan):
        if len(self) >= MAX_PLANS:
            self.clear()
        self[key] = plan
        return plan


def dtype_of(x, name, ndim):
    code = DTYPES.get(x.dtype)
    if code is None:
        raise bad("%s must be float32, bfloat16 or float16, it is %s" % (name, x.dtype))
    if x.dim() != ndim:
        raise bad("%s must have %d axes, it has %d" % (name, ndim, x.dim()))
    return code


def act_of(name, allowed):
    if name not in allowed:
        raise bad("act must be one of %s" % ", ".join(allowed))
    return ACTS[name]


def strides(shape, stride, name, tail=1):
    """item and row stride of an activation [items, rows, ...] whose last `tail` axes must be contiguous"""
    want = 1
    for k in range(1, tail + 1):
        if shape[-k] > 1 and stride[-k] != want:
            raise bad("the channels of %s must be contiguous" % name)
        want *= shape[-k]
    rows = shape[1] if len(shape) - tail > 1 else 1
    return (stride[0] if shape[0] > 1 else 0), (stride[1] if rows > 1 else want)


def like(t, x, name, shape, device):
    """t has x's type and the shape, on x's GPU"""
    if t.dtype is not x.dtype or t.shape != shape or t.get_device() != device:
        raise bad("%s must be %s %s on %s" % (name, x.dtype, tuple(shape), x.device))


def dense(t, x, name, shape, device):
    """the address of a contiguous tensor of x's type (None for None)"""
    if t is None:
        return None
    if t.dtype is not x.dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise bad("%s must be contiguous %s %s on %s" % (name, x.dtype, tuple(shape), x.device))
    return t.data_ptr()


def floats(t, x, name, shape, device):
    """the address of a float32 parameter, statistic or state (None for None)"""
    if t is None:
        return None
    if t.dtype is not F32 or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise bad("%s must be contiguous float32 %s on %s" % (name, tuple(shape), x.device))
    return t.data_ptr()


def lengths_of(t, x, items, device):
    if t is None:
        return None
    if t.dtype is not I32 or t.shape != (items,) or t.get_device() != device or not t.is_contiguous():
        raise bad("lengths must be contiguous int32 [%d] on %s" % (items, x.device))
    return t.data_ptr()


def size_of(ctx, fn, *args):
    """a size the library works out: fn(*args, &size)"""
    n = C.c_int64()
    if fn(*args, C.byref(n)) != capi.AUD_OK:
        return None  # the call itself says what is wrong
    return n.value


def scratch(nbytes, x):
    """a call's workspace, or None; torch's allocator keeps it for this stream (and, in a capture, for this graph) until its
    kernels have run"""
    return torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
