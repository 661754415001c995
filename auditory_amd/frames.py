"""Argument handling shared by the feature-map and frame-sequence operators (norm.py, scan.py): tensors on one device,
channels contiguous, float32 parameters; addresses and strides for the C ABI.  No arithmetic."""
import torch

from . import capi, runtime

DTYPES = {torch.float32: capi.AUD_F32, torch.bfloat16: capi.AUD_BF16, torch.float16: capi.AUD_F16}
ACTS = {"none": capi.AUD_ACT_NONE, "relu": capi.AUD_ACT_RELU, "silu": capi.AUD_ACT_SILU, "gelu": capi.AUD_ACT_GELU}


def bad(msg):
    return capi.AuditoryError(capi.AUD_EINVAL, msg)


def device_of(t, name):
    """the index of the GPU a tensor lives on (there is no CPU path)"""
    if t.device.type != "cuda":
        raise bad("%s must be a tensor on a GPU, it is on %s" % (name, t.device))
    return t.device.index


def stream_of(index):
    """torch's current stream of that GPU: the operators queue their kernels there"""
    return torch.cuda.current_stream(index).cuda_stream


class Call:
    """One call's context, stream and checks: every tensor is on the device of the first one and has the shape and type it
    should have."""

    def __init__(self, x, name, ndim):
        self.index = device_of(x, name)
        self.dtype = DTYPES.get(x.dtype)
        if self.dtype is None:
            raise bad("%s must be float32, bfloat16 or float16, it is %s" % (name, x.dtype))
        if x.dim() != ndim:
            raise bad("%s must have %d axes, it has %d" % (name, ndim, x.dim()))
        self.x, self.device = x, x.device
        self.ctx = runtime.get_ctx(self.index)
        self.lib, self.handle = self.ctx.lib, self.ctx.handle

    def act(self, name, allowed):
        if name not in allowed:
            raise bad("act must be one of %s" % ", ".join(allowed))
        return ACTS[name]

    def rows(self, t, name, shape, tail=1):
        """an activation [items, rows, ...] of x's type whose last `tail` axes are contiguous: its item and row strides"""
        if t.dtype is not self.x.dtype or t.device != self.device or t.shape != shape:
            raise bad("%s must be %s %s on %s" % (name, self.x.dtype, tuple(shape), self.device))
        st, want = t.stride(), 1
        for k in range(1, tail + 1):
            if t.shape[-k] > 1 and st[-k] != want:
                raise bad("the channels of %s must be contiguous" % name)
            want *= t.shape[-k]
        return (st[0] if t.shape[0] > 1 else 0), (st[1] if t.dim() - tail > 1 and t.shape[1] > 1 else want)

    def floats(self, t, name, shape):
        """a float32 parameter, statistic or state, contiguous: its address (0 for None)"""
        if t is None:
            return None
        if t.dtype is not torch.float32 or t.device != self.device or t.shape != shape or not t.is_contiguous():
            raise bad("%s must be contiguous float32 %s on %s" % (name, tuple(shape), self.device))
        return t.data_ptr()

    def same(self, t, name, shape):
        """a contiguous tensor of x's type: its address (0 for None)"""
        if t is None:
            return None
        if t.dtype is not self.x.dtype or t.device != self.device or t.shape != shape or not t.is_contiguous():
            raise bad("%s must be contiguous %s %s on %s" % (name, self.x.dtype, tuple(shape), self.device))
        return t.data_ptr()

    def lengths(self, t, items):
        if t is None:
            return None
        if t.dtype is not torch.int32 or t.device != self.device or t.shape != (items,) or not t.is_contiguous():
            raise bad("lengths must be contiguous int32 [%d] on %s" % (items, self.device))
        return t.data_ptr()

    def out(self, t, name, shape):
        """an output of x's type: the given one, checked, or a new one"""
        if t is None:
            return torch.empty(shape, dtype=self.x.dtype, device=self.device)
        self.same(t, name, shape)
        return t

    def new(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device=self.device)

    def workspace(self, nbytes):
        """(tensor, address) of a call's scratch memory; torch's allocator keeps it for this stream (and, in a capture, for
        this graph) until its kernels have run"""
        if nbytes == 0:
            return None, None
        t = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        return t, t.data_ptr()

    def stream(self):
        return stream_of(self.index)
