"""Operators along the frames of a batch of utterances: the short causal convolution (aud_causal_conv_*, causal_conv.hip) and
the selective state space scan (aud_scan_*, scan.hip), for whole utterances, with gradients, and for one frame at a time
with the state carried between calls.

Device-resident, on torch's current stream; float32, bfloat16 or float16 frames with float32 parameters and scan states."""
import ctypes
from collections import namedtuple

import torch

from . import capi, frames

ConvGrads = namedtuple("ConvGrads", "x weight bias state")
ScanGrads = namedtuple("ScanGrads", "u delta A B C D z delta_bias state")

_CONV_ACTS = ("none", "silu")
_CONV_PLANS, _SCAN_PLANS = frames.Plans(), frames.Plans()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _new_like(x):
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _out(out, x, dev):
    if out is None:
        return _new_like(x)
    frames.dense(out, x, "out", x.shape, dev)
    return out


def _new(shape, x):
    return torch.empty(shape, dtype=frames.F32, device=x.device)


# ---- causal convolution --------------------------------------------------------------------------------------------------
# (a frame alone is [items, channels]: the same layout with one step)

class _ConvPlan:
    def __init__(self, x, weight_shape, act, dy_stride):
        code = frames.dtype_of(x, "x", x.dim() if x.dim() in (2, 3) else 3)
        self.ctx = ctx = frames.context(x, "x")
        items, channels = x.shape[0], x.shape[-1]
        steps = x.shape[1] if x.dim() == 3 else 1
        if len(weight_shape) != 2 or weight_shape[0] != channels or not 1 <= weight_shape[1] <= 4:
            raise frames.bad("weight must be [%d, 1 to 4 taps]" % channels)
        xi, xr = frames.strides(x.shape, x.stride(), "x")
        di, dr = frames.strides(x.shape, dy_stride, "dy") if dy_stride else (0, 0)
        self.p = capi.ConvParams(code, frames.act_of(act, _CONV_ACTS), items, steps, channels, weight_shape[1], xi, xr, di, dr)
        self.ref = ctypes.byref(self.p)
        self.nbytes = 0
        if dy_stride is not None:
            self.nbytes = frames.size_of(ctx, ctx.lib.aud_causal_conv_workspace_bytes, self.ref) or 0
        self.items, self.per_channel, self.weight, self.state = items, (channels,), tuple(weight_shape), (items, weight_shape[1] - 1, channels)


def _conv_plan(x, weight, act, dy_stride=None):
    key = (x.dtype, x.shape, x.stride(), x.get_device(), weight.shape, act, dy_stride)
    return _CONV_PLANS.get(key) or _CONV_PLANS.keep(key, _ConvPlan(x, weight.shape, act, dy_stride))


def _conv(x, weight, bias, act, state, lengths, out, state_out):
    plan = _conv_plan(x, weight, act)
    ctx, dev, kept = plan.ctx, x.get_device(), plan.state
    y = _out(out, x, dev)
    rc = ctx.lib.aud_causal_conv_batch_dev(
        ctx.handle, plan.ref, x.data_ptr(), frames.floats(weight, x, "weight", plan.weight, dev),
        frames.floats(bias, x, "bias", plan.per_channel, dev), frames.dense(state, x, "state", kept, dev),
        frames.lengths_of(lengths, x, plan.items, dev), y.data_ptr(), frames.dense(state_out, x, "state_out", kept, dev),
        frames.current_stream(dev))
    if rc:
        ctx.check(rc)
    return y


def causal_conv(x, weight, bias=None, act="none", state=None, lengths=None, out=None, state_out=None):
    """y_t = act(bias + sum_k weight[:, k] * x_{t - taps + 1 + k}) of every channel by itself; x [items, steps, channels] with
    contiguous channels, weight [channels, taps], taps 1 to 4.

    state [items, taps - 1, channels]: the inputs in front of x, oldest first (None: zeros).  state_out: a tensor of that shape
    that receives the last taps - 1 inputs of each item -- the state of the next call; it may be `state` itself.  lengths: int32
    [items]; y is zero at and behind an item's length, and its state is counted to there."""
    if x.dim() != 3:
        raise frames.bad("x must have 3 axes, it has %d" % x.dim())
    return _conv(x, weight, bias, act, state, lengths, out, state_out)


def causal_conv_step(x, state, weight, bias=None, act="none", out=None, state_out=None):
    """causal_conv of one frame: x [items, channels] -> y [items, channels]; `state` is advanced in place, or into state_out."""
    if x.dim() != 2:
        raise frames.bad("x must have 2 axes, it has %d" % x.dim())
    return _conv(x, weight, bias, act, state, None, out, state if state_out is None else state_out)


def causal_conv_grad(dy, x, weight, bias=None, act="none", state=None, lengths=None, dstate_out=None, out=None):
    """Gradients of causal_conv as ConvGrads(x, weight, bias, state); dstate_out: the gradient of its state_out (None: zero).
    weight's and bias's are float32 sums over the batch; bias's and state's are None where the argument is None."""
    if x.dim() != 3:
        raise frames.bad("x must have 3 axes, it has %d" % x.dim())
    plan = _conv_plan(x, weight, act, dy.stride())
    ctx, dev, kept = plan.ctx, x.get_device(), plan.state
    frames.like(dy, x, "dy", x.shape, dev)
    dx, dweight = _out(out, x, dev), _new(plan.weight, x)
    dbias = _new(plan.per_channel, x) if bias is not None else None
    dstate = torch.empty(kept, dtype=x.dtype, device=x.device) if state is not None else None
    ws = frames.scratch(plan.nbytes, x)
    rc = ctx.lib.aud_causal_conv_grad_dev(
        ctx.handle, plan.ref, dy.data_ptr(), x.data_ptr(), frames.floats(weight, x, "weight", plan.weight, dev),
        frames.floats(bias, x, "bias", plan.per_channel, dev), frames.dense(state, x, "state", kept, dev),
        frames.lengths_of(lengths, x, plan.items, dev), frames.dense(dstate_out, x, "dstate_out", kept, dev), dx.data_ptr(),
        dweight.data_ptr(), _ptr(dbias), _ptr(dstate), _ptr(ws), plan.nbytes, frames.current_stream(dev))
    if rc:
        ctx.check(rc)
    return ConvGrads(dx, dweight, dbias, dstate)


# ---- selective scan ------------------------------------------------------------------------------------------------------

class _ScanPlan:
    """dims 3: u [items, steps, channels], B [items, steps, groups, states]; dims 2: one frame, without the axis of steps"""

    def __init__(self, dims, u, delta, A, B, C, z, softplus, dy_stride):
        code = frames.dtype_of(u, "u", dims)
        self.ctx = ctx = frames.context(u, "u")
        items, channels = u.shape[0], u.shape[-1]
        steps = u.shape[1] if dims == 3 else 1
        if A.dim() != 2 or A.shape[0] != channels or not 1 <= A.shape[1] <= 64:
            raise frames.bad("A must be [%d, 1 to 64 states]" % channels)
        if B.dim() != dims + 1:
            raise frames.bad("B must be [items, %sgroups, states]" % ("steps, " if dims == 3 else ""))
        groups, states = B.shape[-2], A.shape[1]
        if groups < 1 or channels % groups:
            raise frames.bad("channels (%d) must be a multiple of groups (%d)" % (channels, groups))
        dev = u.get_device()
        self.vectors = u.shape[:-1] + (groups, states)
        frames.like(delta, u, "delta", u.shape, dev)
        frames.like(B, u, "B", self.vectors, dev)
        frames.like(C, u, "C", self.vectors, dev)
        if z is not None:
            frames.like(z, u, "z", u.shape, dev)
        one = lambda t, name, tail=1: frames.strides(t.shape, t.stride(), name, tail)  # noqa: E731
        dy = frames.strides(u.shape, dy_stride, "dy") if dy_stride else (0, channels)
        self.p = capi.ScanParams(code, int(bool(softplus)), items, steps, channels, groups, states, 0, *one(u, "u"), *one(delta, "delta"),
                                 *(one(z, "z") if z is not None else (0, channels)), *one(B, "B", 2), *one(C, "C", 2), *dy)
        self.ref = ctypes.byref(self.p)
        self.nbytes = frames.size_of(ctx, ctx.lib.aud_scan_workspace_bytes, self.ref, int(dy_stride is not None)) or 0
        self.kept = (frames.size_of(ctx, ctx.lib.aud_scan_kept_floats, self.ref) or 0,)
        self.items, self.per_channel, self.A, self.state = items, (channels,), (channels, states), (items, channels, states)


def _scan_plan(dims, u, delta, A, B, C, z, softplus, dy_stride=None):
    gate = z is not None
    key = (dims, u.dtype, u.shape, u.stride(), u.get_device(), delta.dtype, delta.shape, delta.stride(), delta.get_device(), A.shape,
           B.dtype, B.shape, B.stride(), B.get_device(), C.dtype, C.shape, C.stride(), C.get_device(),
           z.dtype if gate else None, z.shape if gate else None, z.stride() if gate else None, z.get_device() if gate else None,
           softplus, dy_stride)
    return _SCAN_PLANS.get(key) or _SCAN_PLANS.keep(key, _ScanPlan(dims, u, delta, A, B, C, z, softplus, dy_stride))


def _scan(dims, u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths, out, state_out, keep):
    plan = _scan_plan(dims, u, delta, A, B, C, z, softplus)
    ctx, dev, ch = plan.ctx, u.get_device(), plan.per_channel
    y = _out(out, u, dev)
    kept = _new(plan.kept, u) if keep else None
    ws = frames.scratch(plan.nbytes, u)
    rc = ctx.lib.aud_scan_batch_dev(
        ctx.handle, plan.ref, u.data_ptr(), delta.data_ptr(), frames.floats(A, u, "A", plan.A, dev), B.data_ptr(), C.data_ptr(),
        frames.floats(D, u, "D", ch, dev), z.data_ptr() if z is not None else None, frames.floats(delta_bias, u, "delta_bias", ch, dev),
        frames.floats(state, u, "state", plan.state, dev), frames.lengths_of(lengths, u, plan.items, dev), y.data_ptr(),
        frames.floats(state_out, u, "state_out", plan.state, dev), _ptr(kept), _ptr(ws), plan.nbytes, frames.current_stream(dev))
    if rc:
        ctx.check(rc)
    return (y, kept) if keep else y


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None, out=None,
                   state_out=None, keep=False):
    """The recurrence h_t = exp(dt A) h_{t-1} + dt B_t u_t with dt = softplus(delta + delta_bias) (softplus=False: the sum
    itself), and y_t = (sum over the states of C_t h_t + D u_t) * silu(z_t) (z=None: no gate), for every channel.

    u, delta, z [items, steps, channels] with contiguous channels; A float32 [channels, states]; B, C [items, steps, groups,
    states], a group serving channels / groups neighbouring channels; D, delta_bias float32 [channels].  state float32 [items,
    channels, states] is the state in front of the first frame (None: zeros); state_out receives the one behind each item's
    last frame and may be `state` itself.  lengths: int32 [items]; behind an item's length y is zero and the state stays.
    keep=True returns (y, kept): the states of every 16th frame, what selective_scan_grad starts from."""
    return _scan(3, u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths, out, state_out, keep)


def selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, softplus=False, out=None, state_out=None):
    """selective_scan of one frame: u, delta, z [items, channels], B, C [items, groups, states] -> y [items, channels]; `state`
    is advanced in place, or into state_out."""
    return _scan(2, u, delta, A, B, C, D, z, delta_bias, softplus, state, None, out, state if state_out is None else state_out, False)


def selective_scan_grad(dy, u, delta, A, B, C, kept, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None,
                        dstate_out=None):
    """Gradients of selective_scan as ScanGrads(u, delta, A, B, C, D, z, delta_bias, state), from the `kept` of the same call;
    dstate_out: the gradient of its state_out (None: zero).  A's, D's, delta_bias's and the state's are float32, the others of
    u's type; None where the argument is None."""
    plan = _scan_plan(3, u, delta, A, B, C, z, softplus, dy.stride())
    ctx, dev, ch = plan.ctx, u.get_device(), plan.per_channel
    frames.like(dy, u, "dy", u.shape, dev)
    if kept is None:
        raise frames.bad("kept of the forward call is needed")
    frames.floats(state, u, "state", plan.state, dev)
    du, ddelta, dz = _new_like(u), _new_like(u), _new_like(u) if z is not None else None
    dB, dC = torch.empty(plan.vectors, dtype=u.dtype, device=u.device), torch.empty(plan.vectors, dtype=u.dtype, device=u.device)
    dA, dD = _new(plan.A, u), _new(ch, u) if D is not None else None
    dbias = _new(ch, u) if delta_bias is not None else None
    dstate = _new(plan.state, u) if state is not None else None
    ws = frames.scratch(plan.nbytes, u)
    rc = ctx.lib.aud_scan_grad_dev(
        ctx.handle, plan.ref, dy.data_ptr(), u.data_ptr(), delta.data_ptr(), frames.floats(A, u, "A", plan.A, dev), B.data_ptr(),
        C.data_ptr(), frames.floats(D, u, "D", ch, dev), _ptr(z), frames.floats(delta_bias, u, "delta_bias", ch, dev),
        frames.lengths_of(lengths, u, plan.items, dev), frames.floats(kept, u, "kept", plan.kept, dev),
        frames.floats(dstate_out, u, "dstate_out", plan.state, dev), du.data_ptr(), ddelta.data_ptr(), dA.data_ptr(), dB.data_ptr(),
        dC.data_ptr(), _ptr(dD), _ptr(dz), _ptr(dbias), _ptr(dstate), _ptr(ws), plan.nbytes, frames.current_stream(dev))
    if rc:
        ctx.check(rc)
    return ScanGrads(du, ddelta, dA, dB, dC, dD, dz, dbias, dstate)
