"""Operators along the frames of a batch of utterances: the short causal convolution (aud_causal_conv_*, causal_conv.hip) and
the selective state space scan (aud_scan_*, scan.hip), for whole utterances, with gradients, and for one frame at a time
with the state carried between calls.

Device-resident, on torch's current stream; float32, bfloat16 or float16 frames with float32 parameters and scan states."""
import ctypes as C
from collections import namedtuple

import torch

from . import capi, frames

ConvGrads = namedtuple("ConvGrads", "x weight bias state")
ScanGrads = namedtuple("ScanGrads", "u delta A B C D z delta_bias state")

_CONV_ACTS = ("none", "silu")


def _ptr(t):
    return t.data_ptr() if t is not None else None


# ---- causal convolution --------------------------------------------------------------------------------------------------

def _conv_params(call, x, weight, act):
    items, steps, channels = x.shape
    if weight.dim() != 2 or weight.shape[0] != channels or not 1 <= weight.shape[1] <= 4:
        raise frames.bad("weight must be [%d, 1 to 4 taps]" % channels)
    xi, xr = call.rows(x, "x", x.shape)
    return capi.ConvParams(call.dtype, call.act(act, _CONV_ACTS), items, steps, channels, weight.shape[1], xi, xr, 0, 0)


def causal_conv(x, weight, bias=None, act="none", state=None, lengths=None, out=None, state_out=None):
    """y_t = act(bias + sum_k weight[:, k] * x_{t - taps + 1 + k}) of every channel by itself; x [items, steps, channels] with
    contiguous channels, weight [channels, taps], taps 1 to 4.

    state [items, taps - 1, channels]: the inputs in front of x, oldest first (None: zeros).  state_out: a tensor of that shape
    that receives the last taps - 1 inputs of each item -- the state of the next call; it may be `state` itself.  lengths: int32
    [items]; y is zero at and behind an item's length, and its state is counted to there."""
    call = frames.Call(x, "x", 3)
    p = _conv_params(call, x, weight, act)
    kept = (x.shape[0], p.taps - 1, x.shape[2])
    y = call.out(out, "out", x.shape)
    call.ctx.check(call.lib.aud_causal_conv_batch_dev(
        call.handle, C.byref(p), x.data_ptr(), call.floats(weight, "weight", weight.shape), call.floats(bias, "bias", (p.channels,)),
        call.same(state, "state", kept), call.lengths(lengths, p.n_items), y.data_ptr(), call.same(state_out, "state_out", kept),
        call.stream()))
    return y


def causal_conv_step(x, state, weight, bias=None, act="none", out=None, state_out=None):
    """causal_conv of one frame: x [items, channels] -> y [items, channels]; `state` is advanced in place, or into state_out."""
    y = causal_conv(x.unsqueeze(1), weight, bias, act, state, None, None if out is None else out.unsqueeze(1),
                    state if state_out is None else state_out)
    return y.squeeze(1) if out is None else out


def causal_conv_grad(dy, x, weight, bias=None, act="none", state=None, lengths=None, dstate_out=None, out=None):
    """Gradients of causal_conv as ConvGrads(x, weight, bias, state); dstate_out: the gradient of its state_out (None: zero).
    weight's and bias's are float32 sums over the batch; bias's and state's are None where the argument is None."""
    call = frames.Call(x, "x", 3)
    p = _conv_params(call, x, weight, act)
    p.dy_item, p.dy_row = call.rows(dy, "dy", x.shape)
    kept = (x.shape[0], p.taps - 1, x.shape[2])
    dx = call.out(out, "out", x.shape)
    dweight = call.new(*weight.shape)
    dbias = call.new(p.channels) if bias is not None else None
    dstate = call.out(None, "", kept) if state is not None else None
    need = C.c_int64()
    call.ctx.check(call.lib.aud_causal_conv_workspace_bytes(C.byref(p), C.byref(need)))
    ws, ws_ptr = call.workspace(need.value)
    call.ctx.check(call.lib.aud_causal_conv_grad_dev(
        call.handle, C.byref(p), dy.data_ptr(), x.data_ptr(), call.floats(weight, "weight", weight.shape),
        call.floats(bias, "bias", (p.channels,)), call.same(state, "state", kept), call.lengths(lengths, p.n_items),
        call.same(dstate_out, "dstate_out", kept), dx.data_ptr(), dweight.data_ptr(), _ptr(dbias), _ptr(dstate), ws_ptr, need.value,
        call.stream()))
    return ConvGrads(dx, dweight, dbias, dstate)


# ---- selective scan ------------------------------------------------------------------------------------------------------

class _Scan:
    """the checked arguments a scan and its gradients share"""

    def __init__(self, u, delta, A, B, C_, D, z, delta_bias, softplus, state, lengths):
        self.call = call = frames.Call(u, "u", 3)
        items, steps, channels = u.shape
        if A.dim() != 2 or A.shape[0] != channels or not 1 <= A.shape[1] <= 64:
            raise frames.bad("A must be [%d, 1 to 64 states]" % channels)
        if B.dim() != 4:
            raise frames.bad("B must be [items, steps, groups, states]")
        groups, states = B.shape[2], A.shape[1]
        if groups < 1 or channels % groups:
            raise frames.bad("channels (%d) must be a multiple of groups (%d)" % (channels, groups))
        vectors = (items, steps, groups, states)
        self.p = capi.ScanParams(call.dtype, int(bool(softplus)), items, steps, channels, groups, states, 0,
                                 *call.rows(u, "u", u.shape), *call.rows(delta, "delta", u.shape),
                                 *(call.rows(z, "z", u.shape) if z is not None else (0, channels)),
                                 *call.rows(B, "B", vectors, 2), *call.rows(C_, "C", vectors, 2), 0, channels)
        self.kept_state = (items, channels, states)
        self.A = call.floats(A, "A", A.shape)
        self.D = call.floats(D, "D", (channels,))
        self.delta_bias = call.floats(delta_bias, "delta_bias", (channels,))
        self.state = call.floats(state, "state", self.kept_state)
        self.lengths = call.lengths(lengths, items)

    def workspace(self, gradients):
        need = C.c_int64()
        self.call.ctx.check(self.call.lib.aud_scan_workspace_bytes(C.byref(self.p), int(gradients), C.byref(need)))
        return self.call.workspace(need.value) + (need.value,)

    def kept_floats(self):
        n = C.c_int64()
        self.call.ctx.check(self.call.lib.aud_scan_kept_floats(C.byref(self.p), C.byref(n)))
        return n.value


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None, out=None,
                   state_out=None, keep=False):
    """The recurrence h_t = exp(dt A) h_{t-1} + dt B_t u_t with dt = softplus(delta + delta_bias) (softplus=False: the sum
    itself), and y_t = (sum over the states of C_t h_t + D u_t) * silu(z_t) (z=None: no gate), for every channel.

    u, delta, z [items, steps, channels] with contiguous channels; A float32 [channels, states]; B, C [items, steps, groups,
    states], a group serving channels / groups neighbouring channels; D, delta_bias float32 [channels].  state float32 [items,
    channels, states] is the state in front of the first frame (None: zeros); state_out receives the one behind each item's
    last frame and may be `state` itself.  lengths: int32 [items]; behind an item's length y is zero and the state stays.
    keep=True returns (y, kept): the states of every 16th frame, what selective_scan_grad starts from."""
    s = _Scan(u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths)
    call = s.call
    y = call.out(out, "out", u.shape)
    kept = call.new(s.kept_floats()) if keep else None
    ws, ws_ptr, nbytes = s.workspace(False)
    call.ctx.check(call.lib.aud_scan_batch_dev(
        call.handle, _ref(s.p), u.data_ptr(), delta.data_ptr(), s.A, B.data_ptr(), C.data_ptr(), s.D, _ptr(z), s.delta_bias, s.state,
        s.lengths, y.data_ptr(), call.floats(state_out, "state_out", s.kept_state), _ptr(kept), ws_ptr, nbytes, call.stream()))
    return (y, kept) if keep else y


def selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, softplus=False, out=None, state_out=None):
    """selective_scan of one frame: u, delta, z [items, channels], B, C [items, groups, states] -> y [items, channels]; `state`
    is advanced in place, or into state_out."""
    y = selective_scan(u.unsqueeze(1), delta.unsqueeze(1), A, B.unsqueeze(1), C.unsqueeze(1), D, None if z is None else z.unsqueeze(1),
                       delta_bias, softplus, state, None, None if out is None else out.unsqueeze(1),
                       state if state_out is None else state_out)
    return y.squeeze(1) if out is None else out


def selective_scan_grad(dy, u, delta, A, B, C, kept, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None,
                        dstate_out=None):
    """Gradients of selective_scan as ScanGrads(u, delta, A, B, C, D, z, delta_bias, state), from the `kept` of the same call;
    dstate_out: the gradient of its state_out (None: zero).  A's, D's, delta_bias's and the state's are float32, the others of
    u's type; None where the argument is None."""
    s = _Scan(u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths)
    call = s.call
    s.p.dy_item, s.p.dy_row = call.rows(dy, "dy", u.shape)
    du, ddelta = torch.empty(u.shape, dtype=u.dtype, device=u.device), torch.empty(u.shape, dtype=u.dtype, device=u.device)
    dz = torch.empty(u.shape, dtype=u.dtype, device=u.device) if z is not None else None
    dB, dC = torch.empty(B.shape, dtype=u.dtype, device=u.device), torch.empty(B.shape, dtype=u.dtype, device=u.device)
    dA = call.new(*A.shape)
    dD = call.new(s.p.channels) if D is not None else None
    dbias = call.new(s.p.channels) if delta_bias is not None else None
    dstate = call.new(*s.kept_state) if state is not None else None
    ws, ws_ptr, nbytes = s.workspace(True)
    call.ctx.check(call.lib.aud_scan_grad_dev(
        call.handle, _ref(s.p), dy.data_ptr(), u.data_ptr(), delta.data_ptr(), s.A, B.data_ptr(), C.data_ptr(), s.D, _ptr(z),
        s.delta_bias, s.lengths, call.floats(kept, "kept", (s.kept_floats(),)), call.floats(dstate_out, "dstate_out", s.kept_state),
        du.data_ptr(), ddelta.data_ptr(), dA.data_ptr(), dB.data_ptr(), dC.data_ptr(), _ptr(dD), _ptr(dz), _ptr(dbias), _ptr(dstate),
        ws_ptr, nbytes, call.stream()))
    return ScanGrads(du, ddelta, dA, dB, dC, dD, dz, dbias, dstate)


_ref = C.byref
