"""Operators along the frames of a batch of utterances: the short causal convolution (aud_causal_conv_*, causal_conv.hip) and
the selective state space scan (aud_scan_*, scan.hip), for whole utterances, with gradients, and for one frame at a time
with the state carried between calls.

Device-resident, on torch's current stream; float32, bfloat16 or float16 frames with float32 parameters and scan states.  The
gradients are functions of their own: nothing here records for torch's autograd, so a tensor that requires grad is refused
while autograd records -- use torch.no_grad(), or an autograd.Function whose backward is the gradients' call."""
from collections import namedtuple

from . import frames

ConvGrads = namedtuple("ConvGrads", "x weight bias state")
ScanGrads = namedtuple("ScanGrads", "u delta A B C D z delta_bias state")

_CONV_ACTS = ("none", "silu")


def causal_conv(x, weight, bias=None, act="none", state=None, lengths=None, out=None, state_out=None):
    """y_t = act(bias + sum_k weight[:, k] * x_{t - taps + 1 + k}) of every channel by itself; x [items, steps, channels] with
    contiguous channels, weight [channels, taps], taps 1 to 4.

    state [items, taps - 1, channels]: the inputs in front of x, oldest first (None: zeros).  state_out: a tensor of that shape
    that receives the last taps - 1 inputs of each item -- the state of the next call; it may be `state` itself.  lengths: int32
    [items]; y is zero at and behind an item's length, and its state is counted to there."""
    return frames.native().causal_conv(frames.context(x, "x"), False, x, weight, bias, frames.act_of(act, _CONV_ACTS), state, lengths, out,
                                       state_out)


def causal_conv_step(x, state, weight, bias=None, act="none", out=None, state_out=None):
    """causal_conv of one frame: x [items, channels] -> y [items, channels]; `state` is advanced in place, or into state_out."""
    return frames.native().causal_conv(frames.context(x, "x"), True, x, weight, bias, frames.act_of(act, _CONV_ACTS), state, None, out,
                                       state if state_out is None else state_out)


def causal_conv_grad(dy, x, weight, bias=None, act="none", state=None, lengths=None, dstate_out=None, out=None):
    """Gradients of causal_conv as ConvGrads(x, weight, bias, state); dstate_out: the gradient of its state_out (None: zero).
    weight's and bias's are float32 sums over the batch; bias's and state's are None where the argument is None."""
    return ConvGrads(*frames.native().causal_conv_grad(frames.context(x, "x"), dy, x, weight, bias, frames.act_of(act, _CONV_ACTS), state,
                                                       lengths, dstate_out, out))


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None, out=None,
                   state_out=None, keep=False):
    """The recurrence h_t = exp(dt A) h_{t-1} + dt B_t u_t with dt = softplus(delta + delta_bias) (softplus=False: the sum
    itself), and y_t = (sum over the states of C_t h_t + D u_t) * silu(z_t) (z=None: no gate), for every channel.  A and the
    states must be finite, and so must exp(dt A) of every single step.

    u, delta, z [items, steps, channels] with contiguous channels; A float32 [channels, states], 1 to 64 states; B, C [items,
    steps, groups, states], a group serving channels / groups neighbouring channels; D, delta_bias float32 [channels].  state
    float32 [items, channels, states] is the state in front of the first frame (None: zeros); state_out receives the one behind
    each item's last frame and may be `state` itself.  lengths: int32 [items]; behind an item's length y is zero and the state
    stays.  keep=True returns (y, kept): the states of every 16th frame, what selective_scan_grad starts from."""
    y, kept = frames.native().selective_scan(frames.context(u, "u"), False, u, delta, A, B, C, D, z, delta_bias, softplus, state, lengths,
                                             out, state_out, keep)
    return (y, kept) if keep else y


def selective_scan_step(u, delta, A, B, C, state, D=None, z=None, delta_bias=None, softplus=False, out=None, state_out=None):
    """selective_scan of one frame: u, delta, z [items, channels], B, C [items, groups, states] -> y [items, channels]; `state`
    is advanced in place, or into state_out."""
    return frames.native().selective_scan(frames.context(u, "u"), True, u, delta, A, B, C, D, z, delta_bias, softplus, state, None, out,
                                          state if state_out is None else state_out, False)[0]


def selective_scan_grad(dy, u, delta, A, B, C, kept, D=None, z=None, delta_bias=None, softplus=False, state=None, lengths=None,
                        dstate_out=None):
    """Gradients of selective_scan as ScanGrads(u, delta, A, B, C, D, z, delta_bias, state), from the `kept` of the same call;
    dstate_out: the gradient of its state_out (None: zero).  A's, D's, delta_bias's and the state's are float32, the others of
    u's type; None where the argument is None."""
    if kept is None:
        raise frames.bad("kept of the forward call is needed")
    return ScanGrads(*frames.native().selective_scan_grad(frames.context(u, "u"), dy, u, delta, A, B, C, kept, D, z, delta_bias, softplus,
                                                          state, lengths, dstate_out))
