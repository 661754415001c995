"""Group norm with an activation on channels-last feature maps (aud_group_norm_*, group_norm.hip): the gabor maps of a batch
[n_items, PY * PX, 2 * n_gabor], mel frames [n_items, T, nf], or whatever a network made of them.

Device-resident, on torch's current stream; float32, bfloat16 or float16 maps with float32 parameters."""
import ctypes as C

from . import capi, frames

_ACTS = ("none", "relu", "silu", "gelu")


def _params(call, x, groups, act, eps):
    items, rows, channels = x.shape
    if groups < 1 or channels % groups:
        raise frames.bad("channels (%d) must be a multiple of groups (%d)" % (channels, groups))
    xi, xr = call.rows(x, "x", x.shape)
    return capi.NormParams(call.dtype, call.act(act, _ACTS), items, rows, channels, groups, eps, 0, xi, xr, 0, 0)


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, act="none", lengths=None, out=None, stats=None, want_stats=False):
    """y = act(group_norm(x) * weight + bias); x [items, rows, channels] with contiguous channels, any item and row strides.

    A group is channels / groups neighbouring channels; its mean and (biased) variance run over the item's rows and the group's
    channels.  lengths: int32 [items]; rows at and behind an item's length do not count and come out as zero.  With
    want_stats (or stats given) returns (y, stats), stats float32 [items, groups, 2] for group_norm_grad."""
    call = frames.Call(x, "x", 3)
    p = _params(call, x, groups, act, eps)
    items, _, channels = x.shape
    y = call.out(out, "out", x.shape)
    if stats is None and want_stats:
        stats = call.new(items, groups, 2)
    need = C.c_int64()
    call.ctx.check(call.lib.aud_group_norm_workspace_bytes(C.byref(p), 0, C.byref(need)))
    ws, ws_ptr = call.workspace(need.value)
    call.ctx.check(call.lib.aud_group_norm_batch_dev(
        call.handle, C.byref(p), x.data_ptr(), call.floats(weight, "weight", (channels,)), call.floats(bias, "bias", (channels,)),
        call.lengths(lengths, items), y.data_ptr(), call.floats(stats, "stats", (items, groups, 2)), ws_ptr, need.value, call.stream()))
    return y if stats is None else (y, stats)


def group_norm_grad(dy, x, stats, groups, weight=None, bias=None, eps=1e-5, act="none", lengths=None, out=None):
    """Gradients of group_norm: (dx, dweight, dbias) from dy [items, rows, channels] and the stats of the same call; dweight
    and dbias float32 [channels], summed over the batch (None where the parameter is None)."""
    call = frames.Call(x, "x", 3)
    p = _params(call, x, groups, act, eps)
    items, _, channels = x.shape
    p.dy_item, p.dy_row = call.rows(dy, "dy", x.shape)
    if stats is None:
        raise frames.bad("stats of the forward call are needed")
    dx = call.out(out, "out", x.shape)
    dweight = call.new(channels) if weight is not None else None
    dbias = call.new(channels) if bias is not None else None
    need = C.c_int64()
    call.ctx.check(call.lib.aud_group_norm_workspace_bytes(C.byref(p), 1, C.byref(need)))
    ws, ws_ptr = call.workspace(need.value)
    call.ctx.check(call.lib.aud_group_norm_grad_dev(
        call.handle, C.byref(p), dy.data_ptr(), x.data_ptr(), call.floats(stats, "stats", (items, groups, 2)),
        call.floats(weight, "weight", (channels,)), call.floats(bias, "bias", (channels,)), call.lengths(lengths, items),
        dx.data_ptr(), dweight.data_ptr() if dweight is not None else None, dbias.data_ptr() if dbias is not None else None,
        ws_ptr, need.value, call.stream()))
    return dx, dweight, dbias
