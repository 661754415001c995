"""Group norm with an activation on channels-last feature maps (aud_group_norm_*, group_norm.hip): the gabor maps of a batch
[n_items, PY * PX, 2 * n_gabor], mel frames [n_items, T, nf], or whatever a network made of them.

Device-resident, on torch's current stream; float32, bfloat16 or float16 maps with float32 parameters."""
import ctypes as C

import torch

from . import capi, frames

_ACTS = ("none", "relu", "silu", "gelu")
_PLANS = frames.Plans()


class _Plan:
    def __init__(self, x, groups, act, eps, dy_stride):
        code = frames.dtype_of(x, "x", 3)
        self.ctx = ctx = frames.context(x, "x")
        items, rows, channels = x.shape
        if groups < 1 or channels % groups:
            raise frames.bad("channels (%d) must be a multiple of groups (%d)" % (channels, groups))
        xi, xr = frames.strides(x.shape, x.stride(), "x")
        di, dr = frames.strides(x.shape, dy_stride, "dy") if dy_stride else (0, 0)
        self.p = capi.NormParams(code, frames.act_of(act, _ACTS), items, rows, channels, groups, eps, 0, xi, xr, di, dr)
        self.ref = C.byref(self.p)
        self.nbytes = frames.size_of(ctx, ctx.lib.aud_group_norm_workspace_bytes, self.ref, int(dy_stride is not None)) or 0
        self.per_channel, self.stats, self.dense = (channels,), (items, groups, 2), x.is_contiguous()


def _plan(x, groups, act, eps, dy_stride=None):
    key = (x.dtype, x.shape, x.stride(), x.get_device(), groups, act, eps, dy_stride)
    return _PLANS.get(key) or _PLANS.keep(key, _Plan(x, groups, act, eps, dy_stride))


def _out(out, x, plan, dev):
    if out is None:
        return torch.empty_like(x) if plan.dense else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    frames.dense(out, x, "out", x.shape, dev)
    return out


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, act="none", lengths=None, out=None, stats=None, want_stats=False):
    """y = act(group_norm(x) * weight + bias); x [items, rows, channels] with contiguous channels, any item and row strides.

    A group is channels / groups neighbouring channels; its mean and (biased) variance run over the item's rows and the group's
    channels.  lengths: int32 [items]; rows at and behind an item's length do not count and come out as zero.  With
    want_stats (or stats given) returns (y, stats), stats float32 [items, groups, 2] for group_norm_grad."""
    plan = _plan(x, groups, act, eps)
    ctx, ch, dev = plan.ctx, plan.per_channel, x.get_device()
    y = _out(out, x, plan, dev)
    if stats is None and want_stats:
        stats = torch.empty(plan.stats, dtype=frames.F32, device=x.device)
    ws = frames.scratch(plan.nbytes, x)
    rc = ctx.lib.aud_group_norm_batch_dev(
        ctx.handle, plan.ref, x.data_ptr(), frames.floats(weight, x, "weight", ch, dev), frames.floats(bias, x, "bias", ch, dev),
        frames.lengths_of(lengths, x, plan.stats[0], dev), y.data_ptr(), frames.floats(stats, x, "stats", plan.stats, dev),
        ws.data_ptr() if ws is not None else None, plan.nbytes, frames.current_stream(dev))
    if rc:
        ctx.check(rc)
    return y if stats is None else (y, stats)


def group_norm_grad(dy, x, stats, groups, weight=None, bias=None, eps=1e-5, act="none", lengths=None, out=None):
    """Gradients of group_norm: (dx, dweight, dbias) from dy [items, rows, channels] and the stats of the same call; dweight
    and dbias float32 [channels], summed over the batch (None where the parameter is None)."""
    plan = _plan(x, groups, act, eps, dy.stride())
    ctx, ch, dev = plan.ctx, plan.per_channel, x.get_device()
    frames.like(dy, x, "dy", x.shape, dev)
    if stats is None:
        raise frames.bad("stats of the forward call are needed")
    dx = _out(out, x, plan, dev)
    dweight = torch.empty(ch, dtype=frames.F32, device=x.device) if weight is not None else None
    dbias = torch.empty(ch, dtype=frames.F32, device=x.device) if bias is not None else None
    ws = frames.scratch(plan.nbytes, x)
    rc = ctx.lib.aud_group_norm_grad_dev(
        ctx.handle, plan.ref, dy.data_ptr(), x.data_ptr(), frames.floats(stats, x, "stats", plan.stats, dev),
        frames.floats(weight, x, "weight", ch, dev), frames.floats(bias, x, "bias", ch, dev),
        frames.lengths_of(lengths, x, plan.stats[0], dev), dx.data_ptr(), dweight.data_ptr() if dweight is not None else None,
        dbias.data_ptr() if dbias is not None else None, ws.data_ptr() if ws is not None else None, plan.nbytes,
        frames.current_stream(dev))
    if rc:
        ctx.check(rc)
    return dx, dweight, dbias
