"""Group norm with an activation on channels-last feature maps (aud_group_norm_*, group_norm.hip): the gabor maps of a batch
[n_items, PY * PX, 2 * n_gabor], mel frames [n_items, T, nf], or whatever a network made of them.

Device-resident, on torch's current stream; float32, bfloat16 or float16 maps with float32 parameters.  The gradients are
functions of their own: nothing here records for torch's autograd, so a tensor that requires grad is refused while autograd
records -- use torch.no_grad(), or an autograd.Function whose backward is the gradients' call."""
from . import frames

_ACTS = ("none", "relu", "silu", "gelu")


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, act="none", lengths=None, out=None, stats=None, want_stats=False):
    """y = act(group_norm(x) * weight + bias); x [items, rows, channels] with contiguous channels, any item and row strides.

    A group is channels / groups neighbouring channels; its mean and (biased) variance run over the item's rows and the group's
    channels.  lengths: int32 [items]; rows at and behind an item's length do not count and come out as zero.  With
    want_stats (or stats given) returns (y, stats), stats float32 [items, groups, 2] for group_norm_grad."""
    y, stats = frames.native().group_norm(frames.context(x, "x"), x, groups, weight, bias, eps, frames.act_of(act, _ACTS), lengths, out,
                                          stats, want_stats)
    return y if stats is None else (y, stats)


def group_norm_grad(dy, x, stats, groups, weight=None, bias=None, eps=1e-5, act="none", lengths=None, out=None):
    """Gradients of group_norm: (dx, dweight, dbias) from dy [items, rows, channels] and the stats of the same call; dweight
    and dbias float32 [channels], summed over the batch (None where the parameter is None)."""
    if stats is None:
        raise frames.bad("stats of the forward call are needed")
    return frames.native().group_norm_grad(frames.context(x, "x"), dy, x, stats, groups, weight, bias, eps, frames.act_of(act, _ACTS),
                                           lengths, out)
