"""The feature-map and frame-sequence operators where a range ends: decays that pass float32 over a run of frames, launches past
what one can hold, inputs that ask for gradients."""
import pytest
import torch

import frame_cases as F
import frame_ref as R
from auditory_amd import capi, norm, scan
from test_norm_widths import emu, emu_lib  # noqa: F401  (fixtures)

gpu = pytest.mark.gpu


# ---- a run of frames whose decay, taken at once, is past float32 -------------------------------------------------------------

def near(name, got, ref, k):
    """all terms of a sum have one sign here, so the value is the magnitude: k half steps of it"""
    got, ref = got.detach().cpu().double(), ref.detach()
    assert torch.isfinite(ref).all() and torch.isfinite(got).all(), name
    assert ((got - ref).abs() <= k * R.U * ref.abs() + 1e-37).all(), (name, float(((got - ref).abs() / ref.abs().clamp(min=1e-37)).max()))


def growing(dev, items, steps, ch, states, grow, rate, u_from, dy_on, first, dy_value):
    """step sizes `rate` in the frames `grow` (0 elsewhere, but where u is), A = 1 .. 2, everything positive"""
    m = F.Make(dev, 5, "f32")
    pos = lambda *s: 0.5 + m.u(*s)  # noqa: E731
    delta = torch.zeros(items, steps, ch, device=dev)
    delta[:, grow] = rate
    u, dy = torch.zeros(items, steps, ch, device=dev), torch.zeros(items, steps, ch, device=dev)
    if u_from is not None:
        u[:, u_from:] = pos(items, steps - u_from, ch)
        delta[:, u_from:] = 0.25
    dy[:, dy_on] = dy_value * pos(items, steps, ch)[:, dy_on]
    A = 1 + m.u(ch, states)
    B, C = pos(items, steps, 1, states), pos(items, steps, 1, states)
    state = first * pos(items, ch, states)
    so = torch.empty_like(state)
    y, kept = scan.selective_scan(u, delta, A, B, C, state=state, state_out=so, keep=True)
    g = scan.selective_scan_grad(dy, u, delta, A, B, C, kept, state=state)
    lv = [R.leaf(t) for t in (u, delta, A, B, C, state)]
    ry, rs = R.scan(*lv[:5], None, None, None, False, lv[5], None)
    rg = R.grads([ry], [dy], lv)
    # a step: 5 half steps, and those of its exponent; the exponent of a run is a sum of its step sizes: at most `steps` more of
    # the whole exponent, which |sum dt A| <= 2 rate frames holds.  Twice that for gradients, which have such a run on both sides
    k = 5 * steps + (steps + 8) * 2 * rate * len(range(*grow.indices(steps))) + states + 16
    near("y", y, ry, k)
    near("state", so, rs, k)
    for name, got, ref in zip(("u", "delta", "A", "B", "C", "state"), (g.u, g.delta, g.A, g.B, g.C, g.state), rg):
        near("d" + name, got, ref, 2 * k + items * steps + ch)


def decays_past_float32(dev, items=1):
    steps = 640
    # nothing to carry: the input comes in the last frames, the gradient from the first, the step sizes are 1 all the way
    growing(dev, items, steps, 4, 3, slice(0, steps), 1.0, steps - 8, slice(0, 8), 0.0, 1.0)
    # something small to carry over 64 frames: 1e-30 e^96 and more
    growing(dev, items, steps, 4, 3, slice(128, 192), 0.75, steps - 8, slice(steps - 8, steps), 1e-33, 1e-33)
    # growth within 40 frames that lie in two chunks, small values on both sides
    growing(dev, items, steps, 4, 3, slice(172, 212), 1.25, steps - 4, slice(steps - 4, steps), 1e-34, 1e-34)


def test_emul_decays_past_float32(emu):  # noqa: F811
    decays_past_float32("cpu")


@gpu
def test_gpu_decays_past_float32():
    decays_past_float32("cuda:0")        # the axis is cut, few chunks
    decays_past_float32("cuda:0", 450)   # not cut


def many_chunks(dev):
    """more chunks than are walked one by one"""
    steps = 1100 if dev == "cpu" else 4200
    growing(dev, 1, steps, 4, 3, slice(0, steps), 1.0, steps - 8, slice(0, 8), 0.0, 1.0)
    growing(dev, 1, steps, 4, 3, slice(128, 192), 0.75, steps - 8, slice(steps - 8, steps), 1e-33, 1e-33)


def test_emul_decays_past_float32_many_chunks(emu):  # noqa: F811
    many_chunks("cpu")


@gpu
def test_gpu_decays_past_float32_many_chunks():
    many_chunks("cuda:0")


# ---- inputs that ask for gradients -------------------------------------------------------------------------------------------

def calls(dev):
    """(name, call, its tensors by argument) of every entry point"""
    m = F.Make(dev, 13, "f32")
    x, dy, w, b = m.n(2, 5, 8), m.n(2, 5, 8), m.n(8), m.n(8)
    _, st = norm.group_norm(x, 2, w, b, want_stats=True)
    cw, cs = m.n(8, 3), m.n(2, 2, 8)
    a = F.scan_inputs(m, 2, 5, 8, 1, 4, True, True, True, True, True)
    one = {n: a[n][:, 0] if n in ("u", "delta", "B", "C", "z") else a[n] for n in a}
    _, kept = scan.selective_scan(**a, softplus=True, keep=True)
    return [
        ("group_norm", lambda **t: norm.group_norm(groups=2, **t), dict(x=x, weight=w, bias=b)),
        ("group_norm_grad", lambda **t: norm.group_norm_grad(groups=2, **t), dict(dy=dy, x=x, stats=st, weight=w, bias=b)),
        ("causal_conv", lambda **t: scan.causal_conv(**t), dict(x=x, weight=cw, bias=b, state=cs)),
        ("causal_conv_step", lambda **t: scan.causal_conv_step(**t), dict(x=x[:, 0], state=cs.clone(), weight=cw, bias=b)),
        ("causal_conv_grad", lambda **t: scan.causal_conv_grad(**t), dict(dy=dy, x=x, weight=cw, bias=b, state=cs, dstate_out=cs)),
        ("selective_scan", lambda **t: scan.selective_scan(softplus=True, **t), a),
        ("selective_scan_step", lambda **t: scan.selective_scan_step(softplus=True, **t), {**one, "state": one["state"].clone()}),
        ("selective_scan_grad", lambda **t: scan.selective_scan_grad(softplus=True, **t), dict(a, dy=dy, kept=kept, dstate_out=a["state"])),
    ]


def flat(out):
    return [t for t in (out if isinstance(out, tuple) else (out,)) if t is not None]


def gradients_asked_for(dev):
    """nothing is recorded for autograd, so a call that autograd would have to record is refused; within no_grad (and so in the
    forward and backward of an autograd.Function) the same tensors are taken"""
    for name, call, tensors in calls(dev):
        fresh = lambda: {n: t.clone() for n, t in tensors.items()}  # noqa: E731
        want = flat(call(**fresh()))
        for n in tensors:
            asks = fresh()
            asks[n].requires_grad_(True)
            with pytest.raises(capi.AuditoryError) as e:
                call(**asks)
            assert e.value.status == capi.AUD_EINVAL and "no_grad" in str(e.value), (name, n)
            with torch.no_grad():
                got = flat(call(**asks))
            assert all(torch.equal(p, q) and not p.requires_grad for p, q in zip(got, want)), (name, n)
    with pytest.raises(capi.AuditoryError):
        x = torch.zeros(2, 5, 8, device=dev)
        norm.group_norm(x, 2, out=torch.zeros_like(x).requires_grad_(True))


def test_emul_gradients_asked_for(emu):  # noqa: F811
    gradients_asked_for("cpu")


@gpu
def test_gpu_gradients_asked_for():
    gradients_asked_for("cuda:0")


class Normed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        y, stats = norm.group_norm(x, 2, w, b, act="silu", want_stats=True)
        ctx.save_for_backward(x, w, b, stats)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, b, stats = ctx.saved_tensors
        return norm.group_norm_grad(dy.contiguous(), x, stats, 2, w, b, act="silu")


def in_a_function(dev):
    m = F.Make(dev, 17, "f32")
    x, dy, w, b = m.n(2, 5, 8), m.n(2, 5, 8), m.n(8), m.n(8)
    _, st = norm.group_norm(x, 2, w, b, act="silu", want_stats=True)
    want = norm.group_norm_grad(dy, x, st, 2, w, b, act="silu")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    (Normed.apply(*leaves) * dy).sum().backward()
    assert all(torch.equal(t.grad, q) for t, q in zip(leaves, want))


def test_emul_in_a_function(emu):  # noqa: F811
    in_a_function("cpu")


@gpu
def test_gpu_in_a_function():
    in_a_function("cuda:0")
