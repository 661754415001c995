"""The feature-map and frame-sequence operators where a range ends: decays that pass float32 over a run of frames, launches past
what one can hold, inputs that ask for gradients."""
import pytest
import torch

import frame_cases as F
import frame_ref as R
from auditory_amd import scan
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
