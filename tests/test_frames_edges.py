"""The feature-map and frame-sequence operators where a range ends: decays that pass float32 over a run of frames, inputs that ask
for gradients, grids of more threads than a launch can hold."""
import ctypes as C

import pytest
import torch

import frame_cases as F
import frame_ref as R
import norm_cases as N
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


# ---- grids of more threads than a launch can hold ----------------------------------------------------------------------------

@pytest.fixture
def small_launches(emu):  # noqa: F811
    """the emulator refuses launches past its build's limit"""
    import build_emul
    limit = C.c_longlong.in_dll(emu, "aud_emul_launch_threads")
    before, limit.value = limit.value, build_emul.LAUNCH_THREADS
    yield
    limit.value = before


SLICED = [
    (N.case, (10, 3, 24, 3, "f32", "silu", True, None, 0)),                    # items held in registers, the gradients' item kernel
    (N.case, (9, 6, 1300, 13, "bf16", "gelu", True, None, 0)),                 # items read twice, the parameters' column sums
    (N.case, (5, 24, 1024, 1024, "f32", "none", True, None, 0)),               # chunks, many groups
    (N.case, (2, 600, 32, 4, "f32", "silu", True, "mixed", 0)),                # chunks, joined by all
    (F.conv_case, (5, 70, 130, 4, "bf16", "silu", True, True, "mixed", 1)),
    (F.scan_case, (2, 34, 130, 2, 17, "f32", True, True, True, True, True, "mixed", 0)),   # two blocks a group, chunks
    (F.scan_case, (33, 1, 65, 1, 4, "f32", True, True, True, True, True, None, 0)),        # one frame
    (F.scan_case, (1, 560, 65, 1, 32, "f32", True, True, True, True, True, None, 0)),      # the gradients' chunks joined by a kernel
]


@pytest.mark.parametrize("i", range(len(SLICED)))
def test_emul_launches_in_slices(small_launches, i):
    fn, case = SLICED[i]
    fn("cpu", *case)


@gpu
def test_gpu_norm_of_more_items_than_a_launch_holds():
    """2^23 items and some of 512 threads each: every item as it comes out alone"""
    dev, n, k = "cuda:0", 1 << 10, (1 << 13) + 1
    m = F.Make(dev, 23, "bf16")
    x, dy, w, b = m.n(n, 1, 16), m.n(n, 1, 16), m.n(16, f32=True), m.n(16, f32=True)
    y, st = norm.group_norm(x, 4, w, b, act="silu", want_stats=True)
    dx, dw, db = norm.group_norm_grad(dy, x, st, 4, w, b, act="silu")
    many = lambda t: t.repeat(k, *[1] * (t.dim() - 1))  # noqa: E731
    ys, sts = norm.group_norm(many(x), 4, w, b, act="silu", want_stats=True)
    assert torch.equal(ys.view(k, n, 16), y.view(1, n, 16).expand(k, n, 16))
    assert torch.equal(sts.view(k, n, 8), st.view(1, n, 8).expand(k, n, 8))
    dxs, dws, dbs = norm.group_norm_grad(many(dy), many(x), sts, 4, w, b, act="silu")
    assert torch.equal(dxs.view(k, n, 16), dx.view(1, n, 16).expand(k, n, 16))
    # the sums over k n items: at most k n / 32 + 16 additions follow each other
    e = N.Exact(x, dy, 4, w, b, 1e-5, "silu", None)
    for got, one, bound in ((dws, dw, e.edw), (dbs, db, e.edb)):
        terms = bound / R.U  # (the bound holds (S >= 1) u times the sum of the terms' absolute values)
        assert ((got.cpu().double() - k * one.cpu().double()).abs() <= k * (bound + (k * n / 32 + 16) * R.U * terms)).all()


@gpu
def test_gpu_conv_of_more_threads_than_a_launch_holds():
    """2^32 threads of one element, one frame each"""
    dev, n = "cuda:0", 65537
    m = F.Make(dev, 29, "bf16")
    row, w, b = m.n(1, n), m.n(n, 1, f32=True), m.n(n, f32=True)
    one = scan.causal_conv_step(row, None, w, b, act="silu")
    x = row.expand(n, n).contiguous()
    y = scan.causal_conv_step(x, None, w, b, act="silu")
    assert all(torch.equal(y[i:i + 4096], one.expand(min(4096, n - i), n)) for i in range(0, n, 4096))


@gpu
def test_gpu_scans_of_more_threads_than_a_launch_holds():
    dev = "cuda:0"
    # one frame: 2^30 channels and some, four lanes each
    items, ch = (1 << 15) + 1, 1 << 15
    m = F.Make(dev, 31, "bf16")
    u, delta, z = m.n(1, ch), m.n(1, ch), m.n(1, ch)
    B, Cm, A = m.n(1, 1, 1), m.n(1, 1, 1), -m.u(ch, 1)
    h = m.n(1, ch, 1, f32=True)
    many = lambda t: t.expand(items, *t.shape[1:]).contiguous()  # noqa: E731
    one = h.clone()
    y = scan.selective_scan_step(u, delta, A, B, Cm, one, z=z, softplus=True)
    state = many(h)
    ys = scan.selective_scan_step(many(u), many(delta), A, many(B), many(Cm), state, z=many(z), softplus=True)
    assert torch.equal(ys, many(y)) and torch.equal(state, many(one))
    del ys, state
    # 2^24 workgroups and some: a channel a group
    items, ch = 17, 1 << 20
    u, delta, dy = m.n(1, 2, ch), m.n(1, 2, ch), m.n(1, 2, ch)
    B, Cm, A = m.n(1, 2, ch, 1), m.n(1, 2, ch, 1), -m.u(ch, 1)
    y, kept = scan.selective_scan(u, delta, A, B, Cm, softplus=True, keep=True)
    g = scan.selective_scan_grad(dy, u, delta, A, B, Cm, kept, softplus=True)
    args = [many(u), many(delta), A, many(B), many(Cm)]
    ys, kept = scan.selective_scan(*args, softplus=True, keep=True)
    assert torch.equal(ys, many(y))
    gs = scan.selective_scan_grad(many(dy), *args, kept, softplus=True)
    for p, q in ((gs.u, g.u), (gs.delta, g.delta), (gs.B, g.B), (gs.C, g.C)):
        assert torch.equal(p, many(q))
