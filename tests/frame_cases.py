"""Cases of the feature-map and frame-sequence operators, run by test_frames.py on the CPU thread emulator (tensors on the
CPU) and on the GPU.  Bounds: frame_ref.py."""
import math

import torch

import frame_ref as R
from auditory_amd import norm, scan

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


class Make:
    """inputs from a seed, made in float32 on the CPU and moved"""

    def __init__(self, dev, seed, dtype):
        self.g = torch.Generator().manual_seed(seed)
        self.dev, self.t = dev, TYPES[dtype]

    def n(self, *shape, scale=1.0, shift=0.0, f32=False):
        v = torch.randn(shape, generator=self.g) * scale + shift
        return v.to(torch.float32 if f32 else self.t).to(self.dev)

    def u(self, *shape):
        return torch.rand(shape, generator=self.g).to(self.dev)

    def lengths(self, kind, items, rows):
        if kind is None:
            return None
        v = {"mixed": [rows, 0, 1, max(rows - 1, 0), rows // 2], "zero": [0], "out": [rows + 7, -3, rows]}[kind]
        return torch.tensor([v[i % len(v)] for i in range(items)], dtype=torch.int32).to(self.dev)

    def strided(self, t, pad, last=0):
        """the same values in a wider buffer: row stride + pad, one row of slack an item; NaN in between"""
        b, r, c = t.shape
        wide = torch.full((b, r + 1, c + pad), math.nan, dtype=t.dtype, device=t.device)
        wide[:, :r, last:last + c] = t
        return wide[:, :r, last:last + c]


def poison(t, lengths):
    """NaN and infinities in the rows behind each item's length"""
    if lengths is None:
        return t
    t = t.clone()
    for b, n in enumerate(lengths.cpu().tolist()):
        n = min(max(n, 0), t.shape[1])
        if n < t.shape[1]:
            t[b, n:] = math.nan
            t[b, -1].view(-1)[0] = math.inf
    return t


# ---- group norm: (items, rows, channels, groups, type, activation, affine, lengths, row padding, level) -------------------
NORM = [
    (2, 5, 16, 2, "f32", "none", True, None, 0, 0.0),
    (1, 1, 1, 1, "f32", "relu", False, None, 0, 0.0),          # one value a group: xh = 0
    (3, 7, 40, 8, "f32", "silu", True, "mixed", 0, -3.0),
    (2, 9, 33, 3, "bf16", "gelu", True, "mixed", 0, 0.0),       # odd width: one element at a time
    (2, 33, 24, 24, "f16", "silu", True, None, 0, 0.0),         # a channel a group
    (1, 20, 32, 1, "bf16", "none", True, None, 8, 0.0),         # one group, rows apart
    (2, 6, 32, 4, "bf16", "silu", True, "out", 3, 0.0),         # rows at odd addresses
    (2, 64, 8, 2, "f32", "silu", True, None, 0, 1000.0),        # a level far from zero
    (3, 4, 12, 4, "f16", "gelu", False, "zero", 0, 0.0),        # nothing but padding
]
# the routes that take larger sizes (on the GPU)
NORM_BIG = [
    (2, 600, 32, 4, "f32", "silu", True, "mixed", 0, 0.0),       # an item over several workgroups
    (3, 777, 132, 12, "f16", "gelu", True, "mixed", 0, 0.0),     # packs of four
    (1, 500, 33, 3, "bf16", "silu", True, None, 0, 0.0),         # one element at a time
    (1, 100, 1024, 1024, "f32", "none", True, None, 0, 0.0),     # many groups: the chunks joined by a kernel of their own
    (2, 40, 4096, 64, "bf16", "silu", True, "mixed", 0, 0.0),    # more packs than threads
    (1, 9, 4095, 5, "f32", "relu", True, None, 0, 0.0),
    (300, 5, 64, 4, "f32", "silu", True, "mixed", 0, 0.0),
    (257, 300, 32, 8, "f32", "silu", True, None, 0, 0.0),        # an item in one workgroup, read twice
    (2, 3000, 16, 2, "f32", "relu", True, None, 0, 300.0),
]


def norm_case(dev, items, rows, ch, groups, dtype, name, affine, lens, pad, level, seed=1):
    m = Make(dev, seed + items * rows + ch, dtype)
    x = m.n(items, rows, ch, scale=1.5, shift=level)
    dy = m.n(items, rows, ch)
    w, b = (m.n(ch, f32=True, scale=0.3, shift=1.0), m.n(ch, f32=True, scale=0.3)) if affine else (None, None)
    lengths = m.lengths(lens, items, rows)
    xs, ds = (m.strided(x, pad), m.strided(dy, pad)) if pad else (x, dy)
    xs, ds = poison(xs, lengths) if not pad else xs, poison(ds, lengths) if not pad else ds
    y, stats = norm.group_norm(xs, groups, w, b, act=name, lengths=lengths, want_stats=True)
    y2 = norm.group_norm(xs, groups, w, b, act=name, lengths=lengths)
    assert torch.equal(y, y2)
    dx, dw, db = norm.group_norm_grad(ds, xs, stats, groups, w, b, act=name, lengths=lengths)
    # the definition in 64 bits
    lv = [R.leaf(t) for t in (x, w, b)]
    ry, rst = R.norm(lv[0], groups, lv[1], lv[2], 1e-5, name, lengths)
    rdx, rdw, rdb = R.grads([ry], [dy], lv)
    # Roundings.  The statistics are sums of n values in short runs joined pairwise: at most `run` of them follow each other,
    # run = rows a thread has + rows x channels joined + 16.  With D = the largest |x - x'| of a group, d = D / std:
    # xh carries at most run u (d + |xh| d^2) + 4 u |xh|, |xh| <= d; so k = run + 16 with magnitude (1 + d)^3 covers p, y
    # and, with one more factor (1 + d), the sums of the gradients.
    cg = ch // groups
    n = torch.tensor(R.lens_of(lengths, items, rows))
    run = rows + cg + 32
    v = x.detach().cpu().double().reshape(items, rows, groups, cg)
    live = (torch.arange(rows)[None] < n[:, None])[:, :, None, None]
    hi, lo = torch.where(live, v, -math.inf).amax((1, 3)), torch.where(live, v, math.inf).amin((1, 3))
    D = torch.where(torch.isfinite(hi - lo), hi - lo, 0.0)
    sd = 1 / rst[..., 1].detach()
    d = (1 + D / sd)[:, None, :, None].expand(items, rows, groups, cg).reshape(items, rows, ch)
    one = torch.ones(ch, dtype=torch.float64)
    wa, ba = (w.detach().cpu().double().abs(), b.detach().cpu().double().abs()) if affine else (one, 0 * one)
    on = live[..., 0].expand(items, rows, ch).double()
    R.check("y", y, ry, (d ** 3 * wa + ba) * on * 1.2, run + 16)
    R.check("mean", stats[..., 0], rst[..., 0], D + rst[..., 0].abs() * 0.05, run + 16)
    R.check("rstd", stats[..., 1], rst[..., 1], rst[..., 1] * (1 + D / sd) ** 2, run + 16)
    q = dy.detach().cpu().double().abs() * on * 1.2
    # q is a product of dy and act'(p): act' moves by at most 1.2 x what p moves
    qm = q * (1 + d ** 3 * wa)
    tot = run + rows * items + 64
    if affine:
        R.check("dweight", dw, rdw, (qm * d).sum((0, 1)), tot)
        R.check("dbias", db, rdb, qm.sum((0, 1)), tot)
    tm = (qm * wa).reshape(items, rows, groups, cg)
    cnt = torch.clamp(n * cg, min=1)[:, None, None, None]
    dm = d.reshape(items, rows, groups, cg)
    mag = (tm + tm.sum((1, 3), keepdim=True) / cnt + dm * (tm * dm).sum((1, 3), keepdim=True) / cnt) * dm ** 2
    R.check("dx", dx, rdx, (mag / sd[:, None, :, None]).reshape(items, rows, ch) * on, tot)
    if lengths is not None:
        gone = (live[..., 0].expand(items, rows, ch) == 0)
        assert (y.cpu()[gone] == 0).all() and (dx.cpu()[gone] == 0).all()


# ---- causal convolution: (items, steps, channels, taps, type, activation, bias, state, lengths, row padding) ---------------
CONV = [
    (2, 9, 8, 4, "f32", "silu", True, True, None, 0),
    (1, 1, 1, 1, "f32", "none", False, False, None, 0),
    (3, 1, 24, 4, "f16", "silu", True, True, None, 0),           # one frame
    (5, 11, 7, 3, "bf16", "silu", True, True, "mixed", 0),       # odd width, lengths 11, 0, 1, 10, 5
    (2, 70, 16, 4, "bf16", "silu", True, False, None, 0),        # several runs of steps
    (2, 41, 20, 2, "f16", "none", True, True, "out", 0),
    (2, 6, 16, 4, "bf16", "silu", False, True, "mixed", 8),
    (5, 2, 16, 4, "f32", "none", True, True, "mixed", 5),        # shorter than the filter
    (2, 0, 8, 3, "f32", "silu", True, True, None, 0),            # no frame at all
]
CONV_BIG = [
    (3, 1030, 64, 4, "bf16", "silu", True, True, "mixed", 0),
    (2, 517, 130, 3, "f16", "silu", True, True, None, 6),
    (65, 1, 1024, 4, "f16", "silu", True, True, None, 0),
    (1, 4100, 24, 2, "f32", "none", True, False, None, 0),
]


def conv_case(dev, items, steps, ch, taps, dtype, name, has_bias, has_state, lens, pad, seed=2):
    m = Make(dev, seed + items * steps + ch, dtype)
    x, dy = m.n(items, steps, ch), m.n(items, steps, ch)
    w = m.n(ch, taps, f32=True, scale=0.6)
    b = m.n(ch, f32=True, scale=0.3) if has_bias else None
    s = m.n(items, taps - 1, ch) if has_state else None
    ds = m.n(items, taps - 1, ch)
    lengths = m.lengths(lens, items, steps)
    xs, dys = (m.strided(x, pad), m.strided(dy, pad)) if pad else (poison(x, lengths), poison(dy, lengths))
    so = torch.empty_like(ds)
    y = scan.causal_conv(xs, w, b, act=name, state=s, lengths=lengths, state_out=so)
    if has_state:  # the state advanced in place gives the same
        again = s.clone()
        y2 = scan.causal_conv(xs, w, b, act=name, state=again, lengths=lengths, state_out=again)
        assert torch.equal(y, y2) and torch.equal(again, so)
    g = scan.causal_conv_grad(dys, xs, w, b, act=name, state=s, lengths=lengths, dstate_out=ds)
    lv = [R.leaf(t) for t in (x, w, b, s)]
    ry, rs = R.conv(lv[0], lv[1], lv[2], name, lv[3], lengths)
    rg = R.grads([ry, rs], [dy, ds], lv)
    assert torch.equal(so.cpu().double(), rs.detach())  # the inputs themselves
    # p = b + sum of taps products: taps + 1 roundings of magnitude P; silu and its slope: 1.1 P and 6 more of |y| <= P
    absd = lambda t: None if t is None else t.detach().cpu().double().abs()  # noqa: E731
    P, _ = R.conv(absd(x), absd(w), absd(b), "none", absd(s), lengths)
    R.check("y", y, ry, P, 2 * taps + 10)
    # q = dy act'(p), act' within 1.1 and moving 0.5 x P: magnitude dy (1.1 + 0.5 P)
    q = (absd(dy) * (1.1 + 0.5 * P)).detach()
    al = [R.leaf(absd(t)) for t in (x, w, b, s)]
    my, ms = R.conv(al[0], al[1], al[2], "none", al[3], lengths)
    mg = R.grads([my, ms], [q, absd(ds)], al)
    k = 3 * taps + 16
    R.check("dx", g.x, rg[0], mg[0], k)
    R.check("dweight", g.weight, rg[1], mg[1], k + items * steps)
    if has_bias:
        R.check("dbias", g.bias, rg[2], mg[2], k + items * steps)
    if has_state:
        R.check("dstate", g.state, rg[3], mg[3], k)
    assert (g.bias is None) == (not has_bias) and (g.state is None) == (not has_state)


# ---- selective scan: (items, steps, channels, groups, states, type, D, gate, bias, softplus, state, lengths, row padding) --
SCAN = [
    (1, 1, 1, 1, 1, "f32", False, False, False, False, False, None, 0),
    (2, 5, 8, 1, 4, "f32", True, True, True, True, True, None, 0),
    (5, 20, 8, 2, 8, "f32", True, True, True, True, True, "mixed", 0),
    (2, 17, 9, 3, 5, "bf16", True, True, True, True, True, None, 0),     # odd sizes
    (1, 33, 70, 1, 16, "f16", True, True, True, True, False, None, 0),   # more than one block of channels
    (2, 18, 12, 1, 24, "bf16", False, True, False, True, True, "out", 8),
    (1, 19, 6, 2, 33, "f32", True, False, True, True, True, None, 5),
    (1, 130, 4, 1, 4, "f32", True, True, True, True, True, None, 0),     # a time axis cut into chunks
    (3, 200, 8, 1, 3, "bf16", True, False, True, True, True, "mixed", 0),
    (2, 0, 8, 1, 4, "f32", True, True, True, True, True, None, 0),       # no frame at all
]
SCAN_BIG = [
    (1, 1000, 8, 1, 16, "f32", True, True, True, True, True, None, 0),      # more chunks than are folded
    (170, 20, 8, 1, 4, "bf16", True, True, True, True, True, "mixed", 0),   # enough items: the axis is not cut
    (2, 150, 200, 2, 64, "f16", True, True, True, True, True, "mixed", 0),  # four blocks of channels, 64 states
    (2, 90, 65, 1, 24, "bf16", True, False, True, True, True, None, 3),     # odd blocks
    (70, 1, 130, 1, 16, "bf16", True, True, True, True, True, None, 0),     # one frame
    (450, 18, 8, 1, 8, "f32", True, True, True, True, False, "mixed", 0),   # gradients with an uncut axis
]


def scan_inputs(m, items, steps, ch, groups, states, has_D, gate, has_bias, softplus, has_state):
    a = dict(u=m.n(items, steps, ch))
    if softplus:
        a["delta"] = m.n(items, steps, ch, scale=0.7, shift=0.0 if has_bias else -2.0)
    else:
        a["delta"] = (m.u(items, steps, ch) * 0.3 + 0.01).to(m.t)
    a["A"] = -(torch.arange(1, states + 1, dtype=torch.float32).to(m.dev) * (0.5 + m.u(ch, 1)))
    a["B"], a["C"] = m.n(items, steps, groups, states), m.n(items, steps, groups, states)
    a["D"] = m.n(ch, f32=True) if has_D else None
    a["z"] = m.n(items, steps, ch) if gate else None
    a["delta_bias"] = (m.u(ch) * 3 - 4.5) if has_bias else None
    a["state"] = m.n(items, ch, states, f32=True) if has_state else None
    return a


def scan_case(dev, items, steps, ch, groups, states, dtype, has_D, gate, has_bias, softplus, has_state, lens, pad, seed=3):
    m = Make(dev, seed + items * steps + ch + states, dtype)
    a = scan_inputs(m, items, steps, ch, groups, states, has_D, gate, has_bias, softplus, has_state)
    dy, ds = m.n(items, steps, ch), m.n(items, ch, states, f32=True)
    lengths = m.lengths(lens, items, steps)
    run = dict(a)
    wide = (lambda t: m.strided(t, pad)) if pad else (lambda t: poison(t, lengths))
    for n in ("u", "delta", "z"):
        run[n] = wide(a[n]) if a[n] is not None else None
    for n in ("B", "C"):
        if pad:
            run[n] = m.strided(a[n].reshape(items, steps, groups * states), pad).unflatten(2, (groups, states))
        else:
            run[n] = poison(a[n], lengths)
    dys = wide(dy)
    so = torch.empty((items, ch, states), device=dy.device)
    kw = dict(D=run["D"], z=run["z"], delta_bias=run["delta_bias"], softplus=softplus, state=run["state"], lengths=lengths)
    args = [run[n] for n in ("u", "delta", "A", "B", "C")]
    y, kept = scan.selective_scan(*args, state_out=so, keep=True, **kw)
    g = scan.selective_scan_grad(dys, *args, kept, dstate_out=ds, **kw)
    if has_state:
        again = run["state"].clone()
        y2 = scan.selective_scan(*args, state_out=again, **{**kw, "state": again})
        if steps != 1:  # (one frame without `keep` is another kernel)
            assert torch.equal(y, y2) and torch.equal(so, again)
    scan_check(a, lengths, softplus, dy, ds, y, so, g)


def scan_check(a, lengths, softplus, dy, ds, y, so, g):
    names = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")
    lv = {n: R.leaf(a[n]) for n in names}
    ry, rs = R.scan(*[lv[n] for n in names[:5]], lv["D"], lv["z"], lv["delta_bias"], softplus, lv["state"], lengths)
    rg = dict(zip(names, R.grads([ry, rs], [dy, ds], [lv[n] for n in names])))
    # Magnitudes: the same recurrences over absolute values.  dt and its decay are taken as they are; dt depends on delta, so
    # the gradient of delta is that of dt, taken through a leaf of its own.
    absd = lambda t: None if t is None else t.detach().cpu().double().abs()  # noqa: E731
    raw = a["delta"].detach().cpu().double() + (a["delta_bias"].detach().cpu().double() if a["delta_bias"] is not None else 0.0)
    dt = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    zz = a["z"].detach().cpu().double() if a["z"] is not None else None
    sil = (zz / (1 + torch.exp(-zz))).abs() if zz is not None else None
    ml = {n: R.leaf(absd(a[n])) for n in ("u", "B", "C", "D", "state")}
    mdt, mdecay, mA = R.leaf(dt), R.leaf(dt), R.leaf(a["A"])
    my, ms = R.scan(ml["u"], mdt, mA, ml["B"], ml["C"], ml["D"], None, None, False, ml["state"], lengths, plain_gate=sil, decay=mdecay)
    mg = dict(zip(("u", "delta", "A", "B", "C", "D", "state", "decay"),
                  R.grads([my, ms], [absd(dy), absd(ds)], [ml["u"], mdt, mA, ml["B"], ml["C"], ml["D"], ml["state"], mdecay])))
    # (the two terms of ddt, through the input and through the decay, may have opposite signs: their magnitudes add up)
    mag_dt = mg["delta"].abs() + mg["decay"].abs()
    # Roundings.  dt is good to c1 = 11 + max |raw| half steps (bias added, softplus); a step of h adds a product and a fused
    # product, and moves a by c1 |dt A| + 3: over a run of L steps that is c1 + 5 L at most, because |dt A| weighed by the
    # decay sums to less than 1.  A gradient has such a chain on both sides, and its sums over states, channels or frames.
    items, steps, ch = a["u"].shape
    states = a["A"].shape[1]
    c1 = 11 + float(raw.abs().max()) if raw.numel() else 11.0
    k = c1 + 5 * steps + states + 16
    R.check("y", y, ry, my, k + 8)
    R.check("state", so, rs, ms, k)
    if g is None:
        return
    R.check("du", g.u, rg["u"], mg["u"], 2 * k)
    sig = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    R.check("ddelta", g.delta, rg["delta"], mag_dt * sig, 2 * k + c1)
    R.check("dA", g.A, rg["A"], mg["A"].abs(), 2 * k + items * steps)
    R.check("dB", g.B, rg["B"], mg["B"], 2 * k + ch)
    R.check("dC", g.C, rg["C"], mg["C"], 2 * k + ch)
    if g.D is not None:
        R.check("dD", g.D, rg["D"], mg["D"], 16 + items * steps)
    if g.delta_bias is not None:
        R.check("ddelta_bias", g.delta_bias, rg["delta_bias"], (mag_dt * sig).sum((0, 1)), 2 * k + c1 + items * steps)
    if g.z is not None:
        # dy v silu'(z): silu' within 1.1 and good to 8 half steps of 1 + |z|
        mv = my.detach() / torch.clamp(sil, min=1e-30)
        R.check("dz", g.z, rg["z"], absd(dy) * mv * (1 + zz.abs()), k + 16)
    if g.state is not None:
        R.check("dstate", g.state, rg["state"], mg["state"], 2 * k)
    for n in names:
        assert (getattr(g, n) is None) == (a[n] is None), n



# ---- one frame at a time against the whole ---------------------------------------------------------------------------------

def stream_case(dev, items, steps, ch, groups, states, dtype, seed=5):
    """frames one by one, with the states carried in place, against one call: the convolution bit for bit, the scan within the
    bounds of both"""
    m = Make(dev, seed, dtype)
    x = m.n(items, steps, ch)
    w, b = m.n(ch, 4, f32=True, scale=0.5), m.n(ch, f32=True, scale=0.2)
    s0 = m.n(items, 3, ch)
    s = s0.clone()
    whole = scan.causal_conv(x, w, b, act="silu", state=s0)
    parts = torch.stack([scan.causal_conv_step(x[:, t], s, w, b, act="silu") for t in range(steps)], 1)
    assert torch.equal(whole, parts)
    assert torch.equal(s, torch.cat([s0, x], 1)[:, -3:])
    a = scan_inputs(m, items, steps, ch, groups, states, True, True, True, True, True)
    h = a["state"].clone()
    ys = []
    for t in range(steps):
        ys.append(scan.selective_scan_step(a["u"][:, t], a["delta"][:, t], a["A"], a["B"][:, t], a["C"][:, t], h, D=a["D"],
                                           z=a["z"][:, t], delta_bias=a["delta_bias"], softplus=True))
    scan_check(a, None, True, a["u"], torch.zeros_like(h), torch.stack(ys, 1), h, None)


# ---- gradients against differences -----------------------------------------------------------------------------------------

def difference(name, value, exact, point, grad, direction, h):
    """The directional derivative by central differences.  `value` (the kernels, float32) and `exact` (64 bits) are the loss at
    a point; their differences at the same h have the same truncation, so they may differ by rounding alone: each loss is good
    to r = |loss terms| k u, divided by h.  The gradient is held to the exact difference, whose truncation is 4/3 of what halving
    h changes."""
    up = [p + h * d for p, d in zip(point, direction)]
    down = [p - h * d for p, d in zip(point, direction)]
    (lu, mu), (ld, _) = value(up), value(down)
    got = (lu - ld) / (2 * h)

    def central(step):
        f = [exact([p.double() + s * step * d.double() for p, d in zip(point, direction)]) for s in (1, -1)]
        return (f[0] - f[1]) / (2 * step)

    ref, half = central(h), central(h / 2)
    rounding = mu * 400 * R.U / h
    assert abs(got - ref) <= rounding, (name, got, ref, rounding)
    along = sum(float((g.double() * d.double()).sum()) for g, d in zip(grad, direction))
    truncation = abs(ref - half) * 4 / 3
    assert abs(along - ref) <= 2 * truncation + rounding, (name, along, ref, truncation, rounding)


def difference_cases(dev):
    m = Make(dev, 11, "f32")
    x, w, b, dy = m.n(2, 7, 12), m.n(12, f32=True), m.n(12, f32=True), m.n(2, 7, 12)
    c64 = dy.cpu().double()
    y, st = norm.group_norm(x, 3, w, b, act="silu", want_stats=True)
    g = norm.group_norm_grad(dy, x, st, 3, w, b, act="silu")

    def loss(y):
        t = (y.cpu().double() * c64)
        return float(t.sum()), float(t.abs().sum())

    difference("norm", lambda p: loss(norm.group_norm(p[0], 3, p[1], p[2], act="silu")),
               lambda p: float((R.norm(p[0].cpu(), 3, p[1].cpu(), p[2].cpu(), 1e-5, "silu", None)[0] * c64).sum()),
               [x, w, b], g, [m.n(2, 7, 12), m.n(12), m.n(12)], 2.0 ** -6)
    cw, cb, s = m.n(12, 3), m.n(12), m.n(2, 2, 12)
    g = scan.causal_conv_grad(dy, x, cw, cb, act="silu", state=s)
    difference("conv", lambda p: loss(scan.causal_conv(p[0], p[1], p[2], act="silu", state=p[3])),
               lambda p: float((R.conv(*[t.cpu() for t in p[:3]], "silu", p[3].cpu(), None)[0] * c64).sum()),
               [x, cw, cb, s], g, [m.n(2, 7, 12), m.n(12, 3), m.n(12), m.n(2, 2, 12)], 2.0 ** -6)
    a = scan_inputs(m, 2, 7, 12, 2, 4, True, True, True, True, True)
    names = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")

    def run(p, keep=False):
        q = dict(zip(names, p))
        return scan.selective_scan(q["u"], q["delta"], q["A"], q["B"], q["C"], D=q["D"], z=q["z"], delta_bias=q["delta_bias"],
                                   softplus=True, state=q["state"], keep=keep)

    def ref(p):
        q = dict(zip(names, [t.cpu() for t in p]))
        return float((R.scan(q["u"], q["delta"], q["A"], q["B"], q["C"], q["D"], q["z"], q["delta_bias"], True, q["state"], None)[0]
                      * c64).sum())

    point = [a[n] for n in names]
    _, kept = run(point, True)
    g = scan.selective_scan_grad(dy, a["u"], a["delta"], a["A"], a["B"], a["C"], kept, D=a["D"], z=a["z"],
                                 delta_bias=a["delta_bias"], softplus=True, state=a["state"])
    difference("scan", lambda p: loss(run(p)), ref, point, g, [m.n(*t.shape) for t in point], 2.0 ** -7)
