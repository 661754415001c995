"""Group norm held to bounds near its real error, run by test_norm_widths.py on the CPU thread emulator and on the GPU.

The gradients of the reference are the formula's, in 64 bits (and the formula is held to autograd's).  Inputs: dy has a mean and
a part along xh, so that the two group means in dx, and the channels' sums, are as large as the rest of the result.

Bounds, element by element, first order in u = 2^-24; per group D = max x - min x, s = std, T = rows + channels of the group + 32,
which no chain of additions of a statistic is longer than, S = T + items for the sums over the batch:
  mean   em = (T + 2) u (D + mean |x|) + u |m|     (terms x - k of at most D around a value k of the group, or x itself)
  1/std  er = half of  (T + 4) u (1 + D^2 / s^2) + (em / s)^2,  and 3 u   (relative; squares of at most D^2 where their mean is s^2)
  xh     em / s + |xh| (er + 4 u)
  p      |w| exh + 4 u (|xh w| + |b|)
  y      1.13 ep + u (8 + 2 |p|) |p|               (|act'| <= 1.13; exponential, reciprocal, products)
  q      |dy| (0.8 ep + 1.2 u (12 + 4 |p|))        (|act''| <= 0.8, |act'| <= 1.2)
and the sums by the chain rule, each with S u times the sum of its terms' absolute values.  Results of 16 bits add half a step.
relu's slope jumps: dy is 0 where |p| is below its own bound, so that no element depends on the side."""
import torch

import frame_ref as R
from auditory_amd import norm
from frame_cases import Make, poison

U = R.U


def slope(p, name):
    if name == "relu":
        return (p > 0).double()
    if name == "silu":
        q = torch.sigmoid(p)
        return q * (1 + p * (1 - q))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(p / 2 ** 0.5)) + p * torch.exp(-0.5 * p * p) / (2 * torch.pi) ** 0.5
    return torch.ones_like(p)


class Exact:
    """values, gradients and their bounds in 64 bits; `plant` leaves a part of the formulas out (to see that the bounds notice)"""

    def __init__(self, x, dy, groups, w, b, eps, name, lengths, plant=None):
        items, rows, ch = x.shape
        cg = ch // groups
        n = torch.tensor(R.lens_of(lengths, items, rows), dtype=torch.float64)[:, None, None, None]
        self.on = on = (torch.arange(rows)[None, :, None, None] < n).double()
        x, dy = (t.detach().cpu().double().reshape(items, rows, groups, cg) * on for t in (x, dy))
        w = torch.ones(ch, dtype=torch.float64) if w is None else w.detach().cpu().double()
        b = torch.zeros(ch, dtype=torch.float64) if b is None else b.detach().cpu().double()
        w, b = w.reshape(groups, cg), b.reshape(groups, cg)
        cnt = torch.clamp(n * cg, min=1)

        def mean(t):
            return (t * on).sum((1, 3), keepdim=True) / cnt

        m = mean(x)
        r = 1 / torch.sqrt(mean((x - m) ** 2) + eps)
        xh = (x - m) * r * on
        p = xh * w + b
        # how far p may be off, and with it where relu's side is open
        hi = torch.where(on > 0, x, -torch.inf).amax((1, 3), keepdim=True)
        lo = torch.where(on > 0, x, torch.inf).amin((1, 3), keepdim=True)
        D = torch.where(n > 0, hi - lo, 0.0)
        T = rows + cg + 32
        S = T + items
        em = (T + 2) * U * (D + mean(x.abs())) + U * m.abs()
        er = 0.5 * ((T + 4) * U * (1 + (D * r) ** 2) + (em * r) ** 2) + 3 * U
        exh = em * r + xh.abs() * (er + 4 * U)
        ep = w.abs() * exh + 4 * U * ((xh * w).abs() + b.abs())
        self.open_side = ((p.abs() <= 4 * ep) & (on > 0)).reshape(items, rows, ch)
        y = R.act(p, name) * on
        ey = (1.13 * ep + U * (8 + 2 * p.abs()) * p.abs()) * on
        q = dy * slope(p, name) * on
        eq = dy.abs() * (0.8 * ep + 1.2 * U * (12 + 4 * p.abs())) * on
        if plant == "rows":  # the last rows are left out of the sums
            keep = (torch.arange(rows)[None, :, None, None] < torch.floor(n * 0.75)).double()
        else:
            keep = on
        sums = lambda t: (t * keep).sum((0, 1))  # noqa: E731
        dw, db = sums(q * xh), sums(q)
        edw = sums(eq * xh.abs() + q.abs() * exh + 2 * U * (q * xh).abs()) + S * U * sums((q * xh).abs())
        edb = sums(eq) + S * U * sums(q.abs())
        t, et = q * w, eq * w.abs() + U * (q * w).abs()
        A, B = mean(t * keep), mean(t * xh * keep)
        eA = mean(et) + S * U * mean(t.abs())
        eB = mean(et * xh.abs() + t.abs() * exh) + (S + 4) * U * mean((t * xh).abs())
        if plant == "mean of t":
            A = A * 0
        if plant == "mean of t xh":
            B = B * 0
        dx = r * (t - A - xh * B) * on
        edx = (r * (et + eA + xh.abs() * eB + B.abs() * exh + 4 * U * (t.abs() + A.abs() + (xh * B).abs())) + dx.abs() * er) * on
        flat = lambda v: v.reshape(items, rows, ch)  # noqa: E731
        if plant == "dweight":
            dw = dw * 0
        if plant == "dbias":
            db = db * 0
        if plant == "variance":  # of one value fewer
            y = R.act(xh * torch.sqrt(torch.clamp(cnt - 1, min=1) / cnt) * w + b, name) * on
        col = lambda v: v[:, 0, :, 0]  # noqa: E731
        self.y, self.ey = flat(y), flat(ey)
        self.mean, self.emean, self.rstd, self.erstd = col(m), col(em), col(r), col(r * er)
        self.dx, self.edx = flat(dx), flat(edx)
        self.dw, self.edw, self.db, self.edb = dw.reshape(ch), edw.reshape(ch), db.reshape(ch), edb.reshape(ch)

    def near(self, name, got, ref, bound):
        assert got.shape == ref.shape, name
        g = got.detach().cpu().double()
        assert torch.isfinite(g).all(), "%s: not finite" % name
        half = R.HALF_STEP[got.dtype]
        tol = half * ref.abs() + (1 + half) * 1.02 * bound + R.TINY[got.dtype]  # (second order: 2 % at most)
        over = (g - ref).abs() / tol
        assert over.numel() == 0 or over.max() <= 1, "%s: %.2f times the bound at %d" % (name, over.max(), int(over.argmax()))
        # a bound that lets a wrong result through is no check
        rms = float((ref ** 2).mean().sqrt()) if ref.numel() else 0.0
        assert not rms or float(bound.median()) <= 0.03 * rms, "%s: the bound (%.3g) is not below the values (%.3g)" % (
            name, bound.median(), rms)


def inputs(dev, items, rows, ch, groups, dtype, name, affine, lens, pad, seed=0):
    m = Make(dev, 1000 + seed + 7 * items * rows + ch, dtype)
    x = m.n(items, rows, ch, scale=1.5, shift=0.4)
    dy = (0.7 + 0.5 * (x.float() - 0.4) / 1.5 + 0.5 * m.n(items, rows, ch, f32=True)).to(m.t)
    w, b = (m.n(ch, f32=True, scale=0.3, shift=1.0), m.n(ch, f32=True, scale=0.3)) if affine else (None, None)
    lengths = m.lengths(lens, items, rows)
    if name == "relu":
        side = Exact(x, dy, groups, w, b, 1e-5, name, lengths).open_side
        dy = torch.where(side.to(dev), torch.zeros_like(dy), dy)
    xs, ds = (m.strided(x, pad), m.strided(dy, pad)) if pad else (poison(x, lengths), poison(dy, lengths))
    return x, dy, w, b, lengths, xs, ds


def run(dev, items, rows, ch, groups, dtype, name, affine, lens, pad):
    x, dy, w, b, lengths, xs, ds = inputs(dev, items, rows, ch, groups, dtype, name, affine, lens, pad)
    y, stats = norm.group_norm(xs, groups, w, b, act=name, lengths=lengths, want_stats=True)
    dx, dw, db = norm.group_norm_grad(ds, xs, stats, groups, w, b, act=name, lengths=lengths)
    if dev != "cpu":  # (the emulator's runs are slow, and never differ by timing)
        again = norm.group_norm_grad(ds, xs, stats, groups, w, b, act=name, lengths=lengths)
        assert torch.equal(y, norm.group_norm(xs, groups, w, b, act=name, lengths=lengths))
        assert all(p is None and q is None or torch.equal(p, q) for p, q in zip((dx, dw, db), again))
    return (x, dy, groups, w, b, 1e-5, name, lengths), (y, stats, dx, dw, db)


def held(args, got, plant=None):
    e = Exact(*args, plant=plant)
    y, stats, dx, dw, db = got
    e.near("y", y, e.y, e.ey)
    e.near("mean", stats[..., 0], e.mean, e.emean)
    e.near("rstd", stats[..., 1], e.rstd, e.erstd)
    e.near("dx", dx, e.dx, e.edx)
    if args[3] is not None:
        e.near("dweight", dw, e.dw, e.edw)
        e.near("dbias", db, e.db, e.edb)


def case(dev, *c):
    held(*run(dev, *c))


# (items, rows, channels, groups, type, activation, affine, lengths, row padding).  What a row's packs (channels / elements an
# access) are to the 256 threads of a chunk and the 512 of an item decides how many rows a workgroup has side by side: widths
# beside the fitting ones, with one pack left over, a few, exactly half a sweep, and nearly a whole one
WIDTHS = {257: 1, 301: 7, 384: 6, 513: 27, 514: 2, 602: 14, 768: 24, 769: 1, 1100: 44, 1300: 13}
WIDE = []
for _i, (_c, _g) in enumerate(WIDTHS.items()):
    for _k, _t in enumerate(("f32", "bf16", "f16")):
        _act, _pad = ("silu", "gelu", "none", "relu")[(_i + _k) % 4], 3 if _c in (384, 768) else 0
        WIDE.append((2, 6, _c, _g, _t, _act, True, None, _pad))                          # an item in one workgroup
        WIDE.append((2, 40 if _t == "f32" else 70, _c, _g, _t, _act, True, "mixed" if _k == 1 else None, _pad))  # over several
WIDE += [
    (1, 3, 2052, 4, "f32", "silu", True, None, 0),      # 513 packs of four: one left over behind 512 threads
    (1, 7, 2056, 8, "bf16", "silu", True, None, 0),     # 257 packs of eight in one workgroup
    (2, 9, 2056, 8, "bf16", "silu", True, None, 0),     # ... over several: one left over behind 256 threads
    (2, 33, 1028, 4, "f16", "gelu", True, "mixed", 0),  # 257 packs of four
    (2, 9, 1540, 4, "bf16", "silu", True, None, 5),     # an odd distance between the rows: one element at a time
    (1, 2, 4095, 5, "f32", "silu", True, None, 0),
    (2, 3, 4096, 64, "f32", "silu", False, None, 0),
]
# (on the emulator: every width on both sides, in one of the types)
WIDE_EMUL = [c for c in WIDE if c[2] not in WIDTHS or c[4] == ("f32", "bf16", "f16")[list(WIDTHS).index(c[2]) % 3]]
# the other widths, every route: values held in registers, an item read twice, chunks joined by all or by a kernel of their own
ROUTES = [
    (3, 7, 40, 8, "f32", "silu", True, "mixed", 0),
    (2, 33, 24, 24, "f16", "silu", True, None, 0),
    (2, 300, 16, 2, "f32", "relu", True, None, 0),       # 19 KB: read twice
    (2, 600, 32, 4, "f32", "silu", True, "mixed", 0),    # chunks
    (2, 600, 16, 2, "f32", "gelu", True, None, 3),
    (1, 500, 33, 3, "bf16", "silu", True, None, 0),
    (3, 777, 132, 12, "f16", "gelu", True, "mixed", 0),
    (1, 100, 1024, 1024, "f32", "none", True, None, 0),  # many groups
    (9, 150, 64, 4, "bf16", "relu", True, "mixed", 0),
]
PLANTED = ["mean of t", "mean of t xh", "dweight", "dbias", "rows"]
