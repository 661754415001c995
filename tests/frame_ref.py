"""Plain 64-bit implementations of the feature-map and frame-sequence operators (group norm with an activation, causal
convolution, selective scan), written from their definitions with gradients by torch's autograd in float64, and the bounds the
tests hold the kernels to.

Bounds.  u = 2^-24 is half a step of float32, r half a step of the output's type (r = 0 where the output is float32: its own
rounding is counted in the chain).  A kernel's value is  |got - ref| <= r |ref| + k u M + tiny,  where M is the same formula
with every term's absolute value (what a rounding error can be proportional to) and k counts the roundings of the longest
chain that leads to the value.  `tiny` is the smallest step of the type near zero (subnormals)."""
import math

import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}


def check(name, got, ref, mag, k):
    """|got - ref| <= half a step |ref| + k u mag, element by element"""
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    if got.numel() == 0:
        return
    g, ref, mag = got.detach().cpu().double(), ref.detach().double(), mag.detach().double()
    assert torch.isfinite(g).all(), "%s: not finite" % name
    tol = HALF_STEP[got.dtype] * ref.abs() + (1 + HALF_STEP[got.dtype]) * k * U * mag + TINY[got.dtype]
    over = (g - ref).abs() / tol
    i = int(over.argmax())
    assert over.max() <= 1, "%s: element %d: got %.9g, want %.9g, %.2f times the bound" % (
        name, i, g.reshape(-1)[i], ref.reshape(-1)[i], over.max())


def act(p, name):
    if name == "relu":
        return p * (p > 0)
    if name == "silu":
        return p / (1 + torch.exp(-p))
    if name == "gelu":
        return 0.5 * p * (1 + torch.erf(p / math.sqrt(2)))
    return p


def lens_of(lengths, items, rows):
    return [rows] * items if lengths is None else [min(max(int(v), 0), rows) for v in lengths]


def leaf(t):
    return None if t is None else t.detach().cpu().double().requires_grad_(True)


def grads(outs, cots, leaves):
    live = [t for t in leaves if t is not None]
    pairs = [(o, c) for o, c in zip(outs, cots) if c is not None and o.requires_grad]
    got = torch.autograd.grad([o for o, _ in pairs], live, [c.detach().cpu().double() for _, c in pairs], allow_unused=True) if pairs else [None] * len(live)
    it = iter([g if g is not None else torch.zeros_like(t) for g, t in zip(got, live)])
    return [next(it) if t is not None else None for t in leaves]


# ---- group norm ----------------------------------------------------------------------------------------------------------

def norm(x, groups, weight, bias, eps, name, lengths):
    """(y, stats); x etc. float64 leaves"""
    items, rows, ch = x.shape
    ys, stats = [], []
    for b, n in enumerate(lens_of(lengths, items, rows)):
        v = x[b, :n].reshape(n, groups, ch // groups)
        cnt = max(1, n * (ch // groups))
        m = v.sum((0, 2), keepdim=True) / cnt
        var = ((v - m) ** 2).sum((0, 2), keepdim=True) / cnt
        r = 1 / torch.sqrt(var + eps)
        p = ((v - m) * r).reshape(n, ch)
        if weight is not None:
            p = p * weight
        if bias is not None:
            p = p + bias
        ys.append(torch.cat([act(p, name), x.new_zeros(rows - n, ch)]))
        stats.append(torch.stack([m.reshape(groups), r.reshape(groups)], -1))
    if not ys:
        return x.new_zeros(0, rows, ch), x.new_zeros(0, groups, 2)
    return torch.stack(ys), torch.stack(stats)


# ---- causal convolution --------------------------------------------------------------------------------------------------

def conv(x, weight, bias, name, state, lengths):
    items, steps, ch = x.shape
    taps = weight.shape[1]
    ys, states = [], []
    for b, n in enumerate(lens_of(lengths, items, steps)):
        e = torch.cat([state[b] if state is not None else x.new_zeros(taps - 1, ch), x[b, :n]])
        p = (bias if bias is not None else x.new_zeros(ch)).expand(n, ch)
        for k in range(taps):
            p = p + e[k:k + n] * weight[:, k]
        ys.append(torch.cat([act(p, name), x.new_zeros(steps - n, ch)]))
        states.append(e[n:])
    return torch.stack(ys), torch.stack(states)


# ---- selective scan ------------------------------------------------------------------------------------------------------

def scan(u, delta, A, B, C, D, z, bias, softplus, state, lengths, plain_gate=None, decay=None):
    """(y, state behind the last frame).  The magnitude run gives `plain_gate`, factors in place of silu(z), and `decay`, step
    sizes of their own for the decay"""
    items, steps, ch = u.shape
    rep = ch // B.shape[2]
    lens = torch.tensor(lens_of(lengths, items, steps))
    h = state if state is not None else u.new_zeros(items, ch, A.shape[1])
    ys = []
    for t in range(steps):
        on = (lens > t)[:, None]
        raw = delta[:, t] + (bias if bias is not None else 0.0)
        dt = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
        b, c = B[:, t].repeat_interleave(rep, 1), C[:, t].repeat_interleave(rep, 1)
        new = torch.exp((dt if decay is None else decay[:, t])[..., None] * A) * h + (dt * u[:, t])[..., None] * b
        h = torch.where(on[..., None], new, h)
        y = (h * c).sum(-1)
        if D is not None:
            y = y + D * u[:, t]
        if plain_gate is not None:
            y = y * plain_gate[:, t]
        elif z is not None:
            y = y * z[:, t] / (1 + torch.exp(-z[:, t]))
        ys.append(torch.where(on, y, torch.zeros_like(y)))
    return (torch.stack(ys, 1) if ys else u.new_zeros(u.shape)), h
