"""Workloads of the feature-map and frame-sequence operators: group normalisation with an activation (channels last), the
short causal convolution over frames and the selective state space scan over frames, for whole utterances and for one
frame at a time.

A case names the operator, what is run of it ("apply": the values; "train": values and gradients; "step": one frame with
its carried state) and its sizes.  `run` computes it in plain torch operations, or with the library's kernels where `own`
is true."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_DEV = "cuda:0"


def listed():
    return [
        # the gabor maps of 256 one-second utterances (11 x 32 positions, 2 polarities x 8 filters), one group a polarity
        dict(name="norm_gabor_maps", op="norm", mode="apply", dtype="f32", B=256, S=352, C=16, G=2, act="relu", ragged=False),
        # one utterance's mel frames behind a microphone: latency
        dict(name="norm_one_utterance", op="norm", mode="apply", dtype="f32", B=1, S=98, C=40, G=8, act="silu", ragged=False),
        # an encoder's feature maps in training
        dict(name="norm_train_maps", op="norm", mode="train", dtype="bf16", B=16, S=4096, C=512, G=32, act="silu", ragged=False),
        # a padded batch of utterances of different lengths, odd widths, in training
        dict(name="norm_train_ragged", op="norm", mode="train", dtype="f16", B=7, S=333, C=132, G=12, act="gelu", ragged=True),
        # the convolution in front of the scan over long utterances
        dict(name="conv_prompt", op="conv", mode="apply", dtype="bf16", B=8, L=2048, D=1536, K=4, act="silu", ragged=False),
        # 64 live streams, one frame each
        dict(name="conv_step", op="conv", mode="step", dtype="f16", B=64, L=1, D=1024, K=4, act="silu", ragged=False),
        # a padded batch in training
        dict(name="conv_train_ragged", op="conv", mode="train", dtype="f32", B=5, L=777, D=260, K=3, act="silu", ragged=True),
        # the scan over long utterances
        dict(name="scan_prompt", op="scan", mode="apply", dtype="bf16", B=8, L=2048, D=1536, N=16, G=1, gate=True, ragged=False),
        # one long recording: few rows, a long axis
        dict(name="scan_recording", op="scan", mode="apply", dtype="f32", B=1, L=8192, D=256, N=16, G=1, gate=True, ragged=False),
        # 64 live streams, one frame each
        dict(name="scan_step", op="scan", mode="step", dtype="bf16", B=64, L=1, D=1024, N=16, G=1, gate=True, ragged=False),
        # training on long utterances
        dict(name="scan_train", op="scan", mode="train", dtype="bf16", B=4, L=2048, D=1024, N=16, G=1, gate=True, ragged=False),
        # a padded batch of short utterances in training, two groups of input and output vectors, no gate
        dict(name="scan_train_ragged", op="scan", mode="train", dtype="f16", B=3, L=501, D=72, N=8, G=2, gate=False, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "conv", "scan"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        mode = rng.choice(["apply", "train"])
        cg = rng.choice([1, 2, 3, 4, 5, 8, 11, 16, 20, 32, 64])
        groups = _log(rng, 1, max(1, 1024 // cg))
        C = cg * groups
        B = _log(rng, 1, 256)
        least = -(-32 // cg)  # positions: a group holds 32 values at least
        S = _log(rng, least, max(least, min(8192, (1 << 24) // (B * C))))
        # (relu's gradient jumps at 0: a value next to it would be compared by its rounding)
        act = rng.choice(["none", "silu", "gelu"] if mode == "train" else ["none", "relu", "silu", "gelu"])
        return dict(op=op, mode=mode, dtype=dtype, B=B, S=S, C=C, G=groups, act=act, ragged=rng.random() < 0.4)
    if op == "conv":
        mode = rng.choice(["apply", "train", "step"])
        D = _log(rng, 8, 2048)
        B = _log(rng, 1, 256 if mode == "step" else 32)
        L = 1 if mode == "step" else _log(rng, 2, max(2, min(8192, (3 << 22) // (B * D))))
        return dict(op=op, mode=mode, dtype=dtype, B=B, L=L, D=D, K=rng.choice([2, 3, 4]), act=rng.choice(["none", "silu"]),
                    ragged=mode != "step" and rng.random() < 0.4)
    mode = rng.choice(["apply", "train", "step"])
    G = rng.choice([1, 1, 1, 2, 4])
    D = G * _log(rng, 8, 2048 // G)
    N = rng.choice([4, 8, 16, 16, 16, 24, 32])
    B = _log(rng, 1, 256 if mode == "step" else 32)
    most, wide = ((1 << 26), (3 << 21)) if mode == "train" else ((1 << 28), (3 << 22))
    L = 1 if mode == "step" else _log(rng, 2, max(2, min(8192, most // (B * D * N), wide // (B * D))))
    return dict(op=op, mode=mode, dtype=dtype, B=B, L=L, D=D, N=N, G=G, gate=rng.random() < 0.6,
                ragged=mode != "step" and rng.random() < 0.4)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    B = case["B"]
    if case["op"] == "norm":
        n = B * case["S"] * case["C"]
        train = case["mode"] == "train"
        return {"bytes": e * n * (5 if train else 2) + 8 * case["C"] * (2 if train else 1), "flops": n * (37 if train else 12)}
    n = B * case["L"] * case["D"]
    if case["op"] == "conv":
        K, st = case["K"], B * (case["K"] - 1) * case["D"] * e
        if case["mode"] == "train":
            return {"bytes": e * n * 5 + 8 * case["D"] * (K + 1) + 3 * st, "flops": n * (8 * K + 20)}
        return {"bytes": e * n * 2 + 4 * case["D"] * (K + 1) + 2 * st, "flops": n * (2 * K + 6)}
    N, bc, st = case["N"], 2 * B * case["L"] * case["G"] * case["N"] * e, 4 * B * case["D"] * case["N"]
    big = 4 if case["gate"] else 3
    if case["mode"] == "train":
        # the values (u, delta, z -> y), then the gradients (dy and the same again -> as many)
        return {"bytes": e * n * (3 * big - 1) + 3 * bc + 8 * case["D"] * (N + 2) + 3 * st, "flops": n * (24 * N + 60)}
    return {"bytes": e * n * big + bc + 4 * case["D"] * (N + 2) + 2 * st, "flops": n * (7 * N + 25)}


# ---- inputs -----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=_DEV)
    g.manual_seed(int(seed))
    t = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=_DEV, dtype=torch.float32)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=_DEV, dtype=torch.float32)

    s = {"case": case, "dtype": t, "lengths": None}
    B = case["B"]
    rows = case["S"] if case["op"] == "norm" else case["L"]
    if case["ragged"]:
        s["lengths"] = (uniform(B) * (rows + 1)).floor().clamp(max=rows).to(torch.int32)
        s["lengths"][0] = rows
    train = case["mode"] == "train"
    if case["op"] == "norm":
        C = case["C"]
        x = normal(B, rows, C)
        # filter responses are rectified (half of them zero); frame values sit around a level that differs by channel
        s["x"] = (x.clamp(min=0) if C == 16 else x * 1.7 + normal(C) - 1.5).to(t)
        s["weight"], s["bias"] = 1 + 0.2 * normal(C), 0.2 * normal(C)
        if train:
            s["dy"] = normal(B, rows, C).to(t)
        return s
    D = case["D"]
    if case["op"] == "conv":
        K = case["K"]
        s["x"] = normal(B, rows, D).to(t)
        s["weight"], s["bias"] = normal(D, K) / math.sqrt(K), 0.2 * normal(D)
        s["state"] = normal(B, K - 1, D).to(t)
        if train:
            s["dy"], s["dstate_out"] = normal(B, rows, D).to(t), normal(B, K - 1, D).to(t)
        return s
    N, G = case["N"], case["G"]
    v = normal(B, rows, D)
    s["u"] = (v * torch.sigmoid(v)).to(t)
    s["delta"] = (0.5 * normal(B, rows, D)).to(t)
    s["A"] = -(torch.arange(1, N + 1, device=_DEV, dtype=torch.float32) * (0.8 + 0.4 * uniform(D, 1)))
    step = torch.exp(uniform(D) * math.log(100.0) + math.log(1e-3))  # step sizes from 0.001 to 0.1
    s["delta_bias"] = step + torch.log(-torch.expm1(-step))
    s["B"], s["C"] = normal(B, rows, G, N).to(t), normal(B, rows, G, N).to(t)
    s["D"] = 1 + 0.1 * normal(D)
    s["z"] = normal(B, rows, D).to(t) if case["gate"] else None
    s["state"] = normal(B, D, N)
    if train:
        s["dy"], s["dstate_out"] = normal(B, rows, D).to(t), normal(B, D, N)
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"norm": _plain_norm, "conv": _plain_conv, "scan": _plain_scan}[state["case"]["op"]](state)


def _run_own(s):
    from auditory_amd import norm, scan
    c = s["case"]
    if c["op"] == "norm":
        if c["mode"] == "apply":
            return norm.group_norm(s["x"], c["G"], s["weight"], s["bias"], act=c["act"], lengths=s["lengths"])
        y, stats = norm.group_norm(s["x"], c["G"], s["weight"], s["bias"], act=c["act"], lengths=s["lengths"], want_stats=True)
        dx, dweight, dbias = norm.group_norm_grad(s["dy"], s["x"], stats, c["G"], s["weight"], s["bias"], act=c["act"],
                                                  lengths=s["lengths"])
        return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}
    if c["op"] == "conv":
        state_out = torch.empty_like(s["state"])
        if c["mode"] == "step":
            y = scan.causal_conv_step(s["x"][:, 0], s["state"], s["weight"], s["bias"], act=c["act"], state_out=state_out)
            return {"y": y, "state": state_out}
        y = scan.causal_conv(s["x"], s["weight"], s["bias"], act=c["act"], state=s["state"], lengths=s["lengths"],
                             state_out=state_out)
        out = {"y": y, "state": state_out}
        if c["mode"] == "train":
            g = scan.causal_conv_grad(s["dy"], s["x"], s["weight"], s["bias"], act=c["act"], state=s["state"],
                                      lengths=s["lengths"], dstate_out=s["dstate_out"])
            out.update(dx=g.x, dweight=g.weight, dbias=g.bias, dstate=g.state)
        return out
    state_out = torch.empty_like(s["state"])
    if c["mode"] == "step":
        z = s["z"][:, 0] if s["z"] is not None else None
        y = scan.selective_scan_step(s["u"][:, 0], s["delta"][:, 0], s["A"], s["B"][:, 0], s["C"][:, 0], s["state"], D=s["D"],
                                     z=z, delta_bias=s["delta_bias"], softplus=True, state_out=state_out)
        return {"y": y, "state": state_out}
    if c["mode"] == "apply":
        y = scan.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                                softplus=True, state=s["state"], lengths=s["lengths"], state_out=state_out)
        return {"y": y, "state": state_out}
    y, kept = scan.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], delta_bias=s["delta_bias"],
                                  softplus=True, state=s["state"], lengths=s["lengths"], state_out=state_out, keep=True)
    g = scan.selective_scan_grad(s["dy"], s["u"], s["delta"], s["A"], s["B"], s["C"], kept, D=s["D"], z=s["z"],
                                 delta_bias=s["delta_bias"], softplus=True, state=s["state"], lengths=s["lengths"],
                                 dstate_out=s["dstate_out"])
    return {"y": y, "state": state_out, "du": g.u, "ddelta": g.delta, "dA": g.A, "dB": g.B, "dC": g.C, "dD": g.D, "dz": g.z,
            "ddelta_bias": g.delta_bias, "dstate": g.state}


def _live(s, rows):
    """[B, rows, 1] truth values: the rows that an utterance has"""
    if s["lengths"] is None:
        return None
    return (torch.arange(rows, device=_DEV)[None, :] < s["lengths"][:, None])[:, :, None]


def _act(p, name):
    if name == "relu":
        return torch.clamp(p, min=0)
    if name == "silu":
        return p * torch.sigmoid(p)
    if name == "gelu":
        return 0.5 * p * (1 + torch.erf(p * math.sqrt(0.5)))
    return p


def _act_grad(p, name):
    if name == "relu":
        return (p > 0).to(p.dtype)
    if name == "silu":
        q = torch.sigmoid(p)
        return q * (1 + p * (1 - q))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(p * math.sqrt(0.5))) + p * torch.exp(-0.5 * p * p) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(p)


def _plain_norm(s):
    c, t = s["case"], s["dtype"]
    B, S, C, G = c["B"], c["S"], c["C"], c["G"]
    live = _live(s, S)
    x = s["x"].float()
    if live is None:
        count = float(S * (C // G))
    else:
        x = torch.where(live, x, 0.0)
        count = (s["lengths"].clamp(min=1).float() * (C // G))[:, None, None, None]
    xg = x.view(B, S, G, C // G)
    off = xg - xg.sum(dim=(1, 3), keepdim=True) / count
    if live is not None:
        off = torch.where(live[..., None], off, 0.0)
    r = torch.rsqrt((off * off).sum(dim=(1, 3), keepdim=True) / count + 1e-5)
    xh = off * r
    p = xh.view(B, S, C) * s["weight"] + s["bias"]
    y = _act(p, c["act"])
    if live is not None:
        y = torch.where(live, y, 0.0)
    y = y.to(t)
    if c["mode"] == "apply":
        return y
    q = s["dy"].float() * _act_grad(p, c["act"])
    if live is not None:
        q = torch.where(live, q, 0.0)
    dweight, dbias = (q * xh.view(B, S, C)).sum(dim=(0, 1)), q.sum(dim=(0, 1))
    w = (q * s["weight"]).view(B, S, G, C // G)
    dx = r * (w - w.sum(dim=(1, 3), keepdim=True) / count - xh * ((w * xh).sum(dim=(1, 3), keepdim=True) / count))
    dx = dx.reshape(B, S, C)
    if live is not None:
        dx = torch.where(live, dx, 0.0)
    return {"y": y, "dx": dx.to(t), "dweight": dweight, "dbias": dbias}


def _plain_conv(s):
    c, t = s["case"], s["dtype"]
    B, L, D, K = c["B"], c["L"], c["D"], c["K"]
    live = _live(s, L)
    e = torch.cat([s["state"], s["x"]], 1)
    if live is not None:
        e = torch.where(torch.cat([torch.ones_like(live[:, :1]).expand(B, K - 1, 1), live], 1), e, 0.0)
        last = (s["lengths"].long()[:, None] + torch.arange(K - 1, device=_DEV))[:, :, None].expand(B, K - 1, D)
        state = torch.gather(e, 1, last)
    else:
        state = e[:, L:].contiguous()
    ef = e.float()
    win = ef.unfold(1, K, 1)  # [B, L, D, K]
    p = (win * s["weight"]).sum(-1) + s["bias"]
    y = _act(p, c["act"])
    if live is not None:
        y = torch.where(live, y, 0.0)
    out = {"y": y.to(t), "state": state}
    if c["mode"] == "step":
        out["y"] = out["y"][:, 0]
    if c["mode"] != "train":
        return out
    q = s["dy"].float() * _act_grad(p, c["act"])
    if live is not None:
        q = torch.where(live, q, 0.0)
    pad = torch.zeros((B, K - 1, D), device=_DEV)
    qwin = torch.cat([pad, q, pad], 1).unfold(1, K, 1)  # [B, L + K - 1, D, K]: q_{j-K+1} ... q_j
    de = (qwin * s["weight"].flip(1)).sum(-1)
    ds = s["dstate_out"].float()
    if live is not None:
        de = de.scatter_add(1, last, ds)
    else:
        de = torch.cat([de[:, :L], de[:, L:] + ds], 1)
    out.update(dx=de[:, K - 1:].to(t), dweight=(q[..., None] * win).sum(dim=(0, 1)), dbias=q.sum(dim=(0, 1)),
               dstate=de[:, :K - 1].to(t))
    return out


def _recur(a, x):
    """h_t = a_t h_{t-1} + x_t along axis 1, from h = 0: neighbours are joined, the half as long recurrence is solved, and the
    values between are filled in"""
    L = a.shape[1]
    if L == 1:
        return x
    m = 2 * (L // 2)
    odd = _recur(a[:, 1:m:2] * a[:, 0:m:2], torch.addcmul(x[:, 1:m:2], a[:, 1:m:2], x[:, 0:m:2]))
    h = torch.empty_like(x)
    h[:, 0] = x[:, 0]
    h[:, 1::2] = odd
    if L > 2:
        n = a[:, 2::2].shape[1]
        h[:, 2::2] = torch.addcmul(x[:, 2::2], a[:, 2::2], odd[:, :n])
    return h


def _plain_scan(s):
    c, t = s["case"], s["dtype"]
    B, L, D, N, G = c["B"], c["L"], c["D"], c["N"], c["G"]
    live = _live(s, L)
    raw = s["delta"].float() + s["delta_bias"]
    dt = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    if live is not None:
        dt = torch.where(live, dt, 0.0)  # a step of size 0 keeps the state
    u = s["u"].float()
    Bm = s["B"].float()[:, :, :, None].expand(B, L, G, D // G, N).reshape(B, L, D, N)
    Cm = s["C"].float()[:, :, :, None].expand(B, L, G, D // G, N).reshape(B, L, D, N)
    a = torch.exp(dt[..., None] * s["A"])
    x = (dt * u)[..., None] * Bm
    x[:, 0] += a[:, 0] * s["state"]
    h = _recur(a, x)
    del x
    v = (h * Cm).sum(-1) + s["D"] * u
    if c["gate"]:
        z = s["z"].float()
        sz = torch.sigmoid(z)
        y = v * (z * sz)
    else:
        y = v
    if live is not None:
        y = torch.where(live, y, 0.0)
    out = {"y": y.to(t), "state": h[:, -1].contiguous()}
    if c["mode"] == "step":
        out["y"] = out["y"][:, 0]
    if c["mode"] != "train":
        return out
    dy = s["dy"].float()
    if live is not None:
        dy = torch.where(live, dy, 0.0)
    f = dy * (z * sz) if c["gate"] else dy
    gx = f[..., None] * Cm
    gx[:, -1] += s["dstate_out"]
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _recur(after.flip(1), gx.flip(1)).flip(1)
    del gx, after
    before = torch.cat([s["state"][:, None], h[:, :-1]], 1)
    gah = g * a * before
    ddt = (gah * s["A"]).sum(-1) + (g * Bm).sum(-1) * u
    if live is not None:
        ddt = torch.where(live, ddt, 0.0)
    ddelta = ddt * torch.sigmoid(raw)
    out.update(du=((g * Bm).sum(-1) * dt + s["D"] * f).to(t), ddelta=ddelta.to(t), dA=(gah * dt[..., None]).sum(dim=(0, 1)),
               dB=(g * (dt * u)[..., None]).view(B, L, G, D // G, N).sum(3).to(t),
               dC=(f[..., None] * h).view(B, L, G, D // G, N).sum(3).to(t), dD=(f * u).sum(dim=(0, 1)),
               dz=(dy * v * sz * (1 + z * (1 - sz))).to(t) if c["gate"] else None,
               ddelta_bias=ddelta.sum(dim=(0, 1)), dstate=g[:, 0] * a[:, 0])
    return out


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    with torch.enable_grad():
        return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](s, case)


def _f64_act(p, name):
    return {"none": lambda: p, "relu": lambda: torch.relu(p), "silu": lambda: p / (1 + torch.exp(-p)),
            "gelu": lambda: p * 0.5 * torch.erfc(-p / math.sqrt(2))}[name]()


def _lens(s, rows, B):
    return [rows] * B if s["lengths"] is None else [int(v) for v in s["lengths"].cpu()]


def _leaf(s, *names):
    return [s[n].requires_grad_(True) for n in names]


def _exact_norm(s, c):
    B, S, C, G = c["B"], c["S"], c["C"], c["G"]
    train = c["mode"] == "train"
    if train:
        leaves = _leaf(s, "x", "weight", "bias")
    rows = []
    for b, n in enumerate(_lens(s, S, B)):
        if n:
            x = s["x"][b, :n].reshape(n, G, C // G)
            var, mean = torch.var_mean(x, dim=(0, 2), correction=0, keepdim=True)
            p = ((x - mean) / torch.sqrt(var + 1e-5)).reshape(n, C) * s["weight"] + s["bias"]
            rows.append(torch.cat([_f64_act(p, c["act"]), p.new_zeros(S - n, C)]))
        else:
            rows.append(s["x"].new_zeros(S, C))
    y = torch.stack(rows)
    if not train:
        return y
    dx, dw, db = torch.autograd.grad(y, leaves, s["dy"])
    return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}


def _exact_conv(s, c):
    B, L, D, K = c["B"], c["L"], c["D"], c["K"]
    train = c["mode"] == "train"
    if train:
        leaves = _leaf(s, "x", "weight", "bias", "state")
    ys, states = [], []
    for b, n in enumerate(_lens(s, L, B)):
        e = torch.cat([s["state"][b], s["x"][b, :n]])
        p = s["bias"].expand(n, D)
        for k in range(K):
            p = p + e[k:k + n] * s["weight"][:, k]
        ys.append(torch.cat([_f64_act(p, c["act"]), p.new_zeros(L - n, D)]))
        states.append(e[n:])
    y, state = torch.stack(ys), torch.stack(states)
    out = {"y": y.detach()[:, 0] if c["mode"] == "step" else y.detach(), "state": state.detach()}
    if train:
        dx, dw, db, ds = torch.autograd.grad([y, state], leaves, [s["dy"], s["dstate_out"]])
        out.update(dx=dx, dweight=dw, dbias=db, dstate=ds)
    return out


def _exact_scan(s, c):
    B, L, D, N, G = c["B"], c["L"], c["D"], c["N"], c["G"]
    train = c["mode"] == "train"
    if train and L * B * D * N > 3e8:
        return None
    names = ["u", "delta", "A", "B", "C", "D", "delta_bias", "state"] + (["z"] if c["gate"] else [])
    if train:
        leaves = _leaf(s, *names)
    lens = torch.tensor(_lens(s, L, B), device=_DEV)
    h, ys = s["state"], []
    for i in range(L):
        on = (lens > i)[:, None]
        raw = s["delta"][:, i] + s["delta_bias"]
        dt = torch.logaddexp(raw, torch.zeros_like(raw))
        Bi = s["B"][:, i].repeat_interleave(D // G, dim=1)
        Ci = s["C"][:, i].repeat_interleave(D // G, dim=1)
        u = s["u"][:, i]
        new = torch.exp(dt[..., None] * s["A"]) * h + dt[..., None] * Bi * u[..., None]
        h = torch.where(on[..., None], new, h)
        y = (h * Ci).sum(-1) + s["D"] * u
        if c["gate"]:
            y = y * s["z"][:, i] / (1 + torch.exp(-s["z"][:, i]))
        ys.append(torch.where(on, y, torch.zeros_like(y)))
    y = torch.stack(ys, 1)
    out = {"y": y.detach()[:, 0] if c["mode"] == "step" else y.detach(), "state": h.detach()}
    if train:
        g = dict(zip(names, torch.autograd.grad([y, h], leaves, [s["dy"], s["dstate_out"]])))
        out.update(du=g["u"], ddelta=g["delta"], dA=g["A"], dB=g["B"], dC=g["C"], dD=g["D"], dz=g.get("z"),
                   ddelta_bias=g["delta_bias"], dstate=g["state"])
    return out
