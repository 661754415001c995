"""Group norm with an activation, the causal convolution and the selective scan (auditory_amd.norm, auditory_amd.scan) against
their definitions in 64 bits: on the CPU thread emulator (kernel sources compiled unchanged) and on the GPU."""
import ctypes as C
import os
import sys

import pytest
import torch

import frame_cases as F
from auditory_amd import capi, frames, norm, runtime, scan

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emul"))

gpu = pytest.mark.gpu


def ids(cases):
    return ["-".join(str(v) for v in c) for c in cases]


@pytest.fixture(scope="module")
def emu_lib():
    import backend
    with backend.emulated("plain") as lib:
        yield lib


@pytest.fixture
def emu(emu_lib, monkeypatch):
    """the operators on CPU tensors, their kernels run by the thread emulator"""
    native = frames.native()
    monkeypatch.setattr(frames, "context", lambda x, name: runtime.get_ctx(0).handle.value)
    frames.bind(native, emu_lib, False)
    yield emu_lib
    frames.bind(native, C.CDLL(capi.LIB_PATH), True)


# ---- values and gradients ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("case", F.NORM, ids=ids(F.NORM))
def test_emul_norm(emu, case):
    F.norm_case("cpu", *case)


@pytest.mark.parametrize("case", F.CONV, ids=ids(F.CONV))
def test_emul_conv(emu, case):
    F.conv_case("cpu", *case)


@pytest.mark.parametrize("case", F.SCAN, ids=ids(F.SCAN))
def test_emul_scan(emu, case):
    F.scan_case("cpu", *case)


@gpu
@pytest.mark.parametrize("case", F.NORM, ids=ids(F.NORM))
def test_gpu_norm(case):
    F.norm_case("cuda:0", *case)


@gpu
@pytest.mark.parametrize("case", F.CONV, ids=ids(F.CONV))
def test_gpu_conv(case):
    F.conv_case("cuda:0", *case)


@gpu
@pytest.mark.parametrize("case", F.SCAN, ids=ids(F.SCAN))
def test_gpu_scan(case):
    F.scan_case("cuda:0", *case)


@gpu
@pytest.mark.parametrize("case", F.NORM_BIG, ids=ids(F.NORM_BIG))
def test_gpu_norm_routes(case):
    F.norm_case("cuda:0", *case)


@gpu
@pytest.mark.parametrize("case", F.CONV_BIG, ids=ids(F.CONV_BIG))
def test_gpu_conv_routes(case):
    F.conv_case("cuda:0", *case)


@gpu
@pytest.mark.parametrize("case", F.SCAN_BIG, ids=ids(F.SCAN_BIG))
def test_gpu_scan_routes(case):
    F.scan_case("cuda:0", *case)


def test_emul_norm_over_workgroups(emu):
    F.norm_case("cpu", 2, 600, 16, 4, "f32", "silu", True, "mixed", 0, 0.0)


def test_emul_scan_many_chunks(emu):
    F.scan_case("cpu", 1, 600, 4, 1, 2, "f32", True, True, True, True, True, None, 0)


STREAM = [(2, 9, 8, 2, 4, "f32"), (3, 5, 12, 1, 16, "bf16"), (1, 6, 5, 1, 33, "f16")]


@pytest.mark.parametrize("case", STREAM, ids=ids(STREAM))
def test_emul_frame_by_frame(emu, case):
    F.stream_case("cpu", *case)


@gpu
@pytest.mark.parametrize("case", STREAM, ids=ids(STREAM))
def test_gpu_frame_by_frame(case):
    F.stream_case("cuda:0", *case)


def test_emul_gradients_against_differences(emu):
    F.difference_cases("cpu")


@gpu
def test_gpu_gradients_against_differences():
    F.difference_cases("cuda:0")


# ---- refusals ------------------------------------------------------------------------------------------------------------

def refused(fn, *args, **kw):
    with pytest.raises(capi.AuditoryError) as e:
        fn(*args, **kw)
    assert e.value.status == capi.AUD_EINVAL
    return str(e.value)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 4)
    assert "GPU" in refused(norm.group_norm, x, 1)
    assert "GPU" in refused(scan.causal_conv, x, torch.zeros(4, 2))
    assert "GPU" in refused(scan.selective_scan, x, x, torch.zeros(4, 2), torch.zeros(1, 2, 1, 2), torch.zeros(1, 2, 1, 2))


def test_norm_refusals(emu):
    x = torch.zeros(2, 3, 8)
    w = torch.zeros(8)
    refused(norm.group_norm, x.double(), 2)
    refused(norm.group_norm, x[0], 2)
    refused(norm.group_norm, x, 3)
    refused(norm.group_norm, x, 0)
    refused(norm.group_norm, x, 2, act="tanh")
    refused(norm.group_norm, x, 2, eps=0.0)
    refused(norm.group_norm, x, 2, w[:4])
    refused(norm.group_norm, x, 2, w.double())
    refused(norm.group_norm, x, 2, torch.zeros(16)[::2])
    refused(norm.group_norm, x.transpose(1, 2), 3)                       # channels not contiguous
    refused(norm.group_norm, x[:1].expand(2, 3, 8), 2)                   # items on top of one another
    refused(norm.group_norm, x, 2, lengths=torch.zeros(2, dtype=torch.int64))
    refused(norm.group_norm, x, 2, lengths=torch.zeros(3, dtype=torch.int32))
    refused(norm.group_norm, torch.zeros(1, 1, 4097), 1)
    assert "overlaps" in refused(norm.group_norm, x, 2, out=x)
    refused(norm.group_norm, x, 2, out=torch.zeros(2, 3, 9)[..., :8])
    refused(norm.group_norm_grad, x, x, None, 2)
    refused(norm.group_norm_grad, x[:, :2], x, torch.zeros(2, 2, 2), 2)
    refused(norm.group_norm_grad, x, x.clone(), torch.zeros(2, 3, 2), 2)


def test_conv_refusals(emu):
    x, w = torch.zeros(2, 5, 8), torch.zeros(8, 4)
    refused(scan.causal_conv, x, torch.zeros(8, 5))
    refused(scan.causal_conv, x, torch.zeros(8, 0))
    refused(scan.causal_conv, x, torch.zeros(7, 4))
    refused(scan.causal_conv, x, w, act="gelu")
    refused(scan.causal_conv, x, w, state=torch.zeros(2, 4, 8))
    refused(scan.causal_conv, x, w, state=torch.zeros(2, 3, 8, dtype=torch.float16))
    refused(scan.causal_conv, x, w, out=x)
    refused(scan.causal_conv, x[:, 0], w)
    refused(scan.causal_conv_step, x, torch.zeros(2, 3, 8), w)
    s = torch.zeros(2 * 3 * 8 + 8)
    refused(scan.causal_conv, x, w, state=s[:48].view(2, 3, 8), state_out=s[8:].view(2, 3, 8))   # half on top of it
    refused(scan.causal_conv_grad, x, x, w, dstate_out=torch.zeros(2, 2, 8))


def test_scan_refusals(emu):
    x, A, B = torch.zeros(2, 5, 8), torch.zeros(8, 4), torch.zeros(2, 5, 2, 4)
    C = B.clone()
    ok = scan.selective_scan(x, x.clone(), A, B, C)
    assert (ok == 0).all()
    refused(scan.selective_scan, x, x.half(), A, B, C)
    refused(scan.selective_scan, x, x[:, :4], A, B, C)
    refused(scan.selective_scan, x, x, torch.zeros(8, 65), torch.zeros(2, 5, 2, 65), torch.zeros(2, 5, 2, 65))
    refused(scan.selective_scan, x, x, A, torch.zeros(2, 5, 3, 4), torch.zeros(2, 5, 3, 4))
    refused(scan.selective_scan, x, x, A, B[:, :, 0], C[:, :, 0])
    refused(scan.selective_scan, x, x, A, B.transpose(2, 3).contiguous().transpose(2, 3), C)
    refused(scan.selective_scan, x, x, A, B, C, z=torch.zeros(2, 5, 9))
    refused(scan.selective_scan, x, x, A, B, C, state=torch.zeros(2, 8, 5))
    refused(scan.selective_scan, x, x, A, B, C, D=torch.zeros(7))
    refused(scan.selective_scan, x, x, A, B, C, out=x)
    refused(scan.selective_scan_grad, x, x, x, A, B, C, None)
    refused(scan.selective_scan_grad, x, x, x, A, B, C, torch.zeros(5))


def test_abi_refusals(emu):
    """what the Python layer does not let through, at the C ABI"""
    lib, h = emu, runtime.get_ctx(0).handle
    n = C.c_int64()
    p = capi.NormParams(capi.AUD_F32, 0, 2, 600, 32, 4, 1e-5, 0, 600 * 32, 32, 0, 0)
    assert lib.aud_group_norm_workspace_bytes(C.byref(p), 0, C.byref(n)) == 0 and n.value > 0
    x, y = torch.zeros(2, 600, 32), torch.full((2, 600, 32), 7.0)
    ws = torch.zeros(n.value // 4 + 8)
    call = lambda p, x, w, size: lib.aud_group_norm_batch_dev(h, C.byref(p), x, None, None, None, y.data_ptr(), None, w, size, None)  # noqa: E731
    assert call(p, x.data_ptr(), None, 0) == capi.AUD_EINVAL
    assert call(p, x.data_ptr(), ws.data_ptr(), n.value - 4) == capi.AUD_EINVAL
    assert call(p, x.data_ptr(), ws.data_ptr() + 4, n.value) == capi.AUD_EINVAL
    assert call(p, None, ws.data_ptr(), n.value) == capi.AUD_EINVAL
    assert call(p, x.data_ptr() + 2, ws.data_ptr(), n.value) == capi.AUD_EINVAL
    for field, value in (("dtype", capi.AUD_I16), ("dtype", capi.AUD_F64), ("act", 4), ("act", -1), ("groups", 5), ("groups", 0),
                         ("n_items", -1), ("rows", -1), ("rows", (1 << 30) + 1), ("channels", 0), ("eps", float("nan")), ("x_row", 31),
                         ("x_item", 600 * 32 - 1)):
        q = capi.NormParams.from_buffer_copy(p)
        setattr(q, field, value)
        assert call(q, x.data_ptr(), ws.data_ptr(), n.value) == capi.AUD_EINVAL, field
    assert lib.aud_group_norm_batch_dev(None, C.byref(p), x.data_ptr(), None, None, None, y.data_ptr(), None, ws.data_ptr(), n.value,
                                        None) == capi.AUD_EINVAL
    assert (y == 7).all()                                                  # nothing was written
    c = capi.ConvParams(capi.AUD_F32, 1, 1, 4, 8, 3, 32, 8, 32, 8)         # relu is not the convolution's
    assert lib.aud_causal_conv_workspace_bytes(C.byref(c), C.byref(n)) == capi.AUD_EINVAL
    s = capi.ScanParams(capi.AUD_F32, 0, 1, 4, 8, 3, 4, 0)
    assert lib.aud_scan_workspace_bytes(C.byref(s), 0, C.byref(n)) == capi.AUD_EINVAL
    assert lib.aud_scan_kept_floats(C.byref(s), C.byref(n)) == capi.AUD_EINVAL


def test_nothing_to_do(emu):
    """no items, no rows"""
    y, st = norm.group_norm(torch.zeros(0, 3, 8), 2, want_stats=True)
    assert y.shape == (0, 3, 8)
    dx, dw, db = norm.group_norm_grad(torch.zeros(0, 3, 8), torch.zeros(0, 3, 8), st, 2, torch.ones(8), torch.ones(8))
    assert dx.shape == (0, 3, 8) and (dw == 0).all() and (db == 0).all()
    x = torch.zeros(2, 0, 8)
    y, st = norm.group_norm(x, 2, want_stats=True)
    assert torch.equal(st[..., 0], torch.zeros(2, 2)) and torch.allclose(st[..., 1], torch.full((2, 2), 1e-5 ** -0.5))
    dx, dw, db = norm.group_norm_grad(x, x, st, 2, torch.ones(8), torch.ones(8))
    assert (dw == 0).all() and (db == 0).all()
    e = torch.zeros(0, 3, 8)
    g = scan.causal_conv_grad(e, e, torch.zeros(8, 3), torch.zeros(8))
    assert (g.weight == 0).all() and (g.bias == 0).all() and scan.causal_conv(e, torch.zeros(8, 3)).shape == (0, 3, 8)
    v = torch.zeros(0, 3, 1, 4)
    y, kept = scan.selective_scan(e, e, torch.zeros(8, 4), v, v, D=torch.zeros(8), keep=True)
    g = scan.selective_scan_grad(e, e, e, torch.zeros(8, 4), v, v, kept, D=torch.zeros(8))
    assert y.shape == (0, 3, 8) and (g.A == 0).all() and (g.D == 0).all()


def test_outputs_stay_inside(emu):
    """nothing is written beside the outputs"""
    m = F.Make("cpu", 21, "f32")
    x, w = m.n(2, 5, 8), m.n(8, 4)
    for fn in (lambda o: norm.group_norm(x, 2, out=o), lambda o: scan.causal_conv(x, w, out=o),
               lambda o: scan.selective_scan(x, x.abs(), -w.abs(), m.n(2, 5, 1, 4), m.n(2, 5, 1, 4), out=o)):
        buf = torch.full((16 + 80 + 16,), 9.0)
        fn(buf[16:96].view(2, 5, 8))
        assert (buf[:16] == 9).all() and (buf[96:] == 9).all() and (buf[16:96] != 9).all()


# ---- on the GPU: graphs, streams, far addresses, bits ------------------------------------------------------------------------

def _train(m, lens):
    """a run of the three operators with their gradients, as a training step makes it"""
    x = m["x"]
    y, st = norm.group_norm(x, 4, m["gw"], m["gb"], act="silu", lengths=lens, want_stats=True)
    c = scan.causal_conv(y, m["cw"], m["cb"], act="silu", lengths=lens)
    s, kept = scan.selective_scan(c, m["delta"], m["A"], m["B"], m["C"], D=m["D"], z=y, delta_bias=m["bias"], softplus=True, lengths=lens,
                                  keep=True)
    g = scan.selective_scan_grad(m["dy"], c, m["delta"], m["A"], m["B"], m["C"], kept, D=m["D"], z=y, delta_bias=m["bias"],
                                 softplus=True, lengths=lens)
    k = scan.causal_conv_grad(g.u, y, m["cw"], m["cb"], act="silu", lengths=lens)
    dx, dw, db = norm.group_norm_grad(k.x + g.z, x, st, 4, m["gw"], m["gb"], act="silu", lengths=lens)
    return [y, st, c, s, g.delta, g.A, g.B, g.C, g.D, g.delta_bias, k.weight, k.bias, dx, dw, db]


def _train_inputs(dev, seed, items=3, steps=150, ch=32, states=8, dtype="bf16"):
    m = F.Make(dev, seed, dtype)
    a = F.scan_inputs(m, items, steps, ch, 1, states, True, False, True, True, False)
    return dict(x=m.n(items, steps, ch), dy=m.n(items, steps, ch), gw=m.n(ch, f32=True), gb=m.n(ch, f32=True), cw=m.n(ch, 4, f32=True),
                cb=m.n(ch, f32=True), delta=a["delta"], A=a["A"], B=a["B"], C=a["C"], D=a["D"], bias=a["delta_bias"])


@gpu
def test_gpu_captured_training_step():
    """a captured step, replayed with other inputs in the same buffers, an eager run and a second graph in between: every
    replay equals the eager result bit for bit"""
    dev = "cuda:0"
    lens = torch.tensor([150, 0, 77], dtype=torch.int32, device=dev)
    static = [_train_inputs(dev, 31), _train_inputs(dev, 32)]
    for s in static:
        _train(s, lens)  # (the context and the plans)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_train(s, lens))
        graphs.append(g)
    for turn in range(4):
        fresh = [_train_inputs(dev, 40 + 2 * turn + i) for i in (0, 1)]
        for s, f in zip(static, fresh):
            for n in s:
                s[n].copy_(f[n])
        for g in graphs:
            g.replay()
        want = [_train(f, lens) for f in fresh]
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            for i, (p, q) in enumerate(zip(o, w)):
                assert torch.equal(p, q), (turn, i)


@gpu
def test_gpu_other_streams_and_the_same_bits():
    """two streams at once, then one after the other: the same bits"""
    dev = "cuda:0"
    ins = [_train_inputs(dev, 50 + i) for i in range(2)]
    want = [_train(i, None) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = []
    for s, i in zip(streams, ins):
        with torch.cuda.stream(s):
            got.append([_train(i, None) for _ in range(3)])
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            assert all(torch.equal(a, b) for a, b in zip(w, r))


@gpu
def test_gpu_offsets_past_32_bits():
    """items more than 2^31 elements apart, and a batch whose last rows lie behind 2^31"""
    dev = "cuda:0"
    far = (1 << 31) + 64
    buf = torch.zeros(far + 40 * 16, dtype=torch.bfloat16, device=dev)
    m = F.Make(dev, 61, "bf16")
    x = m.n(2, 40, 16)
    xs = buf.as_strided((2, 40, 16), (far, 16, 1))
    xs.copy_(x)
    w, b, cw = m.n(16, f32=True), m.n(16, f32=True), m.n(16, 4, f32=True)
    y, st = norm.group_norm(x, 4, w, b, act="silu", want_stats=True)
    assert torch.equal(norm.group_norm(xs, 4, w, b, act="silu"), y)
    dy = m.n(2, 40, 16)
    for p, q in zip(norm.group_norm_grad(dy, xs, st, 4, w, b, act="silu"), norm.group_norm_grad(dy, x, st, 4, w, b, act="silu")):
        assert torch.equal(p, q)
    assert torch.equal(scan.causal_conv(xs, cw, b), scan.causal_conv(x, cw, b))
    for p, q in zip(scan.causal_conv_grad(dy, xs, cw, b), scan.causal_conv_grad(dy, x, cw, b)):
        assert p is None and q is None or torch.equal(p, q)
    a = F.scan_inputs(m, 2, 40, 16, 1, 4, True, False, True, True, False)
    kw = dict(D=a["D"], delta_bias=a["delta_bias"], softplus=True)
    ya, ka = scan.selective_scan(x, a["delta"], a["A"], a["B"], a["C"], z=x, keep=True, **kw)
    yb, kb = scan.selective_scan(xs, a["delta"], a["A"], a["B"], a["C"], z=xs, keep=True, **kw)
    assert torch.equal(ya, yb) and torch.equal(ka, kb)
    for p, q in zip(scan.selective_scan_grad(dy, x, a["delta"], a["A"], a["B"], a["C"], ka, z=x, **kw),
                    scan.selective_scan_grad(dy, xs, a["delta"], a["A"], a["B"], a["C"], kb, z=xs, **kw)):
        assert p is None and q is None or torch.equal(p, q)
    del buf, xs
    # rows behind 2^31: the last item of a contiguous batch, alone and in it
    items, steps, ch = 5, 8192, 65536
    big = torch.empty((items, steps, ch), dtype=torch.bfloat16, device=dev)
    big[:-1] = 0
    tail = m.n(1, 64, 64).expand(1, 64, 64)
    big[-1] = 0
    big[-1, -64:, -64:] = tail[0]
    wide = torch.zeros(ch, 2, device=dev)
    wide[:, 0], wide[:, 1] = 0.5, 1.0
    out = scan.causal_conv(big, wide)
    ref = scan.causal_conv(big[-1:, -64:, -64:], wide[-64:].contiguous())
    assert torch.equal(out[-1:, -64:, -64:], ref) and (out[:-1] == 0).all()


# ---- a run of them behind the front end --------------------------------------------------------------------------------------

@gpu
def test_gpu_encoder_behind_the_gabor_maps(orc):
    """sound -> gabor maps -> group norm with an activation -> per band: causal convolution -> projections -> gated scan, whole
    and frame by frame, against the same in 64 bits from the maps on"""
    import numpy as np
    import frame_ref as R
    import workloads as W
    from auditory_amd import synth
    from auditory_amd.batch import BatchProcessor
    dev, n, py, px, nf = "cuda:0", 3, 11, 32, 16
    oc = W.OracleCfg(orc, "cfg2_16k_n400_nf40")
    length = oc.full_len()
    sig, _ = synth.batch(9, n, 16000, oc.sr, row_len=length)
    plan = W.product_plan(oc, capi.AUD_F64, dict(size=(9, 9), stride=(3, 3), gain=2.0, specs=W.DEFAULT_GABOR_SPECS))
    bp = BatchProcessor(plan, dev)
    items = bp.upload_items(runtime.make_items(np.arange(n) * length, [length] * n, [0] * n))
    m = F.Make(dev, 71, "f32")
    w, b = m.n(nf, shift=1.0, scale=0.2), m.n(nf, scale=0.2)
    mel, gab, maps = bp.process_norm(torch.from_numpy(sig.astype(np.float32)).to(dev).view(-1), items, n, py, px, 2, w, b, act="silu")
    assert maps.shape == gab.shape == (n, py, px, 2, nf // 2)
    # the settled maps beside them, as before
    from auditory_amd import kwta
    k = kwta.KWTA()
    k.Defaults()
    assert bp.kwta(gab, k).shape == gab.shape
    flat = R.leaf(gab.reshape(n, py * px, nf))
    ref_maps, st = R.norm(flat, 2, R.leaf(w), R.leaf(b), 1e-5, "silu", None)
    d = 1 + flat.detach().abs().amax() * 2 * st[..., 1].detach().amax()
    R.check("maps", maps.reshape(n, py * px, nf), ref_maps, torch.ones_like(ref_maps) * d * (1 + ref_maps.detach().abs()), 64 + py * px)
    x = bp.band_frames(maps)
    assert x.data_ptr() == maps.data_ptr() and x.shape == (n * py, px, nf)
    cw, cb, N = m.n(nf, 4, scale=0.5), m.n(nf, scale=0.2), 8
    pd, pb, pc = m.n(nf, nf, scale=0.2), m.n(nf, N, scale=0.3), m.n(nf, N, scale=0.3)
    A, D = -(torch.arange(1, N + 1, device=dev).float().expand(nf, N) * (0.5 + m.u(nf, 1))), m.n(nf)
    h_end = torch.empty(n * py, nf, N, device=dev)
    c = scan.causal_conv(x, cw, cb, act="silu")
    delta, B, C_ = c @ pd, (c @ pb).unsqueeze(2), (c @ pc).unsqueeze(2)
    y = scan.selective_scan(c, delta, A, B, C_, D=D, z=x, softplus=True, state_out=h_end)
    # frame by frame from the same projections
    cs, h = torch.zeros(n * py, 3, nf, device=dev), torch.zeros(n * py, nf, N, device=dev)
    ys = []
    for t in range(px):
        ct = scan.causal_conv_step(x[:, t], cs, cw, cb, act="silu")
        assert torch.equal(ct, c[:, t])
        ys.append(scan.selective_scan_step(ct, delta[:, t], A, B[:, t], C_[:, t], h, D=D, z=x[:, t], softplus=True))
    a = dict(u=c, delta=delta, A=A.contiguous(), B=B, C=C_, D=D, z=x, delta_bias=None, state=None)
    zero = torch.zeros_like(c)
    F.scan_check(a, None, True, zero, torch.zeros_like(h), y, h_end, None)
    F.scan_check(a, None, True, zero, torch.zeros_like(h), torch.stack(ys, 1), h, None)
    plan.close()


# ---- inputs laid out frames first, seen items first ------------------------------------------------------------------------

def frames_first(dev):
    m = F.Make(dev, 11, "bf16")
    B, L, D, G, N = 3, 40, 32, 2, 8
    lengths = m.lengths("mixed", B, L)

    def both(*shape):
        t = m.n(*shape)
        return t, t.transpose(0, 1).contiguous().transpose(0, 1)

    (x, xt), (dy, dyt), (dt, dtt), (z, zt) = (both(B, L, D) for _ in range(4))
    (Bm, Bt), (Cm, Ct) = (both(B, L, G, N) for _ in range(2))
    A, w = -(0.2 + m.u(D, N)), m.n(D, 3, f32=True)
    y, st = norm.group_norm(x, 4, lengths=lengths, want_stats=True)
    yt, stt = norm.group_norm(xt, 4, lengths=lengths, want_stats=True)
    pairs = [(y, yt), (st, stt)]
    pairs += zip(norm.group_norm_grad(dy, x, st, 4, lengths=lengths)[:1], norm.group_norm_grad(dyt, xt, st, 4, lengths=lengths)[:1])
    pairs.append((scan.causal_conv(x, w, act="silu", lengths=lengths), scan.causal_conv(xt, w, act="silu", lengths=lengths)))
    pairs += list(zip(scan.causal_conv_grad(dy, x, w, lengths=lengths), scan.causal_conv_grad(dyt, xt, w, lengths=lengths)))[:2]
    (v, kept), (vt, _) = (scan.selective_scan(*a, A, *bc, z=g, softplus=True, lengths=lengths, keep=True)
                          for a, bc, g in (((x, dt), (Bm, Cm), z), ((xt, dtt), (Bt, Ct), zt)))
    pairs.append((v, vt))
    got = scan.selective_scan_grad(dy, x, dt, A, Bm, Cm, kept, z=z, softplus=True, lengths=lengths)
    gott = scan.selective_scan_grad(dyt, xt, dtt, A, Bt, Ct, kept, z=zt, softplus=True, lengths=lengths)
    pairs += [(p, q) for p, q in zip(got, gott) if p is not None]
    for i, (p, q) in enumerate(pairs):
        assert q.is_contiguous() and torch.equal(p, q), i


def test_emul_frames_first(emu):
    frames_first("cpu")


@gpu
def test_gpu_frames_first():
    frames_first("cuda:0")


def infinite_input(dev):
    """the weights' gradient of a run of frames that ends in an infinite input: infinite, not NaN"""
    x, dy, w = torch.ones(1, 40, 4), torch.ones(1, 40, 4), torch.ones(4, 2)
    for t in (7, 15, 31):
        x[0, t] = float("inf")
    g = scan.causal_conv_grad(dy.to(dev), x.to(dev), w.to(dev))
    assert torch.isposinf(g.weight).all() and torch.equal(g.x.cpu()[0, :39], torch.full((39, 4), 2.0))


def test_emul_conv_gradients_of_infinite_inputs(emu):
    infinite_input("cpu")


@gpu
def test_gpu_conv_gradients_of_infinite_inputs():
    infinite_input("cuda:0")


def test_axes_past_32_bits_are_refused(emu):
    wide = torch.zeros(1, 1, 1).expand(2 ** 31 + 1, 1, 1)
    assert "2^31" in refused(norm.group_norm, wide, 1)
    assert "2^31" in refused(norm.group_norm, wide.transpose(0, 1), 1)
    assert "2^31" in refused(scan.causal_conv, wide, torch.zeros(1, 2))
    assert "2^31" in refused(scan.causal_conv_step, wide[:, 0], torch.zeros(1, 1, 1), torch.zeros(1, 2))
    assert "2^31" in refused(scan.selective_scan, wide, wide, torch.zeros(1, 2), torch.zeros(1, 1, 1, 2), torch.zeros(1, 1, 1, 2))


def test_strides_that_reach_too_far_are_refused(emu):
    p = capi.NormParams(dtype=capi.AUD_F32, act=0, n_items=2, rows=3, channels=4, groups=1, eps=1e-5, x_item=2 ** 62, x_row=4)
    n = C.c_int64()
    assert emu.aud_group_norm_workspace_bytes(C.byref(p), 0, C.byref(n)) == capi.AUD_EINVAL
    p.x_item, p.x_row = 4, 8                   # frames first
    assert emu.aud_group_norm_workspace_bytes(C.byref(p), 0, C.byref(n)) == capi.AUD_OK
    p.x_item, p.x_row = 4, 7                   # the last channel of an item in the first of another
    assert emu.aud_group_norm_workspace_bytes(C.byref(p), 0, C.byref(n)) == capi.AUD_EINVAL
