"""Group norm at widths that do not fit a workgroup's sweep, and over all of its routes, within bounds near the real error
(norm_cases.py): on the CPU thread emulator and on the GPU."""
import ctypes as C
import os
import sys

import pytest
import torch

import frame_ref as R
import norm_cases as N
from auditory_amd import capi, frames, norm, runtime

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
    native = frames.native()
    monkeypatch.setattr(frames, "context", lambda x, name: runtime.get_ctx(0).handle.value)
    frames.bind(native, emu_lib, False)
    yield emu_lib
    frames.bind(native, C.CDLL(capi.LIB_PATH), True)


@pytest.mark.parametrize("case", N.WIDE_EMUL, ids=ids(N.WIDE_EMUL))
def test_emul_widths(emu, case):
    N.case("cpu", *case)


@pytest.mark.parametrize("case", N.ROUTES, ids=ids(N.ROUTES))
def test_emul_routes(emu, case):
    N.case("cpu", *case)


@gpu
@pytest.mark.parametrize("case", N.WIDE, ids=ids(N.WIDE))
def test_gpu_widths(case):
    N.case("cuda:0", *case)


@gpu
@pytest.mark.parametrize("case", N.ROUTES, ids=ids(N.ROUTES))
def test_gpu_routes(case):
    N.case("cuda:0", *case)


# ---- that the bounds see what they are there to see -----------------------------------------------------------------------

SEEN = [N.ROUTES[0], N.ROUTES[2], N.ROUTES[3], N.ROUTES[5], N.ROUTES[7], (2, 40, 301, 7, "f32", "silu", True, None, 0)]


@pytest.mark.parametrize("case", SEEN, ids=ids(SEEN))
def test_emul_bounds_notice_what_is_left_out(emu, case):
    args, got = N.run("cpu", *case)
    N.held(args, got)
    for plant in N.PLANTED:
        with pytest.raises(AssertionError):
            N.held(args, got, plant)
    small = (2, 4, 16, 4, "f32", "silu", True, None, 0)
    args, got = N.run("cpu", *small)
    with pytest.raises(AssertionError):
        N.held(args, got, "variance")


def test_the_formula_is_the_derivative():
    """norm_cases' gradients against autograd's of the definition, in 64 bits"""
    for name in ("none", "relu", "silu", "gelu"):
        x, dy, w, b, lengths, _, _ = N.inputs("cpu", 3, 9, 12, 3, "f32", name, True, "mixed", 0)
        e = N.Exact(x, dy, 3, w, b, 1e-5, name, lengths)
        lv = [R.leaf(t) for t in (x, w, b)]
        y, st = R.norm(lv[0], 3, lv[1], lv[2], 1e-5, name, lengths)
        for got, ref in zip((e.y, e.dx, e.dw, e.db), [y.detach()] + R.grads([y], [dy], lv)):
            assert torch.allclose(got, ref, rtol=1e-9, atol=1e-12), name


def chunked_difference(dev):
    """the directional derivative of a chunked size by central differences of the kernels' own values: within the rounding of
    the two losses over h, and the truncation that halving h shows in 64 bits"""
    c = (2, 600, 32, 4, "f32", "silu", True, None, 0)
    x, dy, w, b, _, _, _ = N.inputs(dev, *c)
    h = 2.0 ** -3
    _, st = norm.group_norm(x, 4, w, b, act="silu", want_stats=True)
    g = norm.group_norm_grad(dy, x, st, 4, w, b, act="silu")
    # along the gradient, so that the loss changes by much more than its values' rounding (whose bound adds up over all elements)
    point, way = [x, w, b], [g[0], g[1] / g[1].abs().max(), g[2] / g[2].abs().max()]
    c64 = dy.cpu().double()

    def exact(step):
        p = [t.cpu().double() + step * d.cpu().double() for t, d in zip(point, way)]
        e = N.Exact(p[0], dy, 4, p[1], p[2], 1e-5, "silu", None)
        return float((e.y * c64).sum()), float((e.ey * c64.abs()).sum())

    def own(step):
        p = [t + step * d for t, d in zip(point, way)]
        return float((norm.group_norm(p[0], 4, p[1], p[2], act="silu").cpu().double() * c64).sum())

    got = (own(h) - own(-h)) / (2 * h)
    (up, e_up), (down, e_down) = exact(h), exact(-h)
    half = (exact(h / 2)[0] - exact(-h / 2)[0]) / h
    ref = (up - down) / (2 * h)
    # (the points p + h d are rounded too: half a step of each, times the gradient's magnitude)
    moved = sum(float((v.double().abs().cpu() * N.U * (t.cpu().double().abs() + h * d.cpu().double().abs())).sum())
                for v, t, d in zip(g, point, way))
    rounding = (e_up + e_down) / (2 * h) + moved / h
    assert abs(got - ref) <= rounding, (got, ref, rounding)
    along = sum(float((v.cpu().double() * d.cpu().double()).sum()) for v, d in zip(g, way))
    assert abs(along - ref) <= 2 * abs(ref - half) * 4 / 3 + rounding, (along, ref, half, rounding)
    assert rounding < 0.05 * abs(ref), (rounding, ref)


def test_emul_difference_over_chunks(emu):
    chunked_difference("cpu")


@gpu
def test_gpu_difference_over_chunks():
    chunked_difference("cuda:0")
