"""BatchProcessor.group_norm on a padded batch: `lengths` are frames, along the maps' time axis."""
import pytest
import torch

import frame_cases as F
import frame_ref as R
import norm_cases as N
from auditory_amd import capi
from auditory_amd.batch import BatchProcessor
from test_norm_widths import emu, emu_lib  # noqa: F401  (fixtures)

gpu = pytest.mark.gpu


def padded(dev, n, py, px, tail, groups, act, kind):
    m = F.Make(dev, 9, "f32")
    ch = 1
    for v in tail:
        ch *= v
    maps = m.n(n, py, px, *tail)
    w, b = m.n(ch, f32=True, scale=0.3, shift=1.0), m.n(ch, f32=True, scale=0.3)
    lengths = m.lengths(kind, n, px)
    frames = R.lens_of(lengths, n, px)
    given = maps.clone()
    for i, t in enumerate(frames):
        given[i, :, t:] = float("nan")       # what lies behind an utterance has no effect
    bp = BatchProcessor.__new__(BatchProcessor)  # (the plan has no part in this)
    y, stats = bp.group_norm(given, groups, w, b, act=act, lengths=lengths, want_stats=True)
    assert y.shape == maps.shape and y.is_contiguous()
    assert torch.equal(y, bp.group_norm(given, groups, w, b, act=act, lengths=lengths))
    assert bp.band_frames(y).data_ptr() == y.data_ptr()
    for i, t in enumerate(frames):
        assert (y[i, :, t:] == 0).all()
        if t == 0:  # nothing to normalise: mean 0, variance 0
            assert (stats[i, :, 0] == 0).all() and (stats[i, :, 1] - 1e-5 ** -0.5).abs().max() < 1e-3
            continue
        x = maps[i:i + 1, :, :t].reshape(1, py * t, ch)   # all bands, the frames that are there
        e = N.Exact(x, torch.zeros_like(x), groups, w, b, 1e-5, act, None)
        e.near("y", y[i:i + 1, :, :t].reshape(1, py * t, ch), e.y, e.ey)
        e.near("mean", stats[i:i + 1, :, 0], e.mean, e.emean)
        e.near("rstd", stats[i:i + 1, :, 1], e.rstd, e.erstd)
    # without lengths: all of it, and full lengths are the same
    whole = bp.group_norm(maps, groups, w, b, act=act)
    full = bp.group_norm(maps, groups, w, b, act=act, lengths=torch.full((n,), px + 3, dtype=torch.int32, device=dev))
    e = N.Exact(maps.reshape(n, py * px, ch), torch.zeros(n, py * px, ch), groups, w, b, 1e-5, act, None)
    for y in (whole, full):
        e.near("y", y.reshape(n, py * px, ch), e.y, e.ey)


CASES = [(5, 3, 7, (2, 4), 2, "silu", "mixed"), (3, 1, 6, (4,), 1, "relu", "out"), (2, 4, 1, (8,), 4, "none", None)]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_emul_padded_maps(emu, case):  # noqa: F811
    padded("cpu", *case)


@gpu
def test_gpu_padded_maps():
    for case in CASES + [(6, 11, 32, (2, 8), 2, "relu", "mixed")]:
        padded("cuda:0", *case)


def test_lengths_are_checked(emu):  # noqa: F811
    bp = BatchProcessor.__new__(BatchProcessor)
    maps = torch.zeros(2, 3, 4, 8)
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(2)):
        with pytest.raises(capi.AuditoryError) as e:
            bp.group_norm(maps, 2, lengths=bad)
        assert e.value.status == capi.AUD_EINVAL
    huge = torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32)   # held to [0, frames]
    y = bp.group_norm(torch.ones(2, 3, 4, 8), 2, bias=torch.ones(8), lengths=huge)
    assert (y[0] == 1).all() and (y[1] == 0).all()


@gpu
def test_gpu_padded_maps_in_a_graph():
    """captured once, replayed with other maps and lengths in the same buffers, eager work in between"""
    dev = "cuda:0"
    m = F.Make(dev, 19, "f32")
    bp = BatchProcessor.__new__(BatchProcessor)
    maps, w, b = m.n(4, 5, 9, 2, 4), m.n(8, f32=True), m.n(8, f32=True)
    lengths = torch.tensor([9, 3, 0, 7], dtype=torch.int32, device=dev)
    bp.group_norm(maps, 2, w, b, act="silu", lengths=lengths)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = bp.group_norm(maps, 2, w, b, act="silu", lengths=lengths)
    for turn in range(4):
        maps.copy_(m.n(4, 5, 9, 2, 4))
        lengths.copy_(torch.tensor([turn, 9, 5 - turn, 20], dtype=torch.int32))
        g.replay()
        want = bp.group_norm(maps, 2, w, b, act="silu", lengths=lengths)
        torch.cuda.synchronize()
        assert torch.equal(y, want), turn
