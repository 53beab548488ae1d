"""ropePositions and its gradient against the turn in 64 bits."""
import math

import pytest
import torch

import runntime_amd as rt
from runntime_amd import _lib
from tests import dense_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"f32": torch.float32, "f16": torch.float16}


def make(T, width, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + T + width)
    return torch.randn((T, width), generator=g).to(DT[dtype])


def check(x, pos, opts, inverse=False):
    print(list(x.shape), x.dtype, opts.get("layout"), flush=True)
    op = rt.ropePositionsBackward if inverse else rt.ropePositions
    dev = dict(opts, invFreq=opts["invFreq"].to(DEV))
    got = op(x.to(DEV), pos.to(DEV), dev)
    s = opts.get("srcStart", 0)
    w = opts.get("width", x.shape[1] - s)
    want, mag, ang = dense_ref.rope(x[:, s:s + w], pos, opts["invFreq"], opts.get("scale", 1.0),
                                    opts["headDim"], opts.get("rotaryDim", opts["headDim"]),
                                    opts.get("layout", "interleaved"), inverse)
    dense_ref.rope_close(got, want, mag, ang)
    return got


# heads, headDim, rotaryDim: whole heads, parts, widths that no wide unit divides
SHAPES = [(1, 2, 2), (2, 64, 64), (3, 80, 20), (5, 96, 48), (2, 128, 128), (1, 256, 64),
          (7, 6, 4), (3, 10, 2), (2, 36, 12), (16, 64, 32), (1, 2048, 2048)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("heads,hd,rot", SHAPES)
def test_shapes(heads, hd, rot, layout, dtype):
    freq, _ = rt.ropeFrequencies(rot, 10000.0, device="cpu")
    for T in (1, 3, 70):
        x = make(T, heads * hd, dtype)
        pos = torch.arange(T) + 5
        o = {"headDim": hd, "rotaryDim": rot, "layout": layout, "invFreq": freq, "scale": 1.25}
        check(x, pos, o)
        check(x, pos.int(), o, inverse=True)


def test_half_pairs_of_an_odd_head():
    freq, _ = rt.ropeFrequencies(6, 10000.0, device="cpu")
    x = make(9, 3 * 7, "f32")
    check(x, torch.arange(9), {"headDim": 7, "rotaryDim": 6, "layout": "half", "invFreq": freq})


@pytest.mark.parametrize("start", [0, 4095, 1 << 20, (1 << 31) - 3, -7, -(1 << 33)])
def test_far_and_negative_positions(start):
    freq, scale = rt.ropeFrequencies(128, 150000.0, {"type": "yarn", "factor": 32, "context": 4096},
                                     device="cpu")
    x = make(5, 256, "f32")
    check(x, torch.arange(5) + start, {"headDim": 128, "layout": "half", "invFreq": freq,
                                       "scale": scale})


def test_many_rows_and_many_heads():
    freq, _ = rt.ropeFrequencies(64, 10000.0, device="cpu")
    o = {"headDim": 64, "layout": "half", "invFreq": freq}
    check(make(40000, 64, "f16"), torch.randint(0, 9000, (40000,)), o)     # several rows a block
    check(make(3, 64 * 700, "f16"), torch.arange(3), o)                    # several blocks a row
    check(make(2100, 40 * 64, "f32"), torch.arange(2100), dict(o, layout="interleaved"))


def test_windows_strides_and_places():
    freq, _ = rt.ropeFrequencies(16, 10000.0, device="cpu")
    freq_d = freq.to(DEV)
    pos = torch.arange(11)
    for dtype in ("f32", "f16"):
        x = make(11, 112, dtype)
        for s, w in ((0, 64), (32, 48), (33, 32), (7, 80)):
            for layout in ("interleaved", "half"):
                o = {"headDim": 16, "invFreq": freq, "srcStart": s, "width": w, "layout": layout}
                got = check(x, pos, o)
                od = dict(o, invFreq=freq_d)
                # a cache's rows, other columns of the same rows, and in place
                cache = torch.full((20, w), 7.0, dtype=x.dtype, device=DEV)
                rt.ropePositions(x.to(DEV), pos.to(DEV), dict(od, out=cache[4:15]))
                assert torch.equal(cache[4:15], got)
                assert (cache[:4] == 7).all() and (cache[15:] == 7).all()
                xd = x.to(DEV)
                r = rt.ropePositions(xd, pos.to(DEV), dict(od, out=xd[:, s:s + w]))
                assert torch.equal(r, got) and torch.equal(xd[:, s:s + w], got)
                assert torch.equal(xd[:, :s].cpu(), x[:, :s])
                assert torch.equal(xd[:, s + w:].cpu(), x[:, s + w:])
        wide = torch.zeros((11, 64), dtype=x.dtype, device=DEV)
        wide[:, :32] = x[:, :32].to(DEV)
        want = rt.ropePositions(x[:, :32].contiguous().to(DEV), pos.to(DEV),
                                {"headDim": 16, "invFreq": freq_d})
        rt.ropePositions(wide[:, :32], pos.to(DEV), {"headDim": 16, "invFreq": freq_d,
                                                      "out": wide[:, 32:]})
        assert torch.equal(wide[:, 32:], want)
        assert torch.equal(wide[:, :32].cpu(), x[:, :32])


def test_overlapping_out_is_refused():
    freq = torch.ones(8, dtype=torch.float64, device=DEV)
    pos = torch.arange(4, device=DEV)
    buf = torch.zeros((6, 32), device=DEV)
    for out in (buf[1:5], buf.view(-1)[1:129].view(4, 32)):
        with pytest.raises(rt.RunntimeError) as e:
            rt.ropePositions(buf[:4], pos, {"headDim": 16, "invFreq": freq, "out": out})
        assert e.value.code == "INVALID_ARGUMENT" and "overlaps" in str(e.value)


def test_gradient_by_differences():
    """y is linear in x: <dy, y(v)> = <dx(dy), v> up to the f32 rounding."""
    freq, _ = rt.ropeFrequencies(32, 10000.0, device=DEV)
    o = {"headDim": 64, "rotaryDim": 32, "layout": "half", "invFreq": freq, "scale": 0.7}
    pos = torch.arange(33, device=DEV) * 91
    v, dy = make(33, 192, "f32", 1).to(DEV), make(33, 192, "f32", 2).to(DEV)
    a = (rt.ropePositions(v, pos, o).double() * dy.double()).sum()
    b = (rt.ropePositionsBackward(dy, pos, o).double() * v.double()).sum()
    assert abs(a - b) <= 4 * 2.0 ** -24 * math.sqrt(33 * 192) * 8


def test_inf_and_nan_stay_in_their_pair():
    freq, _ = rt.ropeFrequencies(8, 10000.0, device=DEV)
    x = torch.ones((2, 16), device=DEV)
    x[0, 3], x[1, 9] = math.inf, math.nan
    y = rt.ropePositions(x, torch.arange(2, device=DEV), {"headDim": 8, "invFreq": freq})
    bad = ~torch.isfinite(y)
    assert bad[0, 2:4].any() and not bad[0, :2].any() and not bad[0, 4:].any()
    assert bad[1, 8:10].all() and not bad[1, :8].any() and not bad[1, 10:].any()


def test_matches_rope_from_tables():
    """The same turn as rope takes from its f32 tables."""
    freq, _ = rt.ropeFrequencies(64, 10000.0, device=DEV)
    x = make(50, 128, "f32").to(DEV)
    ang = torch.arange(50, device=DEV).double()[:, None] * freq
    cos, sin = (t.float().repeat_interleave(2, 1).contiguous() for t in (ang.cos(), ang.sin()))
    a = rt.rope(x, cos, sin, {"headDim": 64})
    b = rt.ropePositions(x, torch.arange(50, device=DEV), {"headDim": 64, "invFreq": freq})
    assert (a - b).abs().max() <= 8 * 2.0 ** -24 * x.abs().max() * 2
