"""gatedFfn and its gradients against the block in 64 bits."""
import math

import pytest
import torch

import runntime_amd as rt
from runntime_amd import _lib
from tests import dense_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"f32": torch.float32, "f16": torch.float16}
ACTS = ["swiglu", "clampedSwiglu", "geglu"]


def make(T, d, i, dtype, bias=True, seed=0, gain=1.0):
    g = torch.Generator().manual_seed(seed * 131 + T + 3 * d + 7 * i)
    mk = lambda *s, scale=1.0: (torch.randn(s, generator=g) * scale).to(DT[dtype])
    w = [mk(d, i, scale=gain * d ** -0.5), mk(i, scale=0.3) if bias else None,
         mk(d, i, scale=gain * d ** -0.5), mk(i, scale=0.3) if bias else None,
         mk(i, d, scale=i ** -0.5), mk(d, scale=0.3) if bias else None]
    return mk(T, d), w, mk(T, d), mk(T, d)


def up(t):
    return None if t is None else t.to(DEV)


def rel(dtype, d, i, T=0):
    """Relative 2-norm error. f32: the sums. f16: h (or g, l, h, dg and dl, the
    derivatives' argument roundings counted twice) rounded by at most 2^-11
    each, and the output."""
    f32 = dense_ref.sum_rel(torch.float32, d, i, T)
    return f32 if dtype == torch.float32 else f32 + (7 if T else 2) * 2.0 ** -11


def check(T, d, i, dtype, act, train=True, bias=True, residual=True, gain=1.0):
    print(T, d, i, dtype, act, train, flush=True)
    x, w, res, dy = make(T, d, i, dtype, bias, gain=gain)
    res = res if residual else None
    y, grads, size = dense_ref.ffn(x, *w, act, residual=res, grad=dy)
    o = {"activation": act, "residual": up(res)}
    wd = [up(t) for t in w]
    got = rt.gatedFfn(x.to(DEV), *wd, o)
    what = f"{T} {d} {i} {dtype} {act}"
    dense_ref.norm_close(got, y, rel(x.dtype, d, i), what)
    if not train:
        return
    got2, saved = rt.gatedFfn(x.to(DEV), *wd, {**o, "save": True})
    dense_ref.norm_close(got2, y, rel(x.dtype, d, i), what)
    back = rt.gatedFfnBackward(dy.to(DEV), x.to(DEV), *wd, saved, {"activation": act})
    names = ("dx", "dglu_w", "dglu_b", "dlin_w", "dlin_b", "dout_w", "dout_b")
    for n, g, want in zip(names, back, grads):
        assert (g is None) == (want is None)
        if g is not None:
            dense_ref.norm_close(g, want, rel(x.dtype, d, i, T), f"{what} {n}",
                                 size if n == "dx" else None)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("d,i", [(1, 1), (8, 8), (7, 13), (64, 96), (100, 36), (129, 255), (640, 640)])
def test_shapes(d, i, act, dtype):
    for T in (1, 2, 5):
        check(T, d, i, dtype, act, bias=T != 2, residual=T != 5)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("d,i", [(256, 328), (200, 513), (321, 264)])
@pytest.mark.parametrize("T", [3, 4, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 77, 127, 129, 255, 300])
def test_rows(T, d, i, dtype):
    check(T, d, i, dtype, ACTS[T % 3], bias=T % 2 == 1, residual=T % 4 < 2)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("T,d,i", [(1100, 512, 1408), (1500, 640, 640), (513, 1000, 1001),
                                   (2050, 264, 520), (1, 2048, 5632), (40, 2048, 1408)])
def test_large(T, d, i, dtype):
    check(T, d, i, dtype, ACTS[T % 3])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("T,d,i", [(70, 1025, 4001), (300, 1031, 2047), (17, 2048, 6144),
                                   (150, 1500, 2102), (33, 1290, 646), (1, 1999, 2050)])
def test_tiles_in_parts_and_rows_of_every_width(T, d, i, dtype):
    check(T, d, i, dtype, "swiglu")


def test_a_long_batch_sums_in_full():
    """Weight and bias gradients over many rows."""
    check(9001, 72, 88, "f16", "swiglu")
    check(9001, 72, 88, "f32", "geglu")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_values_at_the_clamps(dtype):
    """Pre-activations far past the clamps, and at them: d = 1, x = 1."""
    v = torch.tensor([-9.0, -7.0, -6.5, 0.0, 6.5, 7.0, 7.25, 50.0])
    i = 64
    gw = v.repeat_interleave(8)[None].to(DT[dtype])
    lw = v.repeat(8)[None].to(DT[dtype])
    ow = torch.ones((i, 1), dtype=DT[dtype]) / i
    x = torch.ones((3, 1), dtype=DT[dtype])
    dy = torch.ones((3, 1), dtype=DT[dtype])
    for act in ACTS:
        print(act, flush=True)
        y, grads, size = dense_ref.ffn(x, gw, None, lw, None, ow, None, act, grad=dy)
        w = [t.to(DEV) for t in (gw, lw, ow)]
        got, saved = rt.gatedFfn(x.to(DEV), w[0], None, w[1], None, w[2], None,
                                 {"activation": act, "save": True})
        back = rt.gatedFfnBackward(dy.to(DEV), x.to(DEV), w[0], None, w[1], None, w[2], None, saved,
                                   {"activation": act})
        dense_ref.norm_close(got, y, rel(x.dtype, 1, i))
        for n, (g, want) in enumerate(zip(back, grads)):
            if g is not None:
                dense_ref.norm_close(g, want, rel(x.dtype, 1, i, 3), size=None if n else size)


@pytest.mark.parametrize("act", ACTS)
def test_large_pre_activations_stay_finite(act):
    check(5, 64, 96, "f32", act, gain=30.0)


def test_gradient_by_differences():
    x, w, _, dy = make(6, 48, 80, "f32")
    wd = [up(t) for t in w]
    xd, dyd = x.to(DEV), dy.to(DEV)
    _, saved = rt.gatedFfn(xd, *wd, {"save": True})
    back = rt.gatedFfnBackward(dyd, xd, *wd, saved)
    g = torch.Generator().manual_seed(5)
    for n in range(7):
        t = ([xd] + wd)[n]
        v = torch.randn(t.shape, generator=g).to(DEV)
        e = 2.0 ** -7
        moved = lambda s: [a + s * e * v if m == n else a for m, a in enumerate([xd] + wd)]
        diff = ((rt.gatedFfn(*moved(1)).double() - rt.gatedFfn(*moved(-1)).double())
                * dyd.double()).sum() / (2 * e)
        want = (back[n].double() * v.double()).sum()
        # the third derivatives' e² and the f32 outputs' rounding over 2e
        size = back[n].double().norm() * v.double().norm()
        assert abs(diff - want) <= 2e-3 * size + 2.0 ** -24 / e * 50, n


def test_some_gradients_only():
    """The C entry computes what it is given room for."""
    lib = _lib.load()
    T, d, i = 33, 40, 56
    x, w, _, dy = make(T, d, i, "f32")
    wd = [up(t) for t in w]
    xd, dyd = x.to(DEV), dy.to(DEV)
    _, saved = rt.gatedFfn(xd, *wd, {"save": True})
    want = rt.gatedFfnBackward(dyd, xd, *wd, saved)
    ctx = _lib.thread_context(0, torch.cuda.current_stream().cuda_stream)
    for n in range(7):
        outs = [torch.empty_like(t) if m == n else None for m, t in enumerate(want)]
        _lib.check(lib.moe_gated_ffn_backward(
            ctx, dyd.data_ptr(), xd.data_ptr(), 0, 0, wd[0].data_ptr(), wd[2].data_ptr(),
            wd[4].data_ptr(), saved.data_ptr(), T, d, i,
            *[None if t is None else t.data_ptr() for t in outs], None, 0))
        assert torch.equal(outs[n], want[n]), n


def test_refusals_on_the_device():
    lib = _lib.load()
    x, w, _, dy = make(4, 16, 16, "f32")
    wd = [up(t) for t in w]
    xd = x.to(DEV)
    ctx = _lib.thread_context(0, torch.cuda.current_stream().cuda_stream)
    p = [t.data_ptr() for t in wd]
    rc = lib.moe_gated_ffn(ctx, xd.data_ptr(), 0, 0, *p, None, 4, 16, 16, None, xd.data_ptr(), None, 0)
    assert rc == 1 and b"out overlaps x" in lib.moe_last_error()
    out = torch.empty_like(xd)
    ws = torch.empty(4096, dtype=torch.uint8, device=DEV)
    rc = lib.moe_gated_ffn(ctx, xd.data_ptr(), 0, 0, *p, None, 4, 16, 16, None, out.data_ptr(),
                           ws.data_ptr(), 16)
    assert rc == 1 and b"workspace holds 16 bytes" in lib.moe_last_error()
    rc = lib.moe_gated_ffn(ctx, xd.data_ptr(), 0, 0, *p, None, 4, 16, 16, None, out.data_ptr(),
                           ws.data_ptr() + 8, 4088)
    assert rc == 1 and b"256-byte aligned" in lib.moe_last_error()
    with pytest.raises(rt.RunntimeError, match="must be contiguous"):
        rt.gatedFfn(xd.t(), wd[0][:4], None, wd[2][:4], None, wd[4][:, :4], None)
    with pytest.raises(rt.RunntimeError, match="no elements"):
        rt.gatedFfn(xd[:0], *wd)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_tensors_off_an_aligned_address(dtype):
    x, w, res, dy = make(9, 40, 72, dtype)
    y, grads, size = dense_ref.ffn(x, *w, "swiglu", residual=res, grad=dy)
    off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)]).to(DEV)[1:].view(t.shape)
    wd = [off(t) for t in w]
    got, saved = rt.gatedFfn(off(x), *wd, {"residual": off(res), "save": True})
    dense_ref.norm_close(got, y, rel(x.dtype, 40, 72))
    back = rt.gatedFfnBackward(off(dy), off(x), *wd, off(saved.cpu()))
    for n, (g, want) in enumerate(zip(back, grads)):
        dense_ref.norm_close(g, want, rel(x.dtype, 40, 72, 9), size=None if n else size)
    lib = _lib.load()
    ctx = _lib.thread_context(0, torch.cuda.current_stream().cuda_stream)
    xo = off(x)
    out = torch.empty_like(got)
    p = [t.data_ptr() if m % 2 else _t.data_ptr() for m, (t, _t) in
         enumerate(zip(wd, [up(t) for t in w]))]
    rc = lib.moe_gated_ffn(ctx, xo.data_ptr(), 1 if dtype == "f16" else 0, 0, *p, None, 9, 40, 72,
                           None, out.data_ptr(), None, 0)
    assert rc == 1 and b"x must be 16-byte aligned" in lib.moe_last_error()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows_of_infinity_and_nan_stay_alone(dtype):
    """Row 3 of x is infinite, row 5 not a number; the other rows, and a K tail
    that shares a stage with them, are as without."""
    for T, d, i in ((8, 72, 40), (70, 200, 136), (300, 328, 264)):
        x, w, _, _ = make(T, d, i, dtype)
        want = dense_ref.ffn(x, *w, "swiglu")
        x[3, 7], x[5] = float("inf"), float("nan")
        got = rt.gatedFfn(x.to(DEV), *[up(t) for t in w]).cpu()
        assert not torch.isfinite(got[3]).all() and torch.isnan(got[5]).all()
        keep = [r for r in range(T) if r not in (3, 5)]
        dense_ref.norm_close(got[keep], want[keep], rel(x.dtype, d, i))


def test_buffers_are_not_read_past_their_end():
    """Tensors at the end of a filled buffer: what lies behind does not enter."""
    for T, d, i in ((3, 40, 56), (33, 100, 36), (129, 264, 200)):
        for dtype in ("f16", "f32"):
            x, w, _, dy = make(T, d, i, dtype, bias=False)
            place = lambda t: torch.cat([t.reshape(-1), t.new_full((8192,), float("nan"))]).to(
                DEV)[:t.numel()].view(t.shape)
            wd = [None if t is None else place(t) for t in w]
            y, grads, size = dense_ref.ffn(x, *w, "geglu", grad=dy)
            got, saved = rt.gatedFfn(place(x), *wd, {"activation": "geglu", "save": True})
            dense_ref.norm_close(got, y, rel(x.dtype, d, i))
            back = rt.gatedFfnBackward(place(dy), place(x), *wd, place(saved.cpu()),
                                       {"activation": "geglu"})
            for n, (g, want) in enumerate(zip(back, grads)):
                if g is not None:
                    dense_ref.norm_close(g, want, rel(x.dtype, d, i, T), size=None if n else size)
