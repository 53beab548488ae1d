"""linearQuant and QuantLinear against the product in 64 bits."""
import ctypes

import numpy as np
import pytest
import torch

import runntime_amd as rt
from runntime_amd import _lib
from tests import dense_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"f32": torch.float32, "f16": torch.float16}


def make(T, K, N, bits, group, dtype, seed=0, bias=True, addend=True):
    rng = np.random.default_rng(seed * 7919 + T * 31 + K * 7 + N + bits + group)
    half = 2 ** (bits - 1)
    q = rng.integers(-half, half, (K, N)).astype(np.int8)
    q[0, 0], q[K - 1, N - 1] = -half, half - 1
    sc = ((0.5 + rng.random((K // group, N))) / (half * K ** 0.5)).astype(np.float32)
    x = torch.from_numpy(rng.standard_normal((T, K)).astype(np.float32)).to(DT[dtype])
    b = torch.from_numpy(rng.standard_normal(N).astype(np.float32)) if bias else None
    a = (torch.from_numpy(rng.standard_normal((T, N)).astype(np.float32)).to(DT[dtype])
         if addend else None)
    words = torch.from_numpy(rt.pack_expert_weights(q[None], bits).view(np.int32))
    w = rt.QuantExpertWeight(rt.QuantW(words.to(DEV), (K, N)), torch.from_numpy(sc).to(DEV),
                             None if b is None else b.to(DEV))
    dense = torch.from_numpy(q).double() * torch.from_numpy(np.repeat(sc, group, 0)).double()
    return x, w, b, a, dense


def want_of(x, dense, b, a):
    y = x.double() @ dense
    y = y if b is None else y + b.double()
    return y if a is None else y + a.double()


def check(T, K, N, bits, group, dtype, **kw):
    print(T, K, N, bits, group, dtype, flush=True)
    x, w, b, a, dense = make(T, K, N, bits, group, dtype, **kw)
    got = rt.linearQuant(x.to(DEV), w, {"bits": bits, "groupSize": group,
                                        "addend": None if a is None else a.to(DEV)})
    assert got.dtype == x.dtype
    dense_ref.norm_close(got, want_of(x, dense, b, a), dense_ref.sum_rel(x.dtype, K),
                         f"{T} {K} {N} {bits} {group} {dtype}")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("K,N,group", [
    (4, 4, 4), (8, 12, 4), (36, 20, 12), (60, 8, 20), (64, 64, 32), (96, 100, 16), (128, 16, 128),
    (640, 1152, 32), (896, 640, 896), (1000, 132, 200), (1408, 260, 64), (2048, 36, 128),
    (260, 68, 52), (512, 512, 8), (4096, 128, 128)])
def test_shapes(K, N, group, bits, dtype):
    for T in (1, 2, 3, 5):
        check(T, K, N, bits, group, dtype, bias=T != 2, addend=T != 3)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("bits,group", [(4, 32), (4, 128), (4, 20), (8, 640), (8, 64)])
@pytest.mark.parametrize("T", [4, 7, 8, 9, 15, 16, 17, 31, 33, 48, 63, 64, 65, 77, 100, 129, 257, 300])
def test_rows(T, bits, group, dtype):
    check(T, 640, 260, bits, group, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("T,K,N,bits,group", [
    (1000, 512, 1024, 4, 64), (513, 2048, 640, 4, 128), (700, 288, 512, 4, 96),
    (640, 1024, 516, 8, 1024), (520, 1024, 512, 8, 32), (1, 8192, 11264, 4, 64)])
def test_large(T, K, N, bits, group, dtype):
    check(T, K, N, bits, group, dtype)


@pytest.mark.parametrize("T", [1, 6, 40, 300])
def test_values_of_wide_range_f32(T):
    """f32 rows keep their range: values that no 16-bit type holds."""
    x, w, b, a, dense = make(T, 256, 64, 4, 32, "f32", bias=False, addend=False)
    for scale in (1e-30, 1e30):
        xs = x * scale
        got = rt.linearQuant(xs.to(DEV), w, {"bits": 4, "groupSize": 32})
        dense_ref.norm_close(got.cpu() / scale, want_of(xs, dense, None, None) / scale,
                             dense_ref.sum_rel(torch.float32, 256) + 2.0 ** -23)


@pytest.mark.parametrize("T", [1, 6, 40, 300])
def test_small_f16_values(T):
    """Subnormal f16 rows count in full: scaled back by the weights."""
    x, w, b, a, dense = make(T, 256, 64, 4, 32, "f16", bias=False, addend=False)
    xs = (x.float() * 2.0 ** -18).half()
    w = rt.QuantExpertWeight(w.w, w.scales * 2.0 ** 18, None)
    got = rt.linearQuant(xs.to(DEV), w, {"bits": 4, "groupSize": 32})
    dense_ref.norm_close(got, want_of(xs, dense * 2.0 ** 18, None, None),
                         dense_ref.sum_rel(torch.float16, 256))


@pytest.mark.parametrize("T", [1, 5, 20, 300])
def test_a_row_of_infinities_stays_alone(T):
    x, w, b, a, dense = make(T, 640, 64, 4, 32, "f16")
    x[T - 1, 77] = float("inf")
    got = rt.linearQuant(x.to(DEV), w, {"bits": 4, "groupSize": 32, "addend": a.to(DEV)})
    assert not torch.isfinite(got[T - 1]).all()
    if T > 1:
        dense_ref.norm_close(got[:T - 1], want_of(x, dense, b, a)[:T - 1],
                             dense_ref.sum_rel(torch.float16, 640))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("T,K,N", [(1, 256, 64), (5, 256, 64), (300, 256, 4096), (600, 4096, 1024)])
def test_an_infinite_value_keeps_the_weights_sign(T, K, N, bits, dtype):
    """inf · q: an infinity of the weight's sign in every column (no weight is zero)."""
    x, w, b, a, dense = make(T, K, N, bits, 32, dtype)
    rng = np.random.default_rng(5)
    q = rng.integers(1, 2 ** (bits - 1), (K, N)) * rng.choice([-1, 1], (K, N))
    q[K - 3, :8] = -(2 ** (bits - 1))
    words = torch.from_numpy(rt.pack_expert_weights(q.astype(np.int8)[None], bits).view(np.int32))
    w = rt.QuantExpertWeight(rt.QuantW(words.to(DEV), (K, N)), w.scales, None)
    x[T - 1, K - 3] = float("inf")
    got = rt.linearQuant(x.to(DEV), w, {"bits": bits, "groupSize": 32}).cpu()
    want = torch.from_numpy(np.sign(q[K - 3]).astype(np.float32)) * float("inf")
    assert torch.equal(got[T - 1].float(), want)
    assert torch.isfinite(got[:T - 1]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("bits,group", [(4, 128), (4, 32), (4, 20), (8, 128), (8, 64)])
@pytest.mark.parametrize("T,K,N", [
    (2, 2560, 1028), (16, 1280, 5000), (17, 640, 8196), (40, 4480, 2052), (96, 3840, 4100),
    (130, 5120, 268), (220, 1920, 1156)])
def test_widths_and_parts(T, K, N, bits, group, dtype):
    """Blocks of every width, x in and out of the LDS, tiles in parts of K."""
    check(T, K, N, bits, group, dtype, bias=T % 2 == 0)


def test_addend_as_out_and_unaligned_tensors():
    lib = _lib.load()
    for dtype in ("f32", "f16"):
        for T in (1, 3, 20, 300):
            x, w, b, a, dense = make(T, 128, 36, 4, 32, dtype)
            print(dtype, T, flush=True)
            want = want_of(x, dense, b, a)
            # every tensor one element past an aligned address
            off = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)]).to(DEV)[1:].view(t.shape)
            words = off(w.w.words.cpu())
            w2 = rt.QuantExpertWeight(rt.QuantW(words, (128, 36)), off(w.scales.cpu()), off(b))
            got = rt.linearQuant(off(x), w2, {"bits": 4, "groupSize": 32, "addend": off(a)})
            dense_ref.norm_close(got, want, dense_ref.sum_rel(x.dtype, 128))
            out = a.to(DEV)
            xd = x.to(DEV)
            wc = _lib.ExpertWeightC(words.data_ptr(), w2.scales.data_ptr(), w2.bias.data_ptr())
            ctx = _lib.thread_context(0, torch.cuda.current_stream().cuda_stream)
            _lib.check(lib.moe_linear_quant(ctx, xd.data_ptr(), 1 if dtype == "f16" else 0,
                                            ctypes.byref(wc), out.data_ptr(), T, 128, 36, 4, 32,
                                            out.data_ptr(), None, 0))
            dense_ref.norm_close(out, want, dense_ref.sum_rel(x.dtype, 128))
            rc = lib.moe_linear_quant(ctx, xd.data_ptr(), 1 if dtype == "f16" else 0,
                                      ctypes.byref(wc), None, T, 128, 36, 4, 32, xd.data_ptr(),
                                      None, 0)
            assert rc == 1 and b"out overlaps x" in lib.moe_last_error()


def test_rows_behind_the_last_are_left():
    for T in (1, 5, 20, 300):
        x, w, b, a, dense = make(T, 128, 36, 4, 32, "f32")
        buf = torch.full((T + 70, 36), 5.0, device=DEV)
        wc = _lib.ExpertWeightC(w.w.words.data_ptr(), w.scales.data_ptr(), w.bias.data_ptr())
        ctx = _lib.thread_context(0, torch.cuda.current_stream().cuda_stream)
        xd = x.to(DEV)
        lib = _lib.load()
        n = ctypes.c_size_t()
        _lib.check(lib.moe_linear_quant_workspace(0, T, 128, 36, 4, 32, ctypes.byref(n)))
        _lib.check(lib.moe_linear_quant(ctx, xd.data_ptr(), 0, ctypes.byref(wc), None, T, 128, 36,
                                        4, 32, buf.data_ptr(), None, 0))
        dense_ref.norm_close(buf[:T], want_of(x, dense, b, None), dense_ref.sum_rel(x.dtype, 128))
        assert (buf[T:] == 5).all()


@pytest.mark.parametrize("bits,groups", [(8, 1), (4, 20)])
def test_quant_linear_equals_linear(bits, groups):
    rng = np.random.default_rng(bits)
    half = 2 ** (bits - 1)
    ints = rng.integers(-half, half, (1152, 640)).astype(np.int8)
    sc = (rng.random((1152, groups)) / (half * 25)).astype(np.float32)
    bias = rng.standard_normal(1152).astype(np.float32)
    a = rt.Linear.from_quant(ints, sc, bits, bias, DEV)
    b = rt.QuantLinear.from_quant(ints, sc, bits, bias, DEV)
    for T in (1, 60, 400):
        x = torch.from_numpy(rng.standard_normal((T, 640)).astype(np.float32)).to(DEV)
        add = torch.from_numpy(rng.standard_normal((T, 1152)).astype(np.float32)).to(DEV)
        p, q = a.forward(x, add), b.forward(x, add)
        assert ((p - q).norm() / p.norm()) <= 2 * dense_ref.sum_rel(torch.float32, 640)
