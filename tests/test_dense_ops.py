"""The dense layer's operators without a GPU: refusals (they come before any
device work, so CPU tensors reach them), frequencies, workspace queries, the
packed Linear's weights, and the reference's own gradients by differences."""
import ctypes
import math

import numpy as np
import pytest
import torch

import runntime_amd as rt
from runntime_amd import _lib
from runntime_amd import privacy_filter as pf
from tests import dense_ref


def z(*dims, dtype=torch.float32):
    return torch.zeros(dims, dtype=dtype)


POS = torch.arange(3)
FREQ = torch.ones(4, dtype=torch.float64)
ROPE = {"headDim": 8, "invFreq": FREQ}


@pytest.mark.parametrize("x,pos,opts,msg", [
    (z(3, 16, 1), POS, ROPE, "expected a 2D f32 or f16 tensor"),
    (z(3, 16, dtype=torch.bfloat16), POS, ROPE, "expected a 2D f32 or f16 tensor"),
    (z(3, 16), POS, {**ROPE, "headDim": 1}, "headDim 1 must be an integer of at least 2"),
    (z(3, 18), POS, {**ROPE, "headDim": 9, "rotaryDim": 8}, "need an even headDim"),
    (z(3, 16), POS, {**ROPE, "rotaryDim": 5}, "rotaryDim 5 must be even"),
    (z(3, 16), POS, {**ROPE, "rotaryDim": 10}, "rotaryDim 10 must be even and in 2..headDim 8"),
    (z(3, 16), POS, {**ROPE, "layout": "spiral"}, "layout must be interleaved or half"),
    (z(3, 17), POS, ROPE, "width 17 must be a multiple of headDim 8"),
    (z(3, 16), POS, {**ROPE, "srcStart": 12, "width": 8}, "exceeds 16 input cols"),
    (z(3, 16), POS, {**ROPE, "srcStart": -1}, "srcStart -1 must be a non-negative integer"),
    (z(3, 16), POS.float(), ROPE, "positions must be int32 or int64"),
    (z(3, 16), POS[:2], ROPE, "positions must be int32 or int64"),
    (z(3, 16), POS, {**ROPE, "invFreq": FREQ.float()}, "invFreq must be f64"),
    (z(3, 16), POS, {**ROPE, "invFreq": FREQ[:3]}, "invFreq must be f64"),
    (z(3, 16), POS, {**ROPE, "scale": math.inf}, "scale must be finite"),
    (z(16, 3).t(), POS, ROPE, "dense columns"),
    (z(1, 16).expand(3, 16), POS, ROPE, "rows that do not overlap"),
    (z(3, 16), POS, {**ROPE, "out": z(3, 8)}, "out must be f32"),
    (z(3, 16), POS, {**ROPE, "out": z(3, 16, dtype=torch.float16)}, "out must be f32"),
])
def test_rope_positions_refusals(x, pos, opts, msg):
    for op in (rt.ropePositions, rt.ropePositionsBackward):
        with pytest.raises(ValueError, match=msg):
            op(x, pos, opts)


@pytest.mark.parametrize("args,msg", [
    ((7,), "must be a positive even integer"),
    ((8, -1.0), "theta must be positive"),
    ((8, 1e4, {"type": "cubic"}), "unknown scaling type"),
    ((8, 1e4, {"type": "linear", "factor": 0.5}), "factor must be at least 1"),
    ((2, 1e4, {"type": "ntk", "factor": 2}), "rotaryDim of at least 4"),
    ((8, 1e4, {"type": "yarn", "factor": 2, "context": 64, "alpha": 9, "beta": 3}), "0 < alpha"),
])
def test_rope_frequency_refusals(args, msg):
    with pytest.raises(ValueError, match=msg):
        rt.ropeFrequencies(*args, device="cpu")


def test_rope_frequencies():
    plain, one = rt.ropeFrequencies(64, 10000.0, device="cpu")
    assert one == 1.0 and plain.dtype == torch.float64
    torch.testing.assert_close(plain, 10000.0 ** (-torch.arange(32).double() / 32), rtol=1e-14, atol=0)
    lin, _ = rt.ropeFrequencies(64, 10000.0, {"type": "linear", "factor": 4}, device="cpu")
    torch.testing.assert_close(lin, plain / 4, rtol=1e-14, atol=0)
    ntk, _ = rt.ropeFrequencies(64, 10000.0, {"type": "ntk", "factor": 4}, device="cpu")
    assert ntk[0] == plain[0]
    assert abs(ntk[-1] / plain[-1] - 0.25) < 1e-12
    # the privacy filter's tables from the same description
    f, a = rt.ropeFrequencies(64, 150000.0, {"type": "yarn", "factor": 32, "context": 4096},
                              device="cpu")
    cos, sin = pf.compute_rope_tables(300, 64, 150000.0, 32.0, 1.0, 32.0, 4096)
    ang = torch.arange(300).double()[:, None] * f
    assert (torch.cos(ang) * a - torch.from_numpy(cos)).abs().max() < 1.5e-7
    assert (torch.sin(ang) * a - torch.from_numpy(sin)).abs().max() < 1.5e-7


def qw(k, n, bits=4):
    return rt.QuantW(torch.zeros(k * n * bits // 32, dtype=torch.int32), (k, n))


def quant(k=8, n=8, g=4, bits=4, bias=None, w=None, scales=None):
    return rt.QuantExpertWeight(w or qw(k, n, bits), z(k // g, n) if scales is None else scales, bias)


@pytest.mark.parametrize("x,w,opts,msg", [
    (z(2, 8, 1), quant(), {}, "expected a 2D"),
    (z(2, 8), quant(), {"bits": 3}, "bits must be 8 or 4, got 3"),
    (z(2, 8), quant(k=12), {}, r"w must be a quantW \[8, N\] weight"),
    (z(2, 6), quant(w=qw(6, 8)), {}, "K 6 and N 8 must be multiples of 4"),
    (z(2, 8), quant(w=qw(8, 6)), {}, "K 8 and N 6 must be multiples of 4"),
    (z(2, 8), quant(), {"bits": 8}, "quantW weight elems 8"),
    (z(2, 8), quant(), {"groupSize": 6}, "groupSize 6 must be a multiple of 4"),
    (z(2, 8), quant(), {"groupSize": 12}, "groupSize 12 must be a multiple of 4 that divides K 8"),
    (z(2, 8), quant(scales=z(3, 8)), {}, r"scales must be f32 \[2, 8\]"),
    (z(2, 8), quant(bias=z(7)), {}, r"bias must be f32 \[8\]"),
    (z(2, 8), quant(), {"addend": z(2, 7)}, r"addend must be f32 \[2, 8\]"),
    (z(2, 8), quant(), {"addend": z(2, 8, dtype=torch.float16)}, r"addend must be f32 \[2, 8\]"),
])
def test_linear_quant_refusals(x, w, opts, msg):
    with pytest.raises(ValueError, match=msg):
        rt.linearQuant(x, w, {"bits": 4, "groupSize": 4, **opts})


def ffn_args(d=8, i=12, dtype=torch.float32, **other):
    a = dict(glu_w=z(d, i, dtype=dtype), glu_b=None, lin_w=z(d, i, dtype=dtype), lin_b=None,
             out_w=z(i, d, dtype=dtype), out_b=None)
    a.update(other)
    return a


@pytest.mark.parametrize("x,other,opts,msg", [
    (z(2, 8, 1), {}, {}, "expected a 2D"),
    (z(2, 8), {"glu_w": z(9, 12)}, {}, r"glu weight must be f32 \[8, I\]"),
    (z(2, 8), {"glu_w": z(8, 12, dtype=torch.float16)}, {}, "glu weight must be f32"),
    (z(2, 8), {"lin_w": z(8, 11)}, {}, r"lin weight must be f32 \[8, 12\]"),
    (z(2, 8), {"out_w": z(8, 12)}, {}, r"out weight must be f32 \[12, 8\]"),
    (z(2, 8), {"lin_b": z(8)}, {}, r"lin bias must be f32 \[12\]"),
    (z(2, 8), {"out_b": z(12)}, {}, r"out bias must be f32 \[8\]"),
    (z(2, 8), {}, {"activation": "relu"}, "activation must be one of swiglu"),
])
def test_gated_ffn_refusals(x, other, opts, msg):
    a = ffn_args(**other)
    with pytest.raises(ValueError, match=msg):
        rt.gatedFfn(x, *a.values(), opts)
    with pytest.raises(ValueError, match=msg):
        rt.gatedFfnBackward(z(2, 8), x, *a.values(), z(3, 2, 12), opts)


def test_gated_ffn_refusals_of_one_direction():
    a = ffn_args().values()
    with pytest.raises(ValueError, match=r"residual must be f32 \[2, 8\]"):
        rt.gatedFfn(z(2, 8), *a, {"residual": z(8)})
    with pytest.raises(ValueError, match=r"grad must be f32 \[2, 8\]"):
        rt.gatedFfnBackward(z(2, 9), z(2, 8), *a, z(3, 2, 12))
    with pytest.raises(ValueError, match=r"saved must be f32 \[3, 2, 12\]"):
        rt.gatedFfnBackward(z(2, 8), z(2, 8), *a, z(2, 2, 12))


def test_tensors_off_the_device_are_refused():
    for call in (lambda: rt.ropePositions(z(3, 16), POS, ROPE),
                 lambda: rt.linearQuant(z(2, 8), quant(), {"bits": 4, "groupSize": 4}),
                 lambda: rt.gatedFfn(z(2, 8), *ffn_args().values())):
        with pytest.raises(rt.RunntimeError) as e:
            call()
        assert e.value.code == "INVALID_ARGUMENT"


def test_null_context_and_workspace_queries():
    lib = _lib.load()
    n = ctypes.c_size_t(1)
    assert lib.moe_rope_positions(None, None, 0, 8, 1, 1, 8, 8, 0, None, 32, None, 1.0, 0, None, 8) == 3
    assert lib.moe_linear_quant(None, None, 0, None, None, 1, 8, 8, 4, 4, None, None, 0) == 3
    assert lib.moe_gated_ffn(None, *[None], 0, 0, *[None] * 7, 1, 8, 8, None, None, None, 0) == 3
    assert lib.moe_linear_quant_workspace(0, 5, 64, 64, 4, 32, ctypes.byref(n)) == 0
    assert lib.moe_linear_quant_workspace(0, 5, 64, 64, 5, 32, ctypes.byref(n)) == 1
    assert lib.moe_linear_quant_workspace(0, 0, 64, 64, 4, 32, ctypes.byref(n)) == 1
    assert lib.moe_linear_quant_workspace(2, 1, 64, 64, 4, 32, ctypes.byref(n)) == 1
    assert lib.moe_gated_ffn_workspace(1, 7, 64, 100, 0, ctypes.byref(n)) == 0 and n.value >= 1400
    assert lib.moe_gated_ffn_workspace(1, 7, 64, 100, 1, ctypes.byref(n)) == 0 and n.value >= 2800
    assert lib.moe_gated_ffn_workspace(1, 0, 64, 100, 1, ctypes.byref(n)) == 1


@pytest.mark.parametrize("bits", [4, 8])
def test_quant_linear_packs_the_checkpoint_weight(bits):
    rng = np.random.default_rng(bits)
    half = 2 ** (bits - 1)
    ints = rng.integers(-half, half, (12, 16)).astype(np.int8)       # [out, in]
    scales = rng.random((12, 4)).astype(np.float32)
    lin = rt.QuantLinear.from_quant(ints, scales, bits, None, "cpu")
    assert (lin.in_features, lin.out_features, lin.group_size) == (16, 12, 4)
    v = lin.weight.w.words.numpy().view(np.uint8)
    if bits == 4:
        v = np.stack([v & 15, v >> 4], -1).reshape(-1)
        q = np.where(v > 7, v.astype(np.int16) - 16, v)
    else:
        q = v.view(np.int8)
    q = q.reshape(3, 4, 4, 4).transpose(0, 2, 1, 3).reshape(12, 16)   # [unit][k4][c][r]
    assert np.array_equal(q, ints)
    assert np.array_equal(lin.weight.scales.numpy(), scales.T)
    with pytest.raises(ValueError, match="multiples of 4"):
        rt.QuantLinear.from_quant(ints[:10], scales[:10], bits, None, "cpu")
    with pytest.raises(rt.RunntimeError):
        rt.QuantLinear.from_quant(ints, scales[:, :3], bits, None, "cpu")


@pytest.mark.parametrize("kind", ["swiglu", "clampedSwiglu", "geglu"])
def test_reference_gradients_by_differences(kind):
    g = torch.Generator().manual_seed(3)
    mk = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)
    t = [mk(3, 5), mk(5, 7) * 2, mk(7), mk(5, 7) * 2, mk(7), mk(7, 5), mk(5)]
    dy = mk(3, 5)
    _, grads, _ = dense_ref.ffn(*t, kind, grad=dy)
    for n, gr in enumerate(grads):
        d = mk(*t[n].shape)
        e = 1e-6
        up = [a + e * d if m == n else a for m, a in enumerate(t)]
        dn = [a - e * d if m == n else a for m, a in enumerate(t)]
        diff = ((dense_ref.ffn(*up, kind) - dense_ref.ffn(*dn, kind)) * dy).sum() / (2 * e)
        assert abs(diff - (gr * d).sum()) < 1e-6 * (1 + abs(diff))
