"""The dense layer's operators on tensors of more than 4 GiB: the rows (columns)
behind that offset equal those of a call on them alone."""
import pytest
import torch

import runntime_amd as rt
from tests import dense_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16 = torch.float16


def near(got, want, *lengths):
    """Two calls' f32 sums of one row, added in another order each."""
    assert got.shape == want.shape and torch.isfinite(got).all()
    err = (got.double() - want.double()).norm()
    assert err <= 2 * dense_ref.sum_rel(got.dtype, *lengths) * want.double().norm()


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_rows(layout):
    T, W = 540_000, 4096
    x = torch.randn(1024, W, device=DEV).to(F16).repeat(T // 1024 + 1, 1)[:T]
    pos = torch.arange(T, device=DEV)
    freq, scale = rt.ropeFrequencies(128)
    o = {"headDim": 128, "layout": layout, "invFreq": freq, "scale": scale}
    got = rt.ropePositions(x, pos, o)
    assert got.numel() * 2 > 1 << 32
    for a in (0, T // 2, T - 70):
        assert torch.equal(got[a:a + 70], rt.ropePositions(x[a:a + 70].contiguous(),
                                                           pos[a:a + 70].contiguous(), o))


def quant(K, N, bits, group):
    words = torch.randint(-(1 << 31), (1 << 31) - 1, (K * N * bits // 32,), dtype=torch.int32,
                          device=DEV)
    sc = torch.rand(K // group, N, device=DEV) * 1e-2
    return rt.QuantExpertWeight(rt.QuantW(words, (K, N)), sc, None)


def test_linear_quant_rows():
    T, K, N = 530_000, 64, 4096
    w = quant(K, N, 4, 32)
    x = torch.randn(T, K, device=DEV).to(F16)
    o = {"bits": 4, "groupSize": 32}
    got = rt.linearQuant(x, w, o)
    assert got.numel() * 2 > 1 << 32
    for a in (0, T // 2, T - 70):
        near(got[a:a + 70], rt.linearQuant(x[a:a + 70].contiguous(), w, o), K)


@pytest.mark.parametrize("T", [1, 20, 200])
@pytest.mark.parametrize("dtype", [torch.float32, F16])
def test_linear_quant_columns(T, dtype):
    K, N, n = 8192, (1 << 20) + 64, 96
    w = quant(K, N, 4, 1024)
    assert w.w.words.numel() * 4 > 1 << 32
    x = torch.randn(T, K, device=DEV).to(dtype)
    o = {"bits": 4, "groupSize": 1024}
    got = rt.linearQuant(x, w, o)
    unit = K // 4 * 2  # words of four columns
    for c in (0, N // 2, N - n):
        part = rt.QuantExpertWeight(
            rt.QuantW(w.w.words[c // 4 * unit:(c + n) // 4 * unit].clone(), (K, n)),
            w.scales[:, c:c + n].contiguous(), None)
        near(got[:, c:c + n], rt.linearQuant(x, part, o), K)


def test_gated_ffn_rows():
    T, d, i = 1_060_000, 16, 2048
    w = [(torch.randn(s, device=DEV) * 0.2).to(F16) for s in ((d, i), (d, i), (i, d))]
    b = [torch.randn(n, device=DEV).to(F16) for n in (i, i, d)]
    x = torch.randn(T, d, device=DEV).to(F16)
    a = (w[0], b[0], w[1], b[1], w[2], b[2])
    got, saved = rt.gatedFfn(x, *a, {"save": True})
    assert saved[0].numel() * 2 > 1 << 32
    for r in (0, T // 2, T - 70):
        want, s = rt.gatedFfn(x[r:r + 70].contiguous(), *a, {"save": True})
        near(got[r:r + 70], want, d, i)
        near(saved[:, r:r + 70], s, d)
    dy = torch.randn(T, d, device=DEV).to(F16)
    dx = rt.gatedFfnBackward(dy, x, *a, saved)[0]
    for r in (0, T // 2, T - 70):
        want = rt.gatedFfnBackward(dy[r:r + 70].contiguous(), x[r:r + 70].contiguous(), *a,
                                   saved[:, r:r + 70].contiguous())[0]
        near(dx[r:r + 70], want, d, 2 * i)


@pytest.mark.parametrize("T", [1, 40])
def test_gated_ffn_weights(T):
    d, i = 4096, 560_000
    g, l = ((torch.randn(256, i, device=DEV) * 0.02).to(F16).repeat(d // 256, 1) for _ in range(2))
    o = (torch.randn(i, 256, device=DEV) * 0.002).to(F16).repeat(1, d // 256)
    assert g.numel() * 2 > 1 << 32
    x = torch.randn(T, d, device=DEV).to(F16)
    y, saved = rt.gatedFfn(x, g, None, l, None, o, None, {"save": True})
    n = 128  # the last columns of the hidden rows, by a block of their own
    _, s = rt.gatedFfn(x, g[:, -n:].contiguous(), None, l[:, -n:].contiguous(), None,
                       o[-n:].contiguous(), None, {"save": True})
    near(saved[:2, :, -n:], s[:2], d)
    near(y, (saved[2].float() @ o.float()).to(F16), i)
