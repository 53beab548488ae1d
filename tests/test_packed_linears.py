"""load_privacy_filter(packed_linears=True): the same network on packed weights."""
import numpy as np
import pytest
import torch

from runntime_amd import privacy_filter as pf
from runntime_amd.linear import Linear, QuantLinear
from runntime_amd.quantw import pack_quant_w
from tests import dense_ref
from tests.test_privacy_filter_load import CLASSES, make_file


def linears(m):
    for b in m.blocks:
        yield b.attn.qkv
        yield b.attn.out
    yield m.unembed


def test_loader_keeps_the_ints(tmp_path):
    p = tmp_path / "m.safetensors"
    raw = make_file(p)
    m = pf.load_privacy_filter(str(p), device="cpu", packed_linears=True)
    assert all(isinstance(v, QuantLinear) for v in linears(m))
    assert all(isinstance(v, Linear) for v in linears(pf.load_privacy_filter(str(p), device="cpu")))
    for b, (qi, qs, qb, oi, os_, ob, _, _) in zip(m.blocks, raw["blocks"]):
        for lin, q, s, bias in ((b.attn.qkv, qi, qs, qb), (b.attn.out, oi, os_, ob)):
            out_f, in_f = q.shape
            assert (lin.in_features, lin.out_features) == (in_f, out_f)
            assert (lin.bits, lin.group_size) == (8, in_f // s.shape[1])
            assert np.array_equal(lin.weight.w.words.numpy().view(np.uint32),
                                  pack_quant_w(q, in_f, out_f, 8))
            assert np.array_equal(lin.weight.scales.numpy(), s.astype(np.float32).T)
            assert np.array_equal(lin.weight.bias.numpy(), bias)
    assert m.unembed.weight.bias is None and m.unembed.out_features == CLASSES


def test_sizes_that_do_not_pack():
    assert QuantLinear.takes(640, 1152, 32)
    assert not QuantLinear.takes(640, 33, 640) and not QuantLinear.takes(642, 32, 642)
    assert not QuantLinear.takes(640, 32, 10)
    with pytest.raises(ValueError, match="multiples of 4"):
        QuantLinear.from_quant(np.zeros((33, 64), np.int8), np.ones((33, 1)), 8, None, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7, 64, 300])
def test_attention_blocks_match(tmp_path, T):
    """Both round their f32 sums of 640 and 896 values. The values v carry qkv's
    relative error e = sum_rel(640); a score q·k of s and its weight exp(s) 2·s·e,
    with |s| < 8 here (q and k of unit variance over 64 columns, scaled); the
    output's sum adds sum_rel(896): 17 e + sum_rel(896), for each of the two."""
    p = tmp_path / "m.safetensors"
    make_file(p)
    m, w = (pf.load_privacy_filter(str(p), device="cuda", packed_linears=k) for k in (True, False))
    cos, sin = (torch.from_numpy(t).cuda() for t in pf.rope_constants(T))
    x = torch.from_numpy(np.random.default_rng(T).standard_normal((T, 640)).astype(np.float32)).cuda()
    f32 = torch.float32
    rel = 2 * (17 * dense_ref.sum_rel(f32, 640) + dense_ref.sum_rel(f32, 896))
    for a, b in zip(m.blocks, w.blocks):
        got, want = a.attn.forward(x, cos, sin), b.attn.forward(x, cos, sin)
        assert got.shape == (T, 640) and torch.isfinite(got).all()
        assert (got - want).norm() <= rel * want.norm()


@pytest.mark.gpu
def test_network_runs_the_same_in_a_graph(tmp_path):
    p = tmp_path / "m.safetensors"
    make_file(p)
    m = pf.load_privacy_filter(str(p), device="cuda", packed_linears=True)
    rng = np.random.default_rng(3)
    g = pf.GraphedForward(m, [64, 17])
    try:
        for t in (64, 17, 64, 17):
            ids = rng.integers(0, 50, size=t)
            got = g(ids).clone()
            want = m.forward(ids)
            assert torch.isfinite(got).all() and torch.equal(got, want)
    finally:
        g.close()
