"""The dense layer's operators in 64 bits on the CPU, from their formulas, and
the bounds their kernels are held to."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11}


def rope(x, pos, freq, scale, head_dim, rotary, layout, inverse=False):
    """(want, magnitude): magnitude bounds what the roundings act on."""
    v = x.double().reshape(x.shape[0], -1, head_dim)
    ang = pos.double()[:, None] * freq[None]
    c, s = (torch.cos(ang) * scale)[:, None], (torch.sin(ang) * scale)[:, None]
    s = -s if inverse else s
    out, mag = v.clone(), torch.zeros_like(v)
    a = slice(0, rotary, 2) if layout == "interleaved" else slice(0, rotary // 2)
    b = slice(1, rotary, 2) if layout == "interleaved" else slice(rotary // 2, rotary)
    out[..., a] = v[..., a] * c - v[..., b] * s
    out[..., b] = v[..., b] * c + v[..., a] * s
    both = (v[..., a].abs() + v[..., b].abs()) * abs(scale)
    mag[..., a] = both
    mag[..., b] = both
    return out.reshape(x.shape), mag.reshape(x.shape), ang.abs().max().item()


def rope_close(got, want, mag, angle):
    """Each of the two products carries the rounding of its table entry and its
    own (2 · 2^-24), the sum one more, and the angle two of 64 bits; then the
    output's."""
    h = HALF_STEP[got.dtype]
    bound = mag * (4 * 2.0 ** -24 + angle * 2.0 ** -51) + want.abs() * h * (1 + 2.0 ** -10)
    if got.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # half a step of the subnormals
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound + 1e-45).all(), (err - bound).max().item()


def norm_close(got, want, rel, what="", size=None):
    """2-norm of the difference over that of the result (or over `size`, where
    the result is a sum of results that may cancel), and no single value ten
    standard deviations of such an error away."""
    g = got.double().cpu()
    assert g.shape == want.shape, (what, g.shape, want.shape)
    assert torch.isfinite(g).all(), what
    n = want.norm().item() if size is None else size
    err = (g - want).norm().item()
    floor = 1e-7 if got.dtype == torch.float16 else 1e-30  # subnormal steps
    assert err <= rel * n + floor * math.sqrt(want.numel()), (what, err / max(n, 1e-300), rel)
    rms = n / math.sqrt(want.numel())
    worst = ((g - want).abs() - 2 * HALF_STEP[got.dtype] * want.abs()).max().item()
    assert worst <= 10 * rel * rms + 10 * floor, (what, worst, rms)


def sum_rel(dtype, *lengths):
    """Relative 2-norm error of f32 sums of these lengths one after the other:
    a chain of n additions of random roundings of at most half a step drifts by
    less than sqrt(n) half steps; 8 more for products, scales and activations;
    plus the output's rounding."""
    return 2.0 ** -24 * (sum(math.sqrt(n) for n in lengths) + 8) + (
        HALF_STEP[dtype] if dtype == torch.float16 else 0.0)


def act(kind, g, l):
    if kind == "swiglu":
        return g * torch.sigmoid(g) * l
    if kind == "geglu":
        return 0.5 * g * torch.erfc(-g / math.sqrt(2.0)) * l
    g = g.clamp(max=7.0)
    return g * torch.sigmoid(1.702 * g) * (l.clamp(-7.0, 7.0) + 1.0)


def ffn(x, glu_w, glu_b, lin_w, lin_b, out_w, out_b, kind, residual=None, grad=None):
    """y, or (y, gradients of the seven tensors, None where there is no bias,
    and what dx's rounding is relative to). dx is the sum of dg·Gᵀ and dl·Lᵀ: the
    error of either is within a bound of its own norm, so dx's is within that
    bound of the sum of their norms, whatever is left of them in dx (1 × 1 × 1,
    clamped: −0.0749 + 0.0973 = 0.0224, and an error of 1.5 half steps of the
    terms is 12 of the sum)."""
    leaves = [None if t is None else t.detach().double().cpu().requires_grad_(grad is not None)
              for t in (x, glu_w, glu_b, lin_w, lin_b, out_w, out_b)]
    x, gw, gb, lw, lb, ow, ob = leaves
    g, l = x @ gw, x @ lw
    g = g if gb is None else g + gb.reshape(-1)
    l = l if lb is None else l + lb.reshape(-1)
    if grad is not None:
        g.retain_grad(), l.retain_grad()
    y = act(kind, g, l) @ ow
    y = y if ob is None else y + ob.reshape(-1)
    y = y if residual is None else y + residual.double().cpu()
    if grad is None:
        return y
    y.backward(grad.double().cpu())
    size = (g.grad @ gw.detach().t()).norm() + (l.grad @ lw.detach().t()).norm()
    return y.detach(), [None if t is None else t.grad for t in leaves], size.item()
