"""The dense layer's operators as they are timed: rotary positions, products with 4- and
8-bit weights, the gated feed-forward block.

    rotary positions   x's heads turned by angles position · frequency, the leading part of a
                       head or all of it, neighbouring or half-split pairs; the gradient turns
                       back
    quantised product  y = x · (q · scale) + bias (+ addend), q a packed int4 or int8 weight
                       with one f32 scale per group of inputs and output
    gated block        y = (act(x·G + g) ⊙ (x·L + l))·O + o (+ residual), and its gradients

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs, weights and frequencies on the GPU, from the seed alone
    run(state)          one pass: `own` false in elementary operations of 32 bits, true
                        through the package's entry points
    work(case)          bytes and operations that a pass cannot do without
    exact(case, seed)   the same result in 64 bits
"""
import math

import torch

own = False
DEV = "cuda"
MOST_FFN = 18.0 * 4096 * 2048 * 5632      # operations of the largest listed block
MOST_QUANT = 2048 * 4096 * 4096           # products of the largest listed quantised product
MOST_ROPE = 4096 * 40 * 128               # values of the largest listed rotation


def listed():
    return [
        # One decoded token's queries and keys (32 + 8 heads) far into a long context.
        dict(name="rope_token_f16", kind="rope", T=1, heads=40, head=128, part=128, pairs="half",
             x="f16", start=130000, packed=False, train=False),
        # A prompt's queries and keys.
        dict(name="rope_prompt_f16", kind="rope", T=4096, heads=40, head=128, part=128,
             pairs="half", x="f16", start=0, packed=False, train=False),
        # A training step on several texts in one batch: the privacy filter's 14 + 2 heads of
        # 64, half of each turned, and the gradient.
        dict(name="rope_train_part_f32", kind="rope", T=1500, heads=16, head=64, part=32,
             pairs="interleaved", x="f32", start=0, packed=True, train=True),
        # One token through a projection of a 4-bit model: the weight stream.
        dict(name="quant_token_f16", kind="quant", T=1, K=4096, N=4096, bits=4, group=128,
             x="f16", bias=False, addend=True),
        # Four sequences' tokens through a wide projection, smaller groups.
        dict(name="quant_tokens4_wide_f16", kind="quant", T=4, K=8192, N=11264, bits=4, group=64,
             x="f16", bias=False, addend=False),
        # One token through the privacy filter's qkv projection, groups of 32, f32.
        dict(name="quant_token_f32", kind="quant", T=1, K=640, N=1152, bits=4, group=32, x="f32",
             bias=True, addend=False),
        # A text through its output projection, 8 bits with one scale a column.
        dict(name="quant_text_int8_f32", kind="quant", T=77, K=896, N=640, bits=8, group=896,
             x="f32", bias=True, addend=True),
        # A prompt through a 4-bit projection.
        dict(name="quant_prompt_f16", kind="quant", T=2048, K=4096, N=4096, bits=4, group=128,
             x="f16", bias=False, addend=False),
        # One token through a dense block: the weight stream.
        dict(name="ffn_token_f16", kind="ffn", T=1, d=4096, I=11264, x="f16", act="swiglu",
             bias=False, residual=True, train=False),
        # A text through one dense expert of the privacy filter's kind.
        dict(name="ffn_text_f32", kind="ffn", T=77, d=640, I=640, x="f32", act="clampedSwiglu",
             bias=True, residual=True, train=False),
        # A ragged batch of prompts.
        dict(name="ffn_prompt_f16", kind="ffn", T=1900, d=2048, I=5632, x="f16", act="geglu",
             bias=False, residual=False, train=False),
        # A training step: the block and all its gradients.
        dict(name="ffn_train_f16", kind="ffn", T=4096, d=2048, I=5632, x="f16", act="swiglu",
             bias=False, residual=False, train=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi, step):
    """A multiple of `step` in [lo, hi], over the logarithm."""
    return max(lo, min(hi, _log_int(rng, lo, hi) // step * step))


def draw(rng):
    kind = rng.choice(["rope", "quant", "quant", "ffn", "ffn"])
    if kind == "rope":
        head = rng.choice([32, 64, 80, 96, 128, 128, 256])
        heads = _log_int(rng, 1, 64)
        part = rng.choice([head, head, head // 2, head // 4])
        T = min(_log_int(rng, 1, 8192), MOST_ROPE // (2 * head * heads))
        return dict(kind=kind, T=max(1, T), heads=heads, head=head, part=part,
                    pairs=rng.choice(["half", "interleaved"]), x=rng.choice(["f16", "f32"]),
                    start=rng.choice([0, _log_int(rng, 1, 1 << 20)]), packed=rng.random() < 0.4,
                    train=rng.random() < 0.4)
    if kind == "quant":
        T = rng.choice([_log_int(rng, 1, 8), _log_int(rng, 1, 2048)])
        group = rng.choice([16, 20, 32, 32, 64, 128, 128, 0])
        K = _size(rng, 256, 8192, group or 4)
        N = _size(rng, 64, 11264, rng.choice([4, 64]))
        T = max(1, min(T, MOST_QUANT // (K * N)))
        return dict(kind=kind, T=T, K=K, N=N, bits=rng.choice([4, 4, 4, 8]), group=group or K,
                    x=rng.choice(["f16", "f16", "f32"]), bias=rng.random() < 0.5,
                    addend=rng.random() < 0.5)
    T = rng.choice([_log_int(rng, 1, 16), _log_int(rng, 1, 4096), _log_int(rng, 64, 4096)])
    d = _size(rng, 128, 4096, rng.choice([64, 64, 8, 1]))
    i = _size(rng, 128, 11264, rng.choice([64, 64, 8, 1]))
    train = rng.random() < 0.4
    T = max(1, min(T, int(MOST_FFN / ((18.0 if train else 6.0) * d * i))))
    return dict(kind=kind, T=T, d=d, I=i, x=rng.choice(["f16", "f16", "f32"]),
                act=rng.choice(["swiglu", "swiglu", "clampedSwiglu", "geglu"]),
                bias=rng.random() < 0.5, residual=rng.random() < 0.5, train=train)


# ------------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 29)
    return g


def _normal(g, dtype, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _frequencies(part):
    """YaRN frequencies for a context stretched 32 times from 4096 (theta 150000, bounds 1 and
    32), and the amplitude that goes with them."""
    half = part // 2
    p = torch.arange(half, dtype=torch.float64, device=DEV)
    plain = 150000.0 ** (-p / half)
    low, high = (half * math.log(4096 / (b * 2 * math.pi)) / math.log(150000.0)
                 for b in (32.0, 1.0))
    ramp = ((p - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
    return plain * (1.0 - ramp) + plain / 32.0 * ramp, 0.1 * math.log(32.0) + 1.0


def prepare(case, seed):
    g = _gen(seed)
    dt = torch.float16 if case["x"] == "f16" else torch.float32
    s = dict(case)
    if case["kind"] == "rope":
        T, width = case["T"], case["heads"] * case["head"]
        s["xs"] = _normal(g, dt, T, width)
        s["dy"] = _normal(g, dt, T, width) if case["train"] else None
        pos = torch.arange(T, device=DEV) + case["start"]
        # several texts in one batch, or tokens of sequences of different lengths
        s["pos"] = torch.remainder(pos * 7919, 4096 + T) if case["packed"] else pos
        s["freq"], s["scale"] = _frequencies(case["part"])
        return s
    if case["kind"] == "quant":
        T, K, N, bits = case["T"], case["K"], case["N"], case["bits"]
        s["xs"] = _normal(g, dt, T, K)
        s["words"] = torch.randint(-(1 << 31), 1 << 31, (K * N * bits // 32,), generator=g,
                                   dtype=torch.int64, device=DEV).to(torch.int32)
        top = 1.0 / ((4.6 if bits == 4 else 74.0) * math.sqrt(K))
        s["scales"] = top * (0.5 + torch.rand((K // case["group"], N), generator=g, device=DEV))
        s["b"] = _normal(g, torch.float32, 1, N, scale=0.1) if case["bias"] else None
        s["add"] = _normal(g, dt, T, N) if case["addend"] else None
        return s
    T, d, i = case["T"], case["d"], case["I"]
    s["xs"] = _normal(g, dt, T, d)
    s["glu"] = _normal(g, dt, d, i, scale=d ** -0.5)
    s["lin"] = _normal(g, dt, d, i, scale=d ** -0.5)
    s["out"] = _normal(g, dt, i, d, scale=i ** -0.5)
    s["glu_b"], s["lin_b"], s["out_b"] = (
        (_normal(g, dt, n, scale=0.1) if case["bias"] else None) for n in (i, i, d))
    s["res"] = _normal(g, dt, T, d) if case["residual"] else None
    # the gradient as it arrives, with the loss scale that half-precision training has
    s["dy"] = _normal(g, dt, T, d, scale=0.25) if case["train"] else None
    return s


# ---------------------------------------------------------------------- run


def _rope_own(s):
    import runntime_amd as rt
    opts = {"headDim": s["head"], "rotaryDim": s["part"], "layout": s["pairs"],
            "invFreq": s["freq"], "scale": s["scale"]}
    y = rt.ropePositions(s["xs"], s["pos"], opts)
    return (y, rt.ropePositionsBackward(s["dy"], s["pos"], opts)) if s["train"] else y


def _turn(x, c, s, head, part, pairs):
    """The pairs of each head's first `part` columns turned by the angles whose cosines and
    sines are c and s [T, part / 2], in 32 bits."""
    v = x.float().reshape(x.shape[0], -1, head)
    p = v[..., :part]
    c, s = c[:, None], s[:, None]
    if pairs == "half":
        a, b = p[..., :part // 2], p[..., part // 2:]
        t = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = p[..., 0::2], p[..., 1::2]
        t = torch.stack([a * c - b * s, b * c + a * s], -1).reshape(p.shape)
    return torch.cat([t, v[..., part:]], -1).reshape(x.shape).to(x.dtype)


def _rope_plain(s):
    angle = s["pos"].double()[:, None] * s["freq"]
    c = (torch.cos(angle) * s["scale"]).float()
    n = (torch.sin(angle) * s["scale"]).float()
    y = _turn(s["xs"], c, n, s["head"], s["part"], s["pairs"])
    return (y, _turn(s["dy"], c, -n, s["head"], s["part"], s["pairs"])) if s["train"] else y


def _quant_own(s):
    import runntime_amd as rt
    w = rt.QuantExpertWeight(rt.QuantW(s["words"], (s["K"], s["N"])), s["scales"], s["b"])
    return rt.linearQuant(s["xs"], w, {"bits": s["bits"], "groupSize": s["group"],
                                       "addend": s["add"]})


def _quant_plain(s):
    K, N = s["K"], s["N"]
    v = s["words"].view(torch.int8)
    if s["bits"] == 4:
        v = torch.stack([(v << 4) >> 4, v >> 4], -1)
    # tiles [unit of 4 columns][4 k], a column's 4 k together
    q = v.reshape(N // 4, K // 4, 4, 4).permute(1, 3, 0, 2).reshape(K, N).float()
    w = (q.reshape(-1, s["group"], N) * s["scales"][:, None]).reshape(K, N)
    y = s["xs"].float() @ w
    y = y if s["b"] is None else y + s["b"]
    y = y if s["add"] is None else y + s["add"].float()
    return y.to(s["xs"].dtype)


def _ffn_own(s):
    import runntime_amd as rt
    w = (s["glu"], s["glu_b"], s["lin"], s["lin_b"], s["out"], s["out_b"])
    if not s["train"]:
        return rt.gatedFfn(s["xs"], *w, {"activation": s["act"], "residual": s["res"]})
    y, saved = rt.gatedFfn(s["xs"], *w, {"activation": s["act"], "residual": s["res"],
                                         "save": True})
    grads = rt.gatedFfnBackward(s["dy"], s["xs"], *w, saved, {"activation": s["act"]})
    return [y, *(t for t in grads if t is not None)]


def _act(kind, g, l):
    """The gated activation of g and l and its derivatives in both, in 32 bits."""
    if kind == "swiglu":
        e = 1.0 / (1.0 + torch.exp(-g))
        return g * e * l, (e + g * e * (1.0 - e)) * l, g * e
    if kind == "geglu":
        p = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * p * l, (p + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)) * l, g * p
    gc, lc = torch.clamp(g, max=7.0), torch.clamp(l, -7.0, 7.0)
    e = 1.0 / (1.0 + torch.exp(-1.702 * gc))
    return (gc * e * (lc + 1.0), (e + 1.702 * gc * e * (1.0 - e)) * (lc + 1.0) * (g <= 7.0),
            gc * e * (l.abs() <= 7.0))


def _ffn_plain(s):
    dt = s["xs"].dtype
    x, gw, lw, ow = (s[n].float() for n in ("xs", "glu", "lin", "out"))
    g, l = x @ gw, x @ lw
    if s["bias"]:
        g, l = g + s["glu_b"].float(), l + s["lin_b"].float()
    h, hg, hl = _act(s["act"], g, l)
    y = h @ ow
    if s["bias"]:
        y = y + s["out_b"].float()
    y = (y if s["res"] is None else y + s["res"].float()).to(dt)
    if not s["train"]:
        return y
    dy = s["dy"].float()
    dh = dy @ ow.t()
    dg, dl = dh * hg, dh * hl
    b = s["bias"]
    grads = [dg @ gw.t() + dl @ lw.t(), x.t() @ dg, dg.sum(0) if b else None, x.t() @ dl,
             dl.sum(0) if b else None, h.t() @ dy, dy.sum(0) if b else None]
    return [y, *(t.to(dt) for t in grads if t is not None)]


def run(state):
    kind = state["kind"]
    if own:
        return {"rope": _rope_own, "quant": _quant_own, "ffn": _ffn_own}[kind](state)
    return {"rope": _rope_plain, "quant": _quant_plain, "ffn": _ffn_plain}[kind](state)


# --------------------------------------------------------------------- work


def work(case):
    b = 2 if case["x"] == "f16" else 4
    T = case["T"]
    if case["kind"] == "rope":
        n = T * case["heads"] * case["head"]
        turned = n * case["part"] / case["head"]
        k = 2 if case["train"] else 1
        return {"bytes": 2.0 * k * n * b + 8.0 * T + 4.0 * case["part"], "flops": 3.0 * k * turned}
    if case["kind"] == "quant":
        K, N = case["K"], case["N"]
        return {"bytes": K * N * case["bits"] / 8 + 4.0 * K // case["group"] * N + T * K * b +
                T * N * b * (2 if case["addend"] else 1) + (4.0 * N if case["bias"] else 0.0),
                "flops": 2.0 * T * K * N}
    d, i = case["d"], case["I"]
    weights, rows = 3.0 * d * i * b, 2.0 * T * d * b + (T * d * b if case["residual"] else 0)
    if case["train"]:
        return {"bytes": 2.0 * weights + rows + 2.0 * T * d * b, "flops": 18.0 * T * d * i}
    return {"bytes": weights + rows, "flops": 6.0 * T * d * i}


# -------------------------------------------------------------------- exact


def _exact_rope(s):
    T, head, part = s["T"], s["head"], s["part"]
    turn = torch.polar(torch.full((), s["scale"], dtype=torch.float64, device=DEV),
                       torch.outer(s["pos"].double(), s["freq"]))[:, None]
    # where the two values of pair p stand in a head
    p = torch.arange(part // 2, device=DEV)
    first, second = (p, p + part // 2) if s["pairs"] == "half" else (2 * p, 2 * p + 1)

    def turned(v, by):
        v = v.double().reshape(T, s["heads"], head)
        z = torch.complex(v[:, :, first], v[:, :, second]) * by
        out = v.clone()
        out[:, :, first], out[:, :, second] = z.real, z.imag
        return out.reshape(T, -1)
    y = turned(s["xs"], turn)
    return (y, turned(s["dy"], turn.conj())) if s["train"] else y


def _exact_quant(s):
    K, N, bits = s["K"], s["N"], s["bits"]
    k = torch.arange(K, device=DEV)[:, None]
    n = torch.arange(N, device=DEV)[None]
    place = ((n // 4) * (K // 4) + k // 4) * 16 + (n % 4) * 4 + k % 4  # of the value
    per = 32 // bits
    v = s["words"][place // per].long() >> (place % per * bits)
    v = (v & ((1 << bits) - 1)).double()
    v = torch.where(v >= 1 << (bits - 1), v - (1 << bits), v)
    y = s["xs"].double() @ (v * s["scales"].double()[torch.arange(K, device=DEV) // s["group"]])
    if s["b"] is not None:
        y = y + s["b"].double()
    return y if s["add"] is None else y + s["add"].double()


def _exact_ffn(s):
    leaf = [None if s[n] is None else s[n].double().requires_grad_(s["train"])
            for n in ("xs", "glu", "glu_b", "lin", "lin_b", "out", "out_b")]
    x, gw, gb, lw, lb, ow, ob = leaf
    g, l = x @ gw, x @ lw
    g, l = (g, l) if gb is None else (g + gb, l + lb)
    if s["act"] == "swiglu":
        h = g * torch.sigmoid(g) * l
    elif s["act"] == "geglu":
        h = 0.5 * g * torch.erfc(-g / math.sqrt(2.0)) * l
    else:
        g = g.clamp(max=7.0)
        h = g * torch.sigmoid(1.702 * g) * (l.clamp(-7.0, 7.0) + 1.0)
    y = h @ ow
    y = y if ob is None else y + ob
    y = y if s["res"] is None else y + s["res"].double()
    if not s["train"]:
        return y
    y.backward(s["dy"].double())
    return [y.detach(), *(t.grad for t in leaf if t is not None)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "quant": _exact_quant, "ffn": _exact_ffn}[case["kind"]](s)
