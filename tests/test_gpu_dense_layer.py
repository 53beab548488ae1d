"""The dense layer's operators together, as a layer uses them: prompt and
decoded tokens over a cache, on other streams and threads, in graphs, and a
training step."""
import threading

import numpy as np
import pytest
import torch

import runntime_amd as rt
from tests import dense_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
D, QH, KH, HD, I = 256, 6, 2, 64, 416
QW, KW = QH * HD, KH * HD


class Layer:
    """norm → 4-bit qkv → rotary positions → sdpa over a cache → 4-bit out
    (+ x) → norm → gated block (+ x), f16."""

    def __init__(self, seed=0):
        rng = np.random.default_rng(seed)
        f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32))
        self.q = {}
        for n, (k, m) in {"qkv": (D, QW + 2 * KW), "out": (QW, D)}.items():
            ints = rng.integers(-8, 8, (m, k)).astype(np.int8)
            sc = ((0.5 + rng.random((m, k // 32))) / (4.6 * k ** 0.5)).astype(np.float32)
            bias = (0.1 * rng.standard_normal(m)).astype(np.float32)
            self.q[n] = (ints, sc, bias)
        self.lin = {n: rt.QuantLinear.from_quant(*v[:2], 4, v[2], DEV) for n, v in self.q.items()}
        self.n1, self.n2 = ((1 + 0.1 * f(D)).half() for _ in range(2))
        self.w = [(f(D, I) * D ** -0.5).half(), (0.1 * f(I)).half(), (f(D, I) * D ** -0.5).half(),
                  (0.1 * f(I)).half(), (f(I, D) * I ** -0.5).half(), (0.1 * f(D)).half()]
        self.wd = [t.to(DEV) for t in self.w]
        self.n1d, self.n2d = self.n1.to(DEV), self.n2.to(DEV)
        self.freq, amp = rt.ropeFrequencies(32, 10000.0, {"type": "yarn", "factor": 4, "context": 64},
                                            device=DEV)
        self.scale = amp * HD ** -0.25

    def forward(self, x, pos, k_cache, v_cache, at):
        """x [T, D] at cache rows at .. at + T − 1."""
        T = x.shape[0]
        qkv = self.lin["qkv"].forward(rt.rmsNorm(x, self.n1d, 1e-5))
        o = {"headDim": HD, "rotaryDim": 32, "layout": "half", "invFreq": self.freq,
             "scale": self.scale}
        q = rt.ropePositions(qkv, pos, {**o, "width": QW})
        rt.ropePositions(qkv, pos, {**o, "srcStart": QW, "width": KW, "out": k_cache[at:at + T]})
        v_cache[at:at + T] = qkv[:, QW + KW:]
        a = rt.sdpa(q, k_cache[:at + T], v_cache[:at + T],
                    {"qHeads": QH, "kvHeads": KH, "headDim": HD, "windowLeft": float("inf"),
                     "windowRight": 0, "qPosOffset": at})
        x = self.lin["out"].forward(a, x)
        return rt.gatedFfn(rt.rmsNorm(x, self.n2d, 1e-5), *self.wd, {"residual": x})

    def reference(self, x, pos):
        """The whole sequence in 64 bits."""
        norm = lambda v, w: v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-5) * w.double()
        x = x.double()
        T = x.shape[0]
        dw = lambda n: (torch.from_numpy(self.q[n][0]).double() * torch.from_numpy(
            np.repeat(self.q[n][1], 32, 1)).double()).t()
        qkv = norm(x, self.n1) @ dw("qkv") + torch.from_numpy(self.q["qkv"][2]).double()
        f = self.freq.cpu()
        q = dense_ref.rope(qkv[:, :QW], pos, f, self.scale, HD, 32, "half")[0].view(T, QH, HD)
        k = dense_ref.rope(qkv[:, QW:QW + KW], pos, f, self.scale, HD, 32, "half")[0].view(T, KH, HD)
        v = qkv[:, QW + KW:].reshape(T, KH, HD)
        mask = torch.ones(T, T, dtype=torch.bool).tril()
        heads = []
        for h in range(QH):
            s = (q[:, h] @ k[:, h // (QH // KH)].t()).masked_fill(~mask, float("-inf"))
            heads.append(torch.softmax(s, 1) @ v[:, h // (QH // KH)])
        x = x + torch.cat(heads, 1) @ dw("out") + torch.from_numpy(self.q["out"][2]).double()
        return dense_ref.ffn(norm(x, self.n2), *self.w, "swiglu", residual=x)


# Ten f16 roundings on the way (norm, qkv, q/k, attention, sum, norm, h, out and
# the inputs' of two products), each at most 2^-11 of its value, through maps
# that keep relative sizes: as if all fell the same way.
LAYER_REL = 10 * 2.0 ** -11


def seq(T, seed=1):
    return torch.randn((T, D), generator=torch.Generator().manual_seed(seed)).half()


def test_prompt_then_tokens_over_a_cache():
    lay = Layer()
    x = seq(40)
    pos = torch.arange(40) + 1000
    want = lay.reference(x, pos)
    kc, vc = (torch.zeros((48, KW), dtype=torch.float16, device=DEV) for _ in range(2))
    xd, pd = x.to(DEV), pos.to(DEV)
    out = [lay.forward(xd[:33], pd[:33], kc, vc, 0)]
    for t in range(33, 40):
        out.append(lay.forward(xd[t:t + 1], pd[t:t + 1], kc, vc, t))
    dense_ref.norm_close(torch.cat(out), want, LAYER_REL)
    assert not kc[40:].any() and not vc[40:].any()


def test_graphs_replayed_between_eager_calls():
    """Two captured graphs of other sizes, replayed in turn with eager work
    between: each equals its eager result every time."""
    lay = Layer()
    cases = []
    for T, seed in ((1, 5), (70, 6)):
        x = seq(T, seed).to(DEV)
        pos = torch.arange(T, device=DEV)
        kc, vc = (torch.zeros((T, KW), dtype=torch.float16, device=DEV) for _ in range(2))
        eager = lay.forward(x, pos, kc, vc, 0).clone()
        cases.append([x, pos, kc, vc, eager])
    graphs = []
    for c in cases:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            lay.forward(*c[:4], 0)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = lay.forward(*c[:4], 0)
        graphs.append((g, out))
    for n in range(4):
        for (g, out), c in zip(graphs, cases):
            out.zero_()
            g.replay()
            lay.forward(seq(90, n).to(DEV), torch.arange(90, device=DEV),
                        torch.zeros((90, KW), dtype=torch.float16, device=DEV),
                        torch.zeros((90, KW), dtype=torch.float16, device=DEV), 0)
            torch.cuda.synchronize()
            assert torch.equal(out, c[4]), n


def run_all(x, pos, lay):
    """The new operators one after the other, gradients included."""
    y = lay.lin["qkv"].forward(x)
    o = {"headDim": HD, "invFreq": lay.freq, "rotaryDim": 32}
    r = rt.ropePositions(y, pos, o)
    out, saved = rt.gatedFfn(x, *lay.wd, {"save": True})
    back = rt.gatedFfnBackward(out, x, *lay.wd, saved)
    return [y, r, out, rt.ropePositionsBackward(r, pos, o), *back]


@pytest.mark.parametrize("T", [1, 50, 600])
def test_other_streams_and_threads(T):
    """Calls from several threads, each on a stream of its own, at once."""
    lay = Layer()
    pos = torch.arange(T, device=DEV)
    xs = [seq(T, 20 + n).to(DEV) for n in range(3)]
    want = [run_all(x, pos, lay) for x in xs]
    torch.cuda.synchronize()
    got, errors = [None] * 3, []

    def work(n):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(5):
                    got[n] = run_all(xs[n], pos, lay)
            s.synchronize()
        except Exception as e:  # told below
            errors.append(e)

    ts = [threading.Thread(target=work, args=(n,)) for n in range(3)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not errors, errors
    for a, b in zip(got, want):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_training_step_in_a_graph():
    """Forward and backward of the block and of the positions captured once and
    replayed, with the eager step between; and the same twice (no atomics)."""
    lay = Layer()
    T = 130
    x = seq(T, 9).to(DEV)
    pos = torch.arange(T, device=DEV)
    want = run_all(x, pos, lay)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run_all(x, pos, lay)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = run_all(x, pos, lay)
    for _ in range(3):
        [t.zero_() for t in out]
        g.replay()
        again = run_all(x, pos, lay)
        torch.cuda.synchronize()
        for a, b, c in zip(out, want, again):
            assert torch.equal(a, b) and torch.equal(c, b)
