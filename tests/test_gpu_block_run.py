"""A residual block's training step as a program runs it (GPU): norm, linear up with GELU, linear down, gated norm onto the residual stream, the
head's loss, every gradient and clipping, through one workspace; eager, captured and on two device handles at once."""
import ctypes as C
import threading

import numpy as np
import pytest
import torch

from anneal_amd import _lib as L
from anneal_amd.backend import Device

pytestmark = pytest.mark.gpu
N, D, F, V, PER = 250, 136, 544, 700, 50
EPS, SCALE, MAX_NORM = 1e-5, 0.5, 0.25
WEIGHTS = {"n1": (1, D), "W1": (F, D), "b1": (1, F), "W2": (D, F), "b2": (1, D), "post": (1, D), "gate": (N // PER, D), "n2": (1, D), "Wv": (V, D)}
# A call's sums lose (K / 4 + 32) 2^-24 of their terms' magnitudes, 2^-16.6 for the longest here, which are up to 24 times the sum's norm (sqrt F for
# random signs); a gradient is the result of eight calls at most: 8 * 24 * 2^-16.6 < 2^-9 of its norm.
TOL = 2.0 ** -9


def values(seed):
    r = np.random.default_rng(seed)
    v = {"H0": 2 * r.standard_normal((N, D)), "W1": D ** -0.5 * r.standard_normal((F, D)), "b1": 0.3 * r.standard_normal((1, F)),
         "W2": F ** -0.5 * r.standard_normal((D, F)), "b2": 0.3 * r.standard_normal((1, D)), "gate": 1 + 0.3 * r.standard_normal((N // PER, D)),
         "Wv": D ** -0.5 * r.standard_normal((V, D))}
    v.update({k: 1 + 0.1 * r.standard_normal((1, D)) for k in ("n1", "post", "n2")})
    v = {k: x.astype(np.float32) for k, x in v.items()}
    v["y"] = r.integers(-70, V, N).astype(np.int32)
    return v


class Step:
    def __init__(self, dev, v):
        self.dev = dev
        b = self.b = {k: dev.buffer(x, L.AH_I32 if k == "y" else L.AH_F32) for k, x in v.items()}
        for k, n in (("O1", N * D), ("Z", N * F), ("A", N * F), ("Y", N * D), ("H1", N * D), ("O2", N * D), ("loss", 1), ("dO2", N * D), ("dH", N * D),
                     ("dY", N * D), ("dA", N * F), ("dO1", N * D), ("norm", 1)):
            b[k] = dev.buffer(n)
        for k, s in WEIGHTS.items():
            b["d" + k], b["c" + k] = dev.buffer(s[0] * s[1]), dev.buffer(s[0] * s[1])
        f = L.AH_F32
        around = dict(dtype=f, N=N, D=D, eps=EPS, scale=SCALE, rows_per_gate=PER, post=L.NORM_RMS, pre=L.NORM_RMS, Y=b["Y"], gate=b["gate"], post_w=b["post"], pre_w=b["n2"])
        first = dict(dtype=f, N=N, D=D, eps=EPS, pre=L.NORM_RMS, pre_w=b["n1"])
        self.calls = [
            ("residual_norm", dict(first, H=b["H0"], O=b["O1"])),
            ("linear", dict(dtype=f, N=N, D=D, F=F, act=L.ACT_GELU_TANH, X=b["O1"], W=b["W1"], bias=b["b1"], Y=b["A"], Z=b["Z"])),
            ("linear", dict(dtype=f, N=N, D=F, F=D, X=b["A"], W=b["W2"], bias=b["b2"], Y=b["Y"])),
            ("residual_norm", dict(around, H=b["H0"], H_out=b["H1"], O=b["O2"])),
            ("linear_ce", dict(dtype=f, N=N, D=D, V=V, X=b["O2"], W=b["Wv"], labels=b["y"], loss=b["loss"], dX=b["dO2"], dW=b["dWv"])),
            ("residual_norm_grad", dict(around, H_out=b["H1"], dO=b["dO2"], dH=b["dH"], dY=b["dY"], dgate=b["dgate"], dpost_w=b["dpost"], dpre_w=b["dn2"])),
            ("linear_grad", dict(dtype=f, N=N, D=F, F=D, X=b["A"], W=b["W2"], dY=b["dY"], dX=b["dA"], dW=b["dW2"], dbias=b["db2"])),
            ("linear_grad", dict(dtype=f, N=N, D=D, F=F, act=L.ACT_GELU_TANH, X=b["O1"], W=b["W1"], Z=b["Z"], dY=b["dA"], dX=b["dO1"], dW=b["dW1"], dbias=b["db1"])),
            # the stream's gradient takes the first norm's on: dH over dH_out
            ("residual_norm_grad", dict(first, H_out=b["H0"], dH_out=b["dH"], dO=b["dO1"], dH=b["dH"], dpre_w=b["dn1"])),
            ("clip_norm", dict(tensors=dev.tensor_list([(b["d" + k], b["c" + k], s[0] * s[1], f, f) for k, s in WEIGHTS.items()]), norm=b["norm"], max_norm=MAX_NORM)),
        ]
        size = max(getattr(dev, n + "_workspace")(**kw) for n, kw in self.calls if n != "residual_norm")
        self.ws = dev.buffer(size // 4 + 4)

    def run(self):
        for n, kw in self.calls:
            getattr(self.dev, n)(**(kw if n == "residual_norm" else dict(kw, ws=self.ws)))

    def outputs(self):
        self.dev.sync()
        return {k: self.b[k].read() for k in ["loss", "norm", "dH", "O2"] + ["d" + k for k in WEIGHTS] + ["c" + k for k in WEIGHTS]}

    def clear(self):
        for k in ["loss", "norm", "dH", "O2"] + ["d" + k for k in WEIGHTS] + ["c" + k for k in WEIGHTS]:
            self.b[k].write(np.full(self.b[k].nbytes // 4, np.nan, np.float32))

    def free(self):
        for x in list(self.b.values()) + [self.ws]:
            x.free()


def exact(v):
    """Loss, gradients and the clipped ones by differentiation in 64 bits on the CPU."""
    p = {k: torch.tensor(v[k].astype(np.float64), requires_grad=True) for k in ["H0", *WEIGHTS]}
    rms = lambda x, w: x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * w   # noqa: E731
    z = rms(p["H0"], p["n1"]) @ p["W1"].T + p["b1"]
    y = torch.nn.functional.gelu(z, approximate="tanh") @ p["W2"].T + p["b2"]
    h = p["H0"] + SCALE * p["gate"].repeat_interleave(PER, 0) * rms(y, p["post"])
    o = rms(h, p["n2"])
    labels = torch.tensor(v["y"].astype(np.int64))
    on = labels >= 0
    loss = torch.nn.functional.cross_entropy((o @ p["Wv"].T)[on], labels[on])
    loss.backward()
    out = {"loss": loss.item(), "O2": o.detach().numpy(), "dH": p["H0"].grad.numpy()}
    out.update({"d" + k: p[k].grad.numpy() for k in WEIGHTS})
    norm = np.sqrt(sum((out["d" + k] ** 2).sum() for k in WEIGHTS))
    c = min(1.0, MAX_NORM / (norm + 1e-6))
    out.update({"c" + k: c * out["d" + k] for k in WEIGHTS}, norm=norm)
    return out


def check(got, want):
    for k, g in got.items():
        w = np.asarray(want[k], np.float64).ravel()
        d = np.linalg.norm(g.astype(np.float64) - w)
        assert d <= TOL * np.linalg.norm(w), (k, d / np.linalg.norm(w))


def test_block(dev):
    v = values(1)
    s = Step(dev, v)
    s.run()
    check(s.outputs(), exact(v))
    s.free()


def test_captured_and_replayed(dev):
    """Two captured steps that hold one workspace, eager calls between their replays: the bits of the eager step each time."""
    v = [values(2), values(3)]
    s = [Step(dev, x) for x in v]
    s[1].ws.free()
    s[1].ws = s[0].ws
    want, graphs = [], []
    for x in s:
        x.run()
        want.append(x.outputs())
        g = C.c_void_p()
        L.check(dev.lib.ah_graph_begin(dev.h))
        x.run()
        L.check(dev.lib.ah_graph_end(dev.h, C.byref(g)))
        graphs.append(g)
    for turn in range(3):
        for i in ((0, 1), (1, 0), (1, 1))[turn]:
            s[i].clear()
            L.check(dev.lib.ah_graph_replay(dev.h, graphs[i]))
            got = s[i].outputs()
            for k in got:
                np.testing.assert_array_equal(got[k], want[i][k], err_msg=k)
            s[1 - i].run()
    for g in graphs:
        dev.lib.ah_graph_destroy(g)
    dev.sync()
    s[1].ws = dev.buffer(4)
    for x in s:
        x.free()


def test_two_handles_at_once(dev):
    """A step on each of two handles from two threads: the bits of each alone."""
    v = [values(4), values(5)]
    alone = []
    for x in v:
        s = Step(dev, x)
        s.run()
        alone.append(s.outputs())
        s.free()
    got, failed = [None, None], []

    def work(i):
        try:
            d = Device(0)
            s = Step(d, v[i])
            for _ in range(8):
                s.run()
            got[i] = s.outputs()
            s.free()
            d.close()
        except Exception as e:   # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for i in range(2):
        for k in got[i]:
            np.testing.assert_array_equal(got[i][k], alone[i][k], err_msg=k)


@pytest.mark.parametrize("n", [1, 7])
def test_single_tokens(dev, n):
    """A token or a few through norm, gated up projection, down projection onto the stream and norm in f16, against 64 bits."""
    r = np.random.default_rng(n)
    f16 = L.AH_F16
    h = lambda *s: r.standard_normal(s).astype(np.float16)   # noqa: E731
    x = {"H": 2 * h(n, D), "w1": 1 + 0.1 * h(1, D), "Wu": (D ** -0.5 * h(F, D)).astype(np.float16), "Wg": (D ** -0.5 * h(F, D)).astype(np.float16),
         "Wd": (F ** -0.5 * h(D, F)).astype(np.float16), "w2": 1 + 0.1 * h(1, D)}
    b = {k: dev.buffer(v.astype(np.float16), f16) for k, v in x.items()}
    for k, c in (("O", D), ("U", F), ("A", F), ("O2", D)):
        b[k] = dev.buffer(np.full((n, c), np.nan, np.float16), f16)
    up = dict(dtype=f16, N=n, D=D, F=F, X=b["O"])
    down = dict(dtype=f16, N=n, D=F, F=D, X=b["A"], W=b["Wd"], R=b["H"], Y=b["H"])
    gated = dict(up, W=b["Wg"], act=L.ACT_SILU, U=b["U"], Y=b["A"])
    ws = dev.buffer(max(dev.linear_workspace(**k) for k in (dict(up, W=b["Wu"], Y=b["U"]), gated, down)) // 4 + 4)
    dev.residual_norm(dtype=f16, N=n, D=D, pre=L.NORM_RMS, H=b["H"], pre_w=b["w1"], O=b["O"])
    dev.linear(ws=ws, **dict(up, W=b["Wu"], Y=b["U"]))
    dev.linear(ws=ws, **gated)
    dev.linear(ws=ws, **down)
    dev.residual_norm(dtype=f16, N=n, D=D, pre=L.NORM_RMS, H=b["H"], pre_w=b["w2"], O=b["O2"])
    dev.sync()
    v = {k: a.astype(np.float64) for k, a in x.items()}
    rms = lambda a, w: a / np.sqrt((a * a).mean(1, keepdims=True) + 1e-6) * w   # noqa: E731
    o = rms(v["H"], v["w1"])
    z = o @ v["Wg"].T
    a = z / (1 + np.exp(-z)) * (o @ v["Wu"].T)
    stream = v["H"] + a @ v["Wd"].T
    # five arrays are rounded to f16 on the way (2^-11 each), and a product's slope and gate at most double what comes in: 8 * 5 * 2^-11 of the norm
    for k, w in (("H", stream), ("O2", rms(stream, v["w2"]))):
        g = b[k].read().astype(np.float64).reshape(w.shape)
        assert np.linalg.norm(g - w) <= 40 * 2.0 ** -11 * np.linalg.norm(w), k
    for q in list(b.values()) + [ws]:
        q.free()
