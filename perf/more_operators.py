"""Timed cases of a residual block of a training step and of the moment before its update: linear layers with bias, activation,
factor and residual in their epilogue, norms fused with gate and residual sum, and clipping by the global gradient norm.

A case is a dict of plain values with a "kind":
  lin       Y = R + s act(z) * U, z = X W^T + b; "keep": z is an output too (a training step's forward pass)
  lin_grad  dZ = s dY * U * act'(z); dX = dZ W, dW = dZ^T X, db = sum dZ, dU = s dY * act(z); "out": type of dX and dW
  norm      u = post(Y), H' = skip H + s gate * u, O = pre(H'); a row of gate serves "per" rows (0: all of them)
  norm_grad from dH' and dO: dH, dY, dgate and the sums over rows for the norms' weights (and biases)
  clip      norm = unscale |G| over all tensors, G'_t = unscale min(1, max_norm / (norm + eps)) G_t

Sizes are those of the training configurations of the benchmark and generic ones. Inputs are drawn on the GPU from the seed.
Device memory handed to Device.* calls is torch's; the library's own stream runs the work.
"""
from __future__ import annotations

import math

import torch

own = False

_EPS = 1e-6
_SKIP, _SCALE = 0.9375, 0.5     # residual scales of a deep network
_UNSCALE, _MAX_NORM = 2.0 ** -10, 1.0   # f16 gradients carry a loss scale of 1024
_DEVICE = None


def _dev():
    """One device handle for the process, as a program holds it."""
    global _DEVICE
    if _DEVICE is None:
        from anneal_amd.backend import Device
        _DEVICE = Device(0)
    return _DEVICE


def _lin(name, dtype, N, D, F, act, bias=False, factor=False, res=False, keep=False):
    return {"name": name, "kind": "lin", "dtype": dtype, "N": N, "D": D, "F": F, "act": act, "bias": bias, "factor": factor, "res": res, "keep": keep}


def _lin_grad(name, dtype, out, N, D, F, act, bias=False, factor=False):
    return {"name": name, "kind": "lin_grad", "dtype": dtype, "out": out, "N": N, "D": D, "F": F, "act": act, "bias": bias, "factor": factor}


def _norm(name, kind, dtype, res, N, D, post, pre, per, gate=True):
    return {"name": name, "kind": kind, "dtype": dtype, "res": res, "N": N, "D": D, "post": post, "pre": pre, "per": per, "gate": gate}


def listed():
    return [
        # the up projection of a large block on 8192 tokens in training: z is kept for the backward pass
        _lin("lin_f16_n8192_d4096_f16384", "f16", 8192, 4096, 16384, "gelu_tanh", bias=True, keep=True),
        # one token through the gated up projection: serving, bound by the weights' bytes
        _lin("lin_f16_n1_d4096_f16384", "f16", 1, 4096, 16384, "silu", factor=True),
        # the down projection onto the residual stream for a small batch of tokens
        _lin("lin_f16_n48_d8192_f2048", "f16", 48, 8192, 2048, "none", bias=True, res=True),
        # f32, sizes that no tile and no 16-byte load divides; a last partial batch
        _lin("lin_f32_ragged_n777_d1001_f2003", "f32", 777, 1001, 2003, "gelu", bias=True, res=True, keep=True),
        # the gradients of a gated up projection, f16 throughout
        _lin_grad("lin_grad_f16_n8192_d2048_f8192", "f16", "f16", 8192, 2048, 8192, "silu", factor=True),
        # a small f32 model's up projection, a last partial batch of odd length
        _lin_grad("lin_grad_f32_n1999_d776_f3104", "f32", "f32", 1999, 776, 3104, "gelu", bias=True),
        # norms on both sides of a block's sum, f16 branches on an f32 residual stream, one gate vector
        _norm("norm_f16_f32_n16384_d4096", "norm", "f16", "f32", 16384, 4096, "rms", "rms", 0),
        # one small batch of the f32 MLP's width: latency
        _norm("norm_f32_n7_d2048", "norm", "f32", "f32", 7, 2048, "none", "layer", 1, gate=False),
        # the same block's backward pass, f16 throughout
        _norm("norm_grad_f16_n16384_d4096", "norm_grad", "f16", "f16", 16384, 4096, "rms", "rms", 0),
        # layer norms, an odd width, a gate for each sequence of 250 tokens
        _norm("norm_grad_f32_n1999_d1001", "norm_grad", "f32", "f32", 1999, 1001, "layer", "layer", 250),
        # all gradients of a 24-layer model of width 1024 (about 350 million), f32
        {"name": "clip_f32_l24_w1024_v50304", "kind": "clip", "dtype": "f32", "layers": 24, "width": 1024, "vocab": 50304},
        # the gradients of the small MLP (784 -> 128 -> 10), f16 to f32: latency
        {"name": "clip_f16_mlp_784_128_10", "kind": "clip", "dtype": "f16", "layers": 0, "width": 128, "vocab": 784},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: mostly multiples of 64 or 8, now and then any number."""
    w, pick = _log(rng, lo, hi), rng.random()
    step = 64 if pick < 0.5 else 8 if pick < 0.8 else 1
    return max(lo, w // step * step)


def draw(rng):
    pick = rng.random()
    dtype = "f16" if rng.random() < 0.65 else "f32"
    if pick < 0.5:
        while True:
            n, d, f = _log(rng, 1, 16384), _width(rng, 32, 8192), _width(rng, 32, 16384)
            if n * d * f <= (1 << 38 if dtype == "f16" else 1 << 35):
                break
        case = {"dtype": dtype, "N": n, "D": d, "F": f, "act": rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")), "bias": rng.random() < 0.5,
                "factor": rng.random() < 0.4}
        if rng.random() < 0.5:
            return dict(case, kind="lin", res=rng.random() < 0.5, keep=rng.random() < 0.5)
        return dict(case, kind="lin_grad", out="f32" if dtype == "f32" or rng.random() < 0.4 else "f16")
    if pick < 0.85:
        while True:
            n, d = _log(rng, 1, 32768), _width(rng, 32, 16384)
            if n * d <= 1 << 26:
                break
        kinds = ("none", "rms", "layer")
        return {"kind": rng.choice(("norm", "norm_grad")), "dtype": dtype, "res": "f32" if dtype == "f32" or rng.random() < 0.5 else "f16", "N": n, "D": d,
                "post": rng.choice(kinds), "pre": rng.choice(kinds[1:]), "per": rng.choice((0, 1, _log(rng, 2, 4096))), "gate": rng.random() < 0.7}
    if rng.random() < 0.3:
        return {"kind": "clip", "dtype": dtype, "layers": 0, "width": _width(rng, 32, 4096), "vocab": _width(rng, 32, 8192)}
    while True:
        layers, width, vocab = rng.randint(1, 32), _width(rng, 64, 2048), _log(rng, 1000, 131072)
        if layers * 12 * width * width + width * vocab <= 1 << 28:
            return {"kind": "clip", "dtype": dtype, "layers": layers, "width": width, "vocab": vocab}


# ── inputs ─────────────────────────────────────────────────────────────────────

_TYPES = {"f16": torch.float16, "f32": torch.float32}


def _clip_shapes(case):
    """A model's parameters: per layer the four projections of a width, two of four widths, biases and norms; with no layers the MLP
    vocab -> width -> 10."""
    w, v = case["width"], case["vocab"]
    if not case["layers"]:
        return [(w, v), (1, w), (10, w), (1, 10)]
    layer = [(w, w)] * 4 + [(4 * w, w), (w, 4 * w), (1, 4 * w)] + [(1, w)] * 9
    return [(v, w)] + layer * case["layers"] + [(1, w)]


def _linear_inputs(case, g):
    """Normed hidden states with a few strong features, weights of unit gain; a tenth of the gradient's rows is padding (zeros), the
    others' sizes differ as losses do. Gradients of f16 carry the loss scale."""
    N, D, F, t = case["N"], case["D"], case["F"], _TYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
    X = randn(N, D)
    X[:, :: max(1, D // 4)] *= 8.0
    p = {"X": X.to(t), "W": (randn(F, D) * D ** -0.5).to(t)}
    if case["factor"]:
        p["U"] = randn(N, F).to(t)
    if case["kind"] == "lin":
        if case["bias"]:
            p["b"] = (0.5 * randn(F)).to(t)
        if case["res"]:
            p["R"] = (2.0 * randn(N, F)).to(t)
        return p
    p["Z"] = (1.2 * randn(N, F)).to(t)
    dY = randn(N, F) * torch.exp(randn(N, 1)) * (1.0 if case["dtype"] == "f16" else 2.0 ** -10)
    p["dY"] = (dY * (torch.rand(N, 1, device="cuda", generator=g) > 0.1)).to(t)
    return p


def _gates(case):
    return 1 if not case["per"] else -(-case["N"] // case["per"])


def _norm_inputs(case, g):
    """A residual stream that has grown over the layers, with strong features; a branch of unit size; weights near one."""
    N, D, t, tr = case["N"], case["D"], _TYPES[case["dtype"]], _TYPES[case["res"]]
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)   # noqa: E731
    H = 3.0 * randn(N, D)
    H[:, :: max(1, D // 4)] *= 8.0
    p = {"H": H.to(tr), "Y": (randn(N, D) + 0.25).to(t)}
    if case["gate"]:
        p["gate"] = (0.5 + 0.25 * randn(_gates(case), D)).to(t)
    for k in ("post", "pre"):
        if case[k] != "none":
            p[k + "_w"] = (1.0 + 0.1 * randn(D)).to(t)
        if case[k] == "layer":
            p[k + "_b"] = (0.1 * randn(D)).to(t)
    if case["kind"] == "norm_grad":
        s = torch.exp(randn(N, 1)) * (1.0 if case["dtype"] == "f16" else 2.0 ** -10)
        s = s * (torch.rand(N, 1, device="cuda", generator=g) > 0.1)
        p["dH"], p["dO"] = (randn(N, D) * s).to(tr), (randn(N, D) * s).to(t)
    return p


def _clip_inputs(case, g):
    """Each tensor's gradient has a size of its own; together they are past the allowed norm."""
    t, scale = _TYPES[case["dtype"]], 1.0 / _UNSCALE if case["dtype"] == "f16" else 1.0
    grads = []
    for s in _clip_shapes(case):
        size = torch.exp(torch.randn(1, device="cuda", generator=g)) * 2e-2
        grads.append((torch.randn(*s, device="cuda", generator=g).mul_(size * scale)).clamp_(-6e4, 6e4).to(t))
    return {"G": grads}


_INPUTS = {"lin": _linear_inputs, "lin_grad": _linear_inputs, "norm": _norm_inputs, "norm_grad": _norm_inputs, "clip": _clip_inputs}


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return _INPUTS[case["kind"]](case, g)


class _Buf:
    """Device memory as Device.* calls take it."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


def _out_shapes(case):
    """Outputs: {name: (type, shape)}."""
    f32, kind, t = torch.float32, case["kind"], _TYPES[case["dtype"]]
    if kind == "clip":
        return {}
    N, D = case["N"], case["D"]
    if kind == "lin":
        F = case["F"]
        return dict({"Y": (t, (N, F))}, **({"Z": (t, (N, F))} if case["keep"] else {}))
    if kind == "lin_grad":
        F, to = case["F"], _TYPES[case["out"]]
        out = {"dX": (to, (N, D)), "dW": (to, (F, D))}
        if case["bias"]:
            out["db"] = (f32, (F,))
        if case["factor"]:
            out["dU"] = (t, (N, F))
        return out
    tr = _TYPES[case["res"]]
    if kind == "norm":
        return {"H": (tr, (N, D)), "O": (t, (N, D))}
    out = {"dH": (tr, (N, D)), "dY": (t, (N, D))}
    if case["gate"]:
        out["dgate"] = (t, (_gates(case), D))
    for k in ("post", "pre"):
        if case[k] != "none":
            out["d" + k + "_w"] = (f32, (D,))
        if case[k] == "layer":
            out["d" + k + "_b"] = (f32, (D,))
    return out


class _State:
    def __init__(self, case, seed):
        self.c, self.p = case, _inputs(case, seed)
        self.out = {k: torch.zeros(*s, device="cuda", dtype=t) for k, (t, s) in _out_shapes(case).items()}
        if case["kind"] == "clip":
            # the clipped gradients lie one after the other in one array, as an optimizer's state does
            self.out = {"G": torch.zeros(sum(v.numel() for v in self.p["G"]), device="cuda"), "norm": torch.zeros(1, device="cuda")}
            self.at = torch.split(self.out["G"], [v.numel() for v in self.p["G"]])
        self.ws = self.list = None


def prepare(case, seed):
    s = _State(case, seed)
    torch.cuda.synchronize()   # the inputs, made on torch's stream, are there before the library's stream reads them
    return s


# ── plain forms: elementary operations in 32 bits, rounded once ────────────────

def _act(act, z):
    if act == "none":
        return z
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z / (1.0 + torch.exp(-z))


def _act_slope(act, z):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0.0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s + z * s * (1.0 - s)


def _plain_lin(case, p):
    t = _TYPES[case["dtype"]]
    z = p["X"].float() @ p["W"].float().T
    if case["bias"]:
        z = z + p["b"].float()
    y = _act(case["act"], z)
    if case["factor"]:
        y = y * p["U"].float()
    y = _SCALE * y
    if case["res"]:
        y = y + p["R"].float()
    return dict({"Y": y.to(t)}, **({"Z": z.to(t)} if case["keep"] else {}))


def _plain_lin_grad(case, p):
    t, to = _TYPES[case["dtype"]], _TYPES[case["out"]]
    z, dy = p["Z"].float(), _SCALE * p["dY"].float()
    dz = dy * _act_slope(case["act"], z)
    out = {}
    if case["factor"]:
        dz = dz * p["U"].float()
        out["dU"] = (dy * _act(case["act"], z)).to(t)
    out["dX"], out["dW"] = (dz @ p["W"].float()).to(to), (dz.T @ p["X"].float()).to(to)
    if case["bias"]:
        out["db"] = dz.sum(0)
    return out


def _unit(kind, x):
    """The normed rows without weights, and the factor that normed them."""
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    r = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + _EPS)
    return x * r, r


def _normed(case, p, k, x):
    if case[k] == "none":
        return x
    v = _unit(case[k], x)[0] * p[k + "_w"].float()
    return v + p[k + "_b"].float() if case[k] == "layer" else v


def _gate_rows(case, p):
    if case["gate"]:
        g = p["gate"].float()
        return g if g.shape[0] == 1 else torch.repeat_interleave(g, case["per"], 0)[: case["N"]]
    return 1.0


def _plain_norm(case, p):
    u = _normed(case, p, "post", p["Y"].float())
    h = _SKIP * p["H"].float() + _SCALE * _gate_rows(case, p) * u
    return {"H": h.to(_TYPES[case["res"]]), "O": _normed(case, p, "pre", h).to(_TYPES[case["dtype"]])}


def _norm_back(case, p, k, x, d, out):
    """The gradient of a norm's input from its output's, and its weights'."""
    if case[k] == "none":
        return d
    xh, r = _unit(case[k], x)
    out["d" + k + "_w"] = (d * xh).sum(0)
    if case[k] == "layer":
        out["d" + k + "_b"] = d.sum(0)
    g = d * p[k + "_w"].float()
    back = g - xh * (g * xh).mean(1, keepdim=True)
    if case[k] == "layer":
        back = back - g.mean(1, keepdim=True)
    return back * r


def _plain_norm_grad(case, p):
    t, out = _TYPES[case["dtype"]], {}
    y = p["Y"].float()
    d = p["dH"].float() + _norm_back(case, p, "pre", p["H"].float(), p["dO"].float(), out)
    out["dH"] = (_SKIP * d).to(_TYPES[case["res"]])
    d = _SCALE * d
    if case["gate"]:
        dg = d * _normed(case, p, "post", y)
        per = case["per"] or case["N"]
        rows = _gates(case) * per
        if rows > case["N"]:
            dg = torch.cat([dg, torch.zeros(rows - case["N"], dg.shape[1], device=dg.device)])
        out["dgate"] = dg.view(_gates(case), per, -1).sum(1).to(t)
    out["dY"] = _norm_back(case, p, "post", y, d * _gate_rows(case, p), out).to(t)
    return out


def _unscale(case):
    return _UNSCALE if case["dtype"] == "f16" else 1.0


def _plain_clip(case, p, out, at):
    s = torch.zeros(1, device="cuda", dtype=torch.float64)
    for g in p["G"]:
        v = g.float()
        s = s + (v * v).sum(dtype=torch.float64)
    norm = _unscale(case) * torch.sqrt(s)
    c = (torch.clamp(_MAX_NORM / (norm + _EPS), max=1.0) * _unscale(case)).float()
    for g, o in zip(p["G"], at):
        torch.mul(g.reshape(-1), c, out=o)
    return dict(out, norm=norm.float())


_PLAIN = {"lin": _plain_lin, "lin_grad": _plain_lin_grad, "norm": _plain_norm, "norm_grad": _plain_norm_grad}


# ── the framework's calls ──────────────────────────────────────────────────────

_AH = {"f32": 0, "f16": 1}                                                        # AH_F32, AH_F16
_ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}              # AH_ACT_*
_NORMS = {"none": 0, "rms": 1, "layer": 2}                                        # AH_NORM_*


def _call(s):
    """The call's name and arguments."""
    c, kind = s.c, s.c["kind"]
    if kind == "clip":
        if s.list is None:
            s.list = _dev().tensor_list([(_Buf(g), _Buf(o), g.numel(), _AH[c["dtype"]], 0) for g, o in zip(s.p["G"], s.at)])
        return "clip_norm", dict(tensors=s.list, norm=_Buf(s.out["norm"]), max_norm=_MAX_NORM, eps=_EPS, unscale=_unscale(c))
    p, o = {k: _Buf(v) for k, v in s.p.items()}, {k: _Buf(v) for k, v in s.out.items()}
    kw = dict(dtype=_AH[c["dtype"]], N=c["N"], D=c["D"], scale=_SCALE)
    if kind == "lin":
        return "linear", dict(kw, F=c["F"], act=_ACTS[c["act"]], X=p["X"], W=p["W"], bias=p.get("b"), U=p.get("U"), R=p.get("R"), Y=o["Y"], Z=o.get("Z"))
    if kind == "lin_grad":
        return "linear_grad", dict(kw, grad_dtype=_AH[c["out"]], F=c["F"], act=_ACTS[c["act"]], X=p["X"], W=p["W"], Z=p["Z"], U=p.get("U"), dY=p["dY"],
                                   dX=o["dX"], dW=o["dW"], dbias=o.get("db"), dU=o.get("dU"))
    kw.update(res_dtype=_AH[c["res"]], Y=p["Y"], gate=p.get("gate"), rows_per_gate=c["per"], post=_NORMS[c["post"]], pre=_NORMS[c["pre"]], eps=_EPS, skip=_SKIP)
    kw.update({k: p.get(k) for k in ("post_w", "post_b", "pre_w")})
    if kind == "norm":
        return "residual_norm", dict(kw, pre_b=p.get("pre_b"), H=p["H"], H_out=o["H"], O=o["O"])
    kw.update({k: o.get(k) for k in ("dH", "dY", "dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b")})
    return "residual_norm_grad", dict(kw, H_out=p["H"], dH_out=p["dH"], dO=p["dO"])


def _own(s):
    name, kw = _call(s)
    dev = _dev()
    if name != "residual_norm":   # needs no workspace
        if s.ws is None:
            s.ws = _Buf(torch.empty(max(16, getattr(dev, name + "_workspace")(**kw)), device="cuda", dtype=torch.uint8))
        kw.update(ws=s.ws, ws_bytes=s.ws.t.numel())
    getattr(dev, name)(**kw)
    return s.out


def run(state):
    if own:
        return _own(state)
    if state.c["kind"] == "clip":
        return _plain_clip(state.c, state.p, state.out, state.at)
    return _PLAIN[state.c["kind"]](state.c, state.p)


# ── work, 64-bit values ────────────────────────────────────────────────────────

def work(case):
    e, kind = 2 if case["dtype"] == "f16" else 4, case["kind"]
    if kind == "clip":
        n = sum(r * c for r, c in _clip_shapes(case))
        return {"bytes": n * (e + 4) + 4, "flops": 3 * n}
    N, D = case["N"], case["D"]
    if kind == "lin":
        F = case["F"]
        arrays = 1 + case["factor"] + case["res"] + case["keep"]
        return {"bytes": e * (N * D + F * D + F * case["bias"] + arrays * N * F), "flops": 2 * N * D * F}
    if kind == "lin_grad":
        F, eo = case["F"], 2 if case["out"] == "f16" else 4
        return {"bytes": e * (N * D + F * D + (2 + 2 * case["factor"]) * N * F) + eo * (N * D + F * D) + 4 * F * case["bias"], "flops": 4 * N * D * F}
    er = 2 if case["res"] == "f16" else 4
    gate, weights = _gates(case) * D * case["gate"], D * sum({"none": 0, "rms": 1, "layer": 2}[case[k]] for k in ("post", "pre"))
    if kind == "norm":
        return {"bytes": 2 * N * D * (e + er) + e * (gate + weights), "flops": 12 * N * D}
    return {"bytes": N * D * 3 * (e + er) + e * (2 * gate + weights) + 4 * weights, "flops": 30 * N * D}


def _exact_act(act, z):
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * z * (1.0 + 0.044715 * z.square()))
    return z * torch.sigmoid(z) if act == "silu" else torch.relu(z) if act == "relu" else z


def _exact_lin(case, p):
    """A block of rows at a time."""
    out = {k: torch.empty(*s, device="cuda", dtype=torch.float64) for k, (_, s) in _out_shapes(case).items()}
    W, block = p["W"].double(), max(1, (1 << 27) // case["F"])
    for k in range(0, case["N"], block):
        r = slice(k, k + block)
        z = torch.addmm(p["b"].double(), p["X"][r].double(), W.T) if case["bias"] else torch.mm(p["X"][r].double(), W.T)
        if case["keep"]:
            out["Z"][r] = z
        y = _exact_act(case["act"], z)
        if case["factor"]:
            y = y * p["U"][r].double()
        out["Y"][r] = torch.add(p["R"][r].double(), y, alpha=_SCALE) if case["res"] else _SCALE * y
    return out


def _exact_lin_grad(case, p):
    """By the chain rule that autograd applies to the definition, a block of rows at a time."""
    out = {k: torch.zeros(*s, device="cuda", dtype=torch.float64) for k, (_, s) in _out_shapes(case).items()}
    W, block = p["W"].double(), max(1, (1 << 27) // case["F"])
    for k in range(0, case["N"], block):
        r = slice(k, k + block)
        with torch.enable_grad():
            z = p["Z"][r].double().requires_grad_()
            u = p["U"][r].double().requires_grad_() if case["factor"] else None
            y = _SCALE * _exact_act(case["act"], z * 1.0)
            got = torch.autograd.grad(y if u is None else y * u, [z] if u is None else [z, u], p["dY"][r].double())
        out["dX"][r] = got[0] @ W
        out["dW"].addmm_(got[0].T, p["X"][r].double())
        if case["bias"]:
            out["db"] += got[0].sum(0)
        if case["factor"]:
            out["dU"][r] = got[1]
    return out


def _exact_sum(case, q, h):
    """H' and O from 64-bit leaves; h: H' itself, where it is given."""
    def norm(k, x):
        if case[k] == "none":
            return x
        if case[k] == "layer":
            return torch.nn.functional.layer_norm(x, x.shape[1:], eps=_EPS) * q[k + "_w"] + q[k + "_b"]
        return x * torch.rsqrt(x.square().mean(1, keepdim=True) + _EPS) * q[k + "_w"]
    u = norm("post", q["Y"])
    if case["gate"]:
        rows = torch.arange(case["N"], device=u.device)
        u = u * q["gate"][torch.div(rows, case["per"], rounding_mode="floor") if case["per"] else torch.zeros_like(rows)]
    s = _SKIP * q["H"] + _SCALE * u
    return s, norm("pre", s if h is None else h + (s - s.detach()))


def _exact_norm(case, p):
    with torch.no_grad():
        H, O = _exact_sum(case, {k: v.double() for k, v in p.items()}, None)
    return {"H": H, "O": O}


def _exact_norm_grad(case, p):
    """The value of H' is the given one; the derivatives run through the sum."""
    names = [k for k in ("H", "Y", "gate", "post_w", "post_b", "pre_w", "pre_b") if k in p]
    with torch.enable_grad():
        q = {k: p[k].double().requires_grad_() for k in names}
        H, O = _exact_sum(case, q, p["H"].double())
        got = torch.autograd.grad([H, O], [q[k] for k in names], [p["dH"].double(), p["dO"].double()])
    return {"d" + k: v for k, v in zip(names, got)}


def _exact_clip(case, p):
    norm = torch.stack([torch.linalg.vector_norm(g.double()) for g in p["G"]]).norm().reshape(1) * _unscale(case)
    c = torch.minimum(torch.ones_like(norm), _MAX_NORM / (norm + _EPS))
    return {"G": torch.cat([(g.double() * (c * _unscale(case))).reshape(-1) for g in p["G"]]), "norm": norm}


def exact(case, seed):
    p = _inputs(case, seed)
    got = {"lin": _exact_lin, "lin_grad": _exact_lin_grad, "norm": _exact_norm, "norm_grad": _exact_norm_grad, "clip": _exact_clip}[case["kind"]](case, p)
    if case["kind"] == "clip":
        return got
    return {k: got[k].reshape(s) for k, (_, s) in _out_shapes(case).items()}
