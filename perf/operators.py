"""Timed cases of the training step's two ends: the softmax cross-entropy of a linear head over a large vocabulary, and the
orthogonalised update of a weight matrix.

A case is a dict of plain values with a "kind":
  lce   loss = mean over the counted rows of (log sum_v exp z_v - z_label), z = X W^T + b, without keeping the logits;
        with "grad" also dX, dW and (with a bias) db. "out" lists the gradients' type. Rows whose label is negative do not count.
  orth  O = the k-th Newton-Schulz iterate X <- a X + b (X X^T) X + c (X X^T)^2 X of X = U / (|U| + eps), one matrix or a batch
  muon  one update: M' = mu M + G, U = G + mu M', O as above, W' = (1 - lr wd) W - lr gamma O, and W' in f16 where the case is f16

Sizes are those of the five training configurations of the benchmark and generic ones. Inputs are drawn on the GPU from the
seed. Device memory handed to Device.* calls is torch's; the library's own stream runs the work.
"""
from __future__ import annotations

import math

import torch

own = False

_COEF = (3.4445, -4.7750, 2.0315)
_STEPS = 5
_EPS = 1e-7
_LR, _MU, _WD = 0.02, 0.95, 0.1
_GRAD_SCALE = 1024.0   # the loss scale of a run with f16 gradients
_DEVICE = None


def _dev():
    """One device handle for the process, as a program holds it."""
    global _DEVICE
    if _DEVICE is None:
        from anneal_amd.backend import Device
        _DEVICE = Device(0)
    return _DEVICE


def listed():
    return [
        # the head of a large language model on one accumulation step of 4096 tokens, all f16: the largest vocabulary
        {"name": "lce_f16_n4096_v131072", "kind": "lce", "dtype": "f16", "out": "f16", "grad": True, "bias": False, "N": 4096, "D": 4096, "V": 131072, "skip": 0.0},
        # a medium head; f16 operands whose gradients go to an f32 optimizer; a quarter of the tokens is prompt or padding
        {"name": "lce_f16_f32grad_n8192_v32000", "kind": "lce", "dtype": "f16", "out": "f32", "grad": True, "bias": False, "N": 8192, "D": 2048, "V": 32000, "skip": 0.25},
        # validation: the loss alone
        {"name": "lce_f16_eval_n4096_v50304", "kind": "lce", "dtype": "f16", "out": "f16", "grad": False, "bias": False, "N": 4096, "D": 2048, "V": 50304, "skip": 0.0},
        # f32 training of a small model, an odd vocabulary, a bias, a last partial batch of odd length
        {"name": "lce_f32_n1999_v50257", "kind": "lce", "dtype": "f32", "out": "f32", "grad": True, "bias": True, "N": 1999, "D": 776, "V": 50257, "skip": 0.1},
        # f16, sizes that no tile, no 16-byte load and no stage divides
        {"name": "lce_f16_ragged_n777_d1001_v32003", "kind": "lce", "dtype": "f16", "out": "f16", "grad": True, "bias": True, "N": 777, "D": 1001, "V": 32003, "skip": 0.5},
        # the output layer of the dynamic-batch MLP (2048 -> 512) at batch 7: latency
        {"name": "lce_f32_n7_v512", "kind": "lce", "dtype": "f32", "out": "f32", "grad": True, "bias": True, "N": 7, "D": 2048, "V": 512, "skip": 0.0},
        # the hidden layers of the large f16 MLP: the square one, and the first (4096 x 1024, tall)
        {"name": "orth_f32_4096x4096", "kind": "orth", "dtype": "f32", "out": "f32", "batch": 1, "R": 4096, "C": 4096},
        {"name": "orth_f32_4096x1024", "kind": "orth", "dtype": "f32", "out": "f32", "batch": 1, "R": 4096, "C": 1024},
        # the same projection of twelve layers in one call, f16 gradients
        {"name": "orth_f16_12x512x2048", "kind": "orth", "dtype": "f16", "out": "f16", "batch": 12, "R": 512, "C": 2048},
        # the first layer of the small MLP (784 -> 128): latency
        {"name": "muon_f32_128x784", "kind": "muon", "dtype": "f32", "batch": 1, "R": 128, "C": 784},
        # a hidden weight with an f16 working copy: f16 gradient, f32 master and momentum
        {"name": "muon_f16_2048x8192", "kind": "muon", "dtype": "f16", "batch": 1, "R": 2048, "C": 8192},
        # odd sizes, tall
        {"name": "muon_f32_1537x1021", "kind": "muon", "dtype": "f32", "batch": 1, "R": 1537, "C": 1021},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: mostly multiples of 64 or 8, now and then any number."""
    w, pick = _log(rng, lo, hi), rng.random()
    step = 64 if pick < 0.5 else 8 if pick < 0.8 else 1
    return max(lo, w // step * step)


def draw(rng):
    if rng.random() < 0.5:
        dtype = "f16" if rng.random() < 0.65 else "f32"
        while True:
            n, d, v = _log(rng, 1, 8192), _width(rng, 32, 8192), _width(rng, 64, 131072)
            if n * d * v <= (1 << 40 if dtype == "f16" else 1 << 37) and v * d <= 1 << 29:
                break
        return {"kind": "lce", "dtype": dtype, "out": "f32" if dtype == "f32" or rng.random() < 0.4 else "f16", "grad": rng.random() < 0.8,
                "bias": rng.random() < 0.4, "N": n, "D": d, "V": v, "skip": rng.choice((0.0, 0.1, 0.3, 0.7))}
    while True:
        batch = 1 if rng.random() < 0.6 else rng.randint(2, 16)
        r, c = _width(rng, 8, 8192), _width(rng, 8, 8192)
        if batch * r * c * min(r, c) <= 4096 ** 3:
            break
    if rng.random() < 0.5:
        return {"kind": "muon", "dtype": rng.choice(("f32", "f16")), "batch": batch, "R": r, "C": c}
    dtype = rng.choice(("f32", "f32", "f16"))
    return {"kind": "orth", "dtype": dtype, "out": dtype, "batch": batch, "R": r, "C": c}


# ── inputs ─────────────────────────────────────────────────────────────────────

_TYPES = {"f16": torch.float16, "f32": torch.float32}


def _skipped(case):
    return min(case["N"] - 1, int(round(case["N"] * case["skip"])))


def _lce_inputs(case, g):
    """Hidden states of a half-trained model: unit variance, pulled towards the label's row of W; labels fall off as
    1/rank. The rows that do not count are the first of the batch (prompt) and the last (padding)."""
    N, D, V, t = case["N"], case["D"], case["V"], _TYPES[case["dtype"]]
    rank = torch.rand(N, device="cuda", generator=g)
    labels = torch.floor(V ** rank.double()).long().sub_(1).clamp_(0, V - 1)
    W = torch.empty(V, D, device="cuda", dtype=torch.float32).normal_(generator=g).mul_(1.5 * D ** -0.5).to(t)
    X = torch.randn(N, D, device="cuda", generator=g) + 2.0 * W[labels].float()
    skip = _skipped(case)
    labels[: skip // 2] = -100
    labels[N - (skip - skip // 2):] = -100
    b = torch.randn(V, device="cuda", generator=g).mul_(0.5).to(t) if case["bias"] else None
    return {"X": X.to(t), "W": W, "labels": labels.to(torch.int32), "b": b}


def _gradient(shape, g):
    """A weight gradient: a few strong directions whose strength falls off, over noise, at the scale of a mean loss."""
    B, R, C = shape
    k = min(R, C, 32)
    s = 0.8 ** torch.arange(k, device="cuda", dtype=torch.float32)
    u, v = torch.randn(B, R, k, device="cuda", generator=g), torch.randn(B, k, C, device="cuda", generator=g)
    return (torch.bmm(u * s, v) + 0.3 * torch.randn(B, R, C, device="cuda", generator=g)) * 1e-3


def _update_inputs(case, g):
    shape, t = (case["batch"], case["R"], case["C"]), _TYPES[case["dtype"]]
    p = {"G": _gradient(shape, g).to(t)}
    if case["kind"] == "muon":
        p["M"] = 8.0 * _gradient(shape, g)
        p["W"] = torch.randn(*shape, device="cuda", generator=g) * case["C"] ** -0.5
    return p


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return _lce_inputs(case, g) if case["kind"] == "lce" else _update_inputs(case, g)


class _Buf:
    """Device memory as Device.* calls take it."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


class _State:
    def __init__(self, case, seed):
        self.c, self.p = case, {k: v for k, v in _inputs(case, seed).items() if v is not None}
        self.ws, self.out = None, {}
        new = lambda t, *shape: torch.zeros(*shape, device="cuda", dtype=t)   # noqa: E731
        p, f32 = self.p, torch.float32
        if case["kind"] == "lce":
            self.out = {"loss": new(f32, 1), "rowloss": new(f32, case["N"])}
            if case["grad"]:
                self.out.update(dX=new(_TYPES[case["out"]], *p["X"].shape), dW=new(_TYPES[case["out"]], *p["W"].shape))
                if case["bias"]:
                    self.out["db"] = new(f32, case["V"])
        elif case["kind"] == "orth":
            self.out = {"O": new(_TYPES[case["out"]], *p["G"].shape)}
        else:
            self.out = {"M": new(f32, *p["G"].shape), "W": new(f32, *p["G"].shape)}
            if case["dtype"] == "f16":
                self.out["W16"] = new(torch.float16, *p["G"].shape)


def prepare(case, seed):
    s = _State(case, seed)
    torch.cuda.synchronize()   # the inputs, made on torch's stream, are there before the library's stream reads them
    return s


# ── plain forms: elementary operations in 32 bits, rounded once ────────────────

def _plain_lce(case, p):
    X, W, N = p["X"].float(), p["W"].float(), case["N"]
    z = X @ W.T
    if case["bias"]:
        z += p["b"].float()
    labels = p["labels"].long()
    counted = labels >= 0
    at = torch.where(counted, labels, 0)
    m = z.amax(1, keepdim=True)
    lse = (z - m).exp().sum(1).log() + m[:, 0]
    rowloss = torch.where(counted, lse - z[torch.arange(N, device=z.device), at], 0.0)
    c = counted.sum().clamp(min=1)
    out = {"loss": (rowloss.sum() / c).reshape(1), "rowloss": rowloss}
    if case["grad"]:
        P = (z - lse[:, None]).exp_()
        P[torch.arange(N, device=z.device), at] -= 1.0
        P *= counted[:, None]
        s, t = _scale_of(case) / c, _TYPES[case["out"]]
        out["dX"], out["dW"] = ((P @ W) * s).to(t), ((P.T @ X) * s).to(t)
        if case["bias"]:
            out["db"] = P.sum(0) * s
    return out


def _scale_of(case):
    """f16 gradients carry the loss scale."""
    return _GRAD_SCALE if case["out"] == "f16" else 1.0


def _iterate(X):
    a, b, c = _COEF
    T = X.transpose(1, 2).contiguous()
    if X.shape[1] <= X.shape[2]:
        A = torch.bmm(X, T)
        return a * X + torch.bmm(b * A + c * torch.bmm(A, A), X)
    A = torch.bmm(T, X)
    return a * X + torch.bmm(X, b * A + c * torch.bmm(A, A))


def _orthogonal(U):
    X = U / (U.square().sum((1, 2), keepdim=True).sqrt() + _EPS)
    for _ in range(_STEPS):
        X = _iterate(X)
    return X


def _gamma(case):
    return math.sqrt(max(1.0, case["R"] / case["C"]))


def _plain_update(case, p, G):
    if case["kind"] == "orth":
        return {"O": _orthogonal(G).to(_TYPES[case["out"]])}
    M = _MU * p["M"].to(G.dtype) + G
    W = (1 - _LR * _WD) * p["W"].to(G.dtype) - _LR * _gamma(case) * _orthogonal(G + _MU * M)
    out = {"M": M, "W": W}
    return dict(out, W16=W.half()) if case["dtype"] == "f16" else out


# ── the framework's calls ──────────────────────────────────────────────────────

def _own(s):
    c, dev = s.c, _dev()
    p, o = {k: _Buf(v) for k, v in s.p.items()}, {k: _Buf(v) for k, v in s.out.items()}
    types = {"f16": 1, "f32": 0}   # AH_F16, AH_F32
    if c["kind"] == "lce":
        kw = dict(dtype=types[c["dtype"]], grad_dtype=types[c["out"]], N=c["N"], D=c["D"], V=c["V"], X=p["X"], W=p["W"], bias=p.get("b"),
                  labels=p["labels"], loss=o["loss"], rowloss=o["rowloss"], dX=o.get("dX"), dW=o.get("dW"), dbias=o.get("db"), grad_scale=_scale_of(c))
        need, call = dev.linear_ce_workspace, dev.linear_ce
    else:
        kw = dict(dtype=types[c["dtype"]], rows=c["R"], cols=c["C"], batch=c["batch"], G=p["G"], steps=_STEPS, coef=_COEF, eps=_EPS)
        if c["kind"] == "orth":
            kw.update(out_dtype=types[c["out"]], O=o["O"])
            need, call = dev.orthogonalize_workspace, dev.orthogonalize
        else:
            kw.update(M=p["M"], M_out=o["M"], W=p["W"], W_out=o["W"], W16_out=o.get("W16"), lr=_LR, momentum=_MU, nesterov=True, decay=_WD, scale=_gamma(c))
            need, call = dev.muon_step_workspace, dev.muon_step
    if s.ws is None:
        s.ws = _Buf(torch.empty(max(16, need(**kw)), device="cuda", dtype=torch.uint8))
    call(ws=s.ws, ws_bytes=s.ws.t.numel(), **kw)
    return s.out


def run(state):
    if own:
        return _own(state)
    c, p = state.c, state.p
    return _plain_lce(c, p) if c["kind"] == "lce" else _plain_update(c, p, p["G"].float())


# ── work, 64-bit values ────────────────────────────────────────────────────────

def work(case):
    if case["kind"] == "lce":
        N, D, V = case["N"], case["D"], case["V"]
        n, e, ge = N - _skipped(case), 2 if case["dtype"] == "f16" else 4, 2 if case["out"] == "f16" else 4
        b = e * (n * D + V * D + V * case["bias"]) + 4 * (2 * N + 1)
        if not case["grad"]:
            return {"bytes": b, "flops": 2 * n * D * V}
        return {"bytes": b + ge * (N * D + V * D) + 4 * V * case["bias"], "flops": 6 * n * D * V}
    B, R, C = case["batch"], case["R"], case["C"]
    s, l, e = min(R, C), max(R, C), 2 if case["dtype"] == "f16" else 4
    # X X^T and its square are symmetric: half of each product
    flops = B * _STEPS * (3 * s * s * l + s ** 3)
    per = e + (2 if case["out"] == "f16" else 4) if case["kind"] == "orth" else e + 16 + (2 if e == 2 else 0)
    return {"bytes": per * B * R * C, "flops": flops}


def _exact_lce(case, p):
    """From the definition: the loss as -log softmax, its gradient by the chain rule, a block of rows at a time."""
    W, N, V = p["W"].double(), case["N"], case["V"]
    bias = p["b"].double() if case["bias"] else torch.zeros(V, device=W.device, dtype=torch.float64)
    y = p["labels"].long()
    rows = torch.nonzero(y >= 0)[:, 0]
    rowloss = torch.zeros(N, device=W.device, dtype=torch.float64)
    dX, dW, db = torch.zeros(N, case["D"], device=W.device, dtype=torch.float64), torch.zeros_like(W), torch.zeros_like(bias)
    s = _scale_of(case) / max(1, len(rows))
    block = max(1, (1 << 28) // V)
    for k in range(0, len(rows), block):
        r = rows[k: k + block]
        x = p["X"][r].double()
        logp = torch.log_softmax(torch.addmm(bias, x, W.T), 1)
        rowloss[r] = -logp.gather(1, y[r, None])[:, 0]
        if case["grad"]:
            d = logp.exp_().scatter_add_(1, y[r, None], torch.full((len(r), 1), -1.0, device=W.device, dtype=torch.float64)).mul_(s)
            dX[r] = d @ W
            dW.addmm_(d.T, x)
            db += d.sum(0)
    out = {"loss": rowloss.sum().reshape(1) / max(1, len(rows)), "rowloss": rowloss}
    if case["grad"]:
        out.update(dX=dX, dW=dW)
        if case["bias"]:
            out["db"] = db
    return out


def _exact_orthogonal(U):
    """The odd polynomial applied to the singular values through the short side's Gram matrix, one matrix at a time."""
    a, b, c = _COEF
    got = []
    for u in U:
        x = (u if u.shape[0] <= u.shape[1] else u.T) / (torch.linalg.norm(u) + _EPS)
        eye = torch.eye(x.shape[0], device=x.device, dtype=x.dtype)
        for _ in range(_STEPS):
            q = x @ x.T
            x = (a * eye + q @ (b * eye + c * q)) @ x
        got.append(x if u.shape[0] <= u.shape[1] else x.T)
    return torch.stack(got)


def exact(case, seed):
    p = _inputs(case, seed)
    if case["kind"] == "lce":
        return _exact_lce(case, p)
    G = p["G"].double()
    if case["kind"] == "orth":
        return {"O": _exact_orthogonal(G)}
    M = p["M"].double() * _MU + G
    W = p["W"].double()
    W = W - _LR * (_WD * W + _gamma(case) * _exact_orthogonal(G + _MU * M))
    return dict({"M": M, "W": W}, **({"W16": W} if case["dtype"] == "f16" else {}))
