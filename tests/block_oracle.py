"""The linear layer, the norms around a block and clipping in 64 bits (numpy), with bounds of what the kernels' roundings may add.

u16 = 2^-11 and u32 = 2^-24 are half steps of f16 and f32 relative to the value; a pair of f16 planes leaves 2^-22 of a value, and 2^-39 of
its row's or array's largest magnitude where that is more (f16's smallest step at a scale that brings the largest to 2^14 or more).
"""
import math

import numpy as np
from scipy.special import erf

from anneal_amd import _lib as L

U16, U32, PLANES, FLOOR = 2.0 ** -11, 2.0 ** -24, 2.0 ** -22, 2.0 ** -39
NP = {L.AH_F16: np.float16, L.AH_F32: np.float32}
ACTS = (L.ACT_NONE, L.ACT_RELU, L.ACT_GELU, L.ACT_GELU_TANH, L.ACT_SILU)
_C = math.sqrt(2.0 / math.pi)


def rounded(v, dtype):
    """How far one rounding of v to dtype may be off (f16: 2^-25 among its subnormals)."""
    return U16 * 1.001 * np.abs(v) + 2.0 ** -25 if dtype == L.AH_F16 else U32 * 1.001 * np.abs(v) + 2.0 ** -149


def act(kind, z):
    """act(z) and act'(z)."""
    with np.errstate(all="ignore"):
        if kind == L.ACT_NONE:
            return z, np.ones_like(z)
        if kind == L.ACT_RELU:
            return np.where(z < 0, 0.0, z), (z > 0).astype(np.float64)
        if kind == L.ACT_GELU:
            p = 0.5 * (1.0 + erf(z / math.sqrt(2.0)))
            return z * p, p + z * np.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
        q = np.ones_like(z) if kind == L.ACT_SILU else 2.0 * _C * (1.0 + 0.044715 * z * z)
        dq = np.ones_like(z) if kind == L.ACT_SILU else 2.0 * _C * (1.0 + 3 * 0.044715 * z * z)
        s = 1.0 / (1.0 + np.exp(-z * q))
        return z * s, s + z * s * (1.0 - s) * dq


# What f32 arithmetic leaves of an activation: the share of |z| of act(z), and of 1 + |z| of the slope. exp and rcp are within 2^-22 of their
# values, z times a polynomial of z^2 with an exponent of up to 90 within 2^-21 where it matters; the tail's fit (f16) within 4e-7.
E_ACT, E_SLOPE = 2.0 ** -20, 2.0 ** -19


def sums(K):
    """Share of the sum of magnitudes that an f32 sum of K products may lose: in fours, in chains of K / 4 at most, and a few joins."""
    return (K / 4 + 32) * U32


def linear(X, W, b=None, U=None, R=None, kind=L.ACT_NONE, scale=1.0, dtype=L.AH_F32):
    """{name: (value, bound)} of Y and Z."""
    X, W = X.astype(np.float64), W.astype(np.float64)
    Z = X @ W.T + (0.0 if b is None else b.astype(np.float64))
    mag = np.abs(X) @ np.abs(W).T
    lost = sums(X.shape[1]) + (3 * PLANES if dtype == L.AH_F32 else 0.0)
    dz = lost * mag + 2 * U32 * (np.abs(Z) + (0.0 if b is None else np.abs(b.astype(np.float64))))
    if dtype == L.AH_F32:
        dz = dz + FLOOR * (np.abs(X).max(1)[:, None] * np.abs(W).sum(1) + np.abs(X).sum(1)[:, None] * np.abs(W).max(1))
    a, _ = act(kind, Z)
    u = np.ones_like(Z) if U is None else U.astype(np.float64)
    r = np.zeros_like(Z) if R is None else R.astype(np.float64)
    Y = r + scale * a * u
    dy = np.abs(scale * u) * (1.13 * dz + E_ACT * np.abs(Z)) + 4 * U32 * (np.abs(r) + np.abs(scale * a * u))
    return {"Z": (Z, dz + rounded(Z, dtype)), "Y": (Y, dy + rounded(Y, dtype))}


def linear_grad(X, W, Z, dY, U=None, kind=L.ACT_NONE, scale=1.0, dtype=L.AH_F32, grad_dtype=L.AH_F32):
    X, W, Z, dY = (v.astype(np.float64) for v in (X, W, Z, dY))
    u = np.ones_like(Z) if U is None else U.astype(np.float64)
    a, slope = act(kind, Z)
    t = scale * dY
    dZ = t * u * slope
    e = np.abs(t * u) * E_SLOPE * (1.0 + np.abs(Z) if kind > L.ACT_RELU else 0.0) + 4 * U32 * np.abs(dZ)
    out = {"dU": (t * a, np.abs(t) * E_ACT * np.abs(Z) + 4 * U32 * np.abs(t * a) + rounded(t * a, dtype))}
    mass = np.abs(dZ)
    out["dbias"] = (dZ.sum(0), e.sum(0) + (len(Z) + 8) * U32 * mass.sum(0) + 2.0 ** -149)
    ez = e + (U16 if grad_dtype == L.AH_F16 else PLANES) * mass + FLOOR * mass.max()
    for name, A, eA, B in (("dX", dZ, ez, W), ("dW", dZ.T, ez.T, X)):
        v = A @ B
        lost = sums(A.shape[1]) + (3 * PLANES if dtype == L.AH_F32 else 0.0)
        tol = eA @ np.abs(B) + lost * (np.abs(A) @ np.abs(B)) + rounded(v, grad_dtype)
        if dtype == L.AH_F32:
            tol = tol + FLOOR * np.abs(B).max() * np.abs(A).sum(1)[:, None]
        out[name] = (v, tol)
    return out


# ── norms ──────────────────────────────────────────────────────────────────────

def _share(D):
    """Share of the sum of magnitudes that a row's f32 sum may lose: chains of D / 1024 at most, 8 at least, and trees."""
    return (D / 128 + 64) * U32


def _unit(kind, x, ex, eps):
    """(x - m) r with its bound, r and its share of error; ex: x's own bound."""
    D = x.shape[1]
    if kind == L.NORM_NONE:
        return x, ex, np.ones((len(x), 1)), np.zeros((len(x), 1))
    s = _share(D)
    m = x.mean(1, keepdims=True) if kind == L.NORM_LAYER else np.zeros((len(x), 1))
    em = (s * np.abs(x).mean(1, keepdims=True) + ex.mean(1, keepdims=True)) if kind == L.NORM_LAYER else 0.0
    c = x - m
    ec = ex + em + U32 * np.abs(c)
    v = (c * c).mean(1, keepdims=True)
    ev = s * v + 2 * (np.abs(c) * ec).mean(1, keepdims=True)
    r = 1.0 / np.sqrt(v + eps)
    er = 0.5 * ev / (v + eps) + 4 * U32
    return c * r, ec * r + np.abs(c * r) * (er + 2 * U32), r, er


def _norm(kind, x, ex, eps, w, b):
    if kind == L.NORM_NONE:
        return x, ex
    xh, e, _, _ = _unit(kind, x, ex, eps)
    w = np.ones(x.shape[1]) if w is None else w.astype(np.float64)
    b = np.zeros(x.shape[1]) if b is None else b.astype(np.float64)
    v = xh * w + b
    return v, e * np.abs(w) + 2 * U32 * (np.abs(xh * w) + np.abs(b))


def _gate_rows(gate, per, N, D):
    if gate is None:
        return np.ones((N, D))
    return gate.astype(np.float64)[np.arange(N) // per if per else np.zeros(N, int)]


def residual_norm(H=None, Y=None, gate=None, per=0, post=0, pre=0, post_w=None, post_b=None, pre_w=None, pre_b=None, eps=1e-6, skip=1.0, scale=1.0,
                  dtype=L.AH_F32, res_dtype=L.AH_F32):
    """{name: (value, bound)} of H_out and, with a pre norm, O."""
    N, D = (H if H is not None else Y).shape
    h, e = np.zeros((N, D)), np.zeros((N, D))
    if H is not None:
        h = h + skip * H.astype(np.float64)
        e = e + U32 * np.abs(h)
    if Y is not None:
        u, eu = _norm(post, Y.astype(np.float64), np.zeros((N, D)), eps, post_w, post_b)
        g = scale * _gate_rows(gate, per, N, D)
        h = h + g * u
        e = e + np.abs(g) * eu + 3 * U32 * np.abs(g * u) + U32 * np.abs(h)
    out = {"H_out": (h, e + rounded(h, res_dtype))}
    if pre != L.NORM_NONE:
        o, eo = _norm(pre, h, e, eps, pre_w, pre_b)
        out["O"] = (o, eo + rounded(o, dtype))
    return out


def _norm_back(kind, x, d, ed, eps, w):
    """The gradient of a norm's input with its bound, xh with its bound."""
    D = x.shape[1]
    xh, exh, r, er = _unit(kind, x, np.zeros_like(x), eps)
    if kind == L.NORM_NONE:
        return d, ed, xh, exh
    w = np.ones(D) if w is None else w.astype(np.float64)
    s = _share(D)
    q, eq = d * w, ed * np.abs(w) + U32 * np.abs(d * w)
    qx = (q * xh).mean(1, keepdims=True)
    eqx = (s * np.abs(q * xh) + eq * np.abs(xh) + np.abs(q) * exh).mean(1, keepdims=True)
    v, e = q - qx * xh, eq + eqx * np.abs(xh) + np.abs(qx) * exh
    if kind == L.NORM_LAYER:
        v = v - q.mean(1, keepdims=True)
        e = e + (s * np.abs(q) + eq).mean(1, keepdims=True)
    e = e + 4 * U32 * (np.abs(q) + np.abs(qx * xh) + np.abs(q).mean(1, keepdims=True))
    return r * v, r * e + np.abs(r * v) * (er + 2 * U32), xh, exh


def residual_norm_grad(H_out=None, Y=None, dH_out=None, dO=None, gate=None, per=0, post=0, pre=0, post_w=None, post_b=None, pre_w=None, eps=1e-6,
                       skip=1.0, scale=1.0, dtype=L.AH_F32, res_dtype=L.AH_F32):
    N, D = (dH_out if dH_out is not None else dO).shape
    S = (N + 32) * U32   # sums over rows: chains of N at most
    t, et, out = np.zeros((N, D)), np.zeros((N, D)), {}
    if dH_out is not None:
        t = t + dH_out.astype(np.float64)
    if pre != L.NORM_NONE:
        d = dO.astype(np.float64)
        b, eb, xh, exh = _norm_back(pre, H_out.astype(np.float64), d, np.zeros_like(d), eps, pre_w)
        t, et = t + b, et + eb + 2 * U32 * (np.abs(t) + np.abs(b))
        out["dpre_w"] = ((d * xh).sum(0), (np.abs(d) * exh).sum(0) + S * np.abs(d * xh).sum(0))
        out["dpre_b"] = (d.sum(0), S * np.abs(d).sum(0))
    out["dH"] = (skip * t, np.abs(skip) * et + U32 * np.abs(skip * t) + rounded(skip * t, res_dtype))
    g = _gate_rows(gate, per, N, D)
    v, ev = scale * t, np.abs(scale) * et + U32 * np.abs(scale * t)
    d, ed = v * g, ev * np.abs(g) + 2 * U32 * np.abs(v * g)
    y = np.zeros((N, D)) if Y is None else Y.astype(np.float64)
    b, eb, yh, eyh = _norm_back(post, y, d, ed, eps, post_w)
    out["dY"] = (b, eb + rounded(b, dtype))
    if post != L.NORM_NONE:
        out["dpost_w"] = ((d * yh).sum(0), (np.abs(d) * eyh + ed * np.abs(yh)).sum(0) + S * np.abs(d * yh).sum(0))
        out["dpost_b"] = (d.sum(0), ed.sum(0) + S * np.abs(d).sum(0))
    if Y is not None:
        u, eu = _norm(post, y, np.zeros((N, D)), eps, post_w, post_b)
        k = np.arange(N) // per if per else np.zeros(N, int)
        n = int(k[-1]) + 1
        sg, tol = np.zeros((n, D)), np.zeros((n, D))
        np.add.at(sg, k, v * u)
        np.add.at(tol, k, ev * np.abs(u) + np.abs(v) * eu + S * np.abs(v * u))
        out["dgate"] = (sg, tol + rounded(sg, dtype))
    return out


def compare(got, want):
    """Every value of got within its bound, element by element."""
    for k, g in got.items():
        v, tol = want[k]
        with np.errstate(invalid="ignore"):
            d = np.abs(g.astype(np.float64).reshape(v.shape) - v)
        bad = ~(d <= tol)
        if g.dtype == np.float16:   # what is 65520 or more in magnitude rounds to an infinity
            bad &= ~(np.isinf(g.reshape(v.shape)) & (np.sign(g.reshape(v.shape)) == np.sign(v)) & (np.abs(v) + tol >= 65520.0))
        assert not bad.any(), (k, "worst ratio", float(np.max(d / np.maximum(tol, 1e-300))), "at", np.argwhere(bad)[:4].tolist(), int(bad.sum()), "of", v.size)
