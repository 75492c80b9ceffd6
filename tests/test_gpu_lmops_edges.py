"""Single roundings, limits and rare states of ah_linear_ce, ah_orthogonalize and ah_muon_step (GPU). Tolerances as in
test_gpu_linear_ce.py and test_gpu_muon.py where none is derived here."""
import numpy as np
import pytest

import test_gpu_linear_ce as TL
from anneal_amd import _lib as L

pytestmark = pytest.mark.gpu
U16, U32 = 2.0 ** -11, 2.0 ** -24


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("D,N", [(64, 1), (64, 140), (72, 3), (65, 2)])
def test_f16_gradients_round_p_once(dev, D, N, bias):
    """dW of one row of powers of two: row v is s P_v X exactly, and P_v in f16 needs no second rounding on the way out. So it is within
    half a step of f16 of s P_v X; two roundings would be up to a whole step off. Logits below 4 in f32 move P by (D/32 + 40) U32 * 16."""
    V = 3000
    c = TL.Case(N, D, V, dtype=L.AH_F16, grad_dtype=L.AH_F16, bias=bias, labels=[7] + [-1] * (N - 1))
    c.X[:] = np.where(c.X < 0, -0.5, 0.5)
    got = TL.run(dev, c, want=("loss", "dX", "dW") + (("dbias",) if bias else ()), grad_scale=2.0 ** 12)
    X = c.X[0].astype(np.float64)
    z = c.W.astype(np.float64) @ X + (c.b.astype(np.float64) if bias else 0.0)
    P = np.exp(z - z.max())
    P /= P.sum()
    P[7] -= 1.0
    want = 2.0 ** 12 * P[:, None] * X
    assert np.abs(want).min() > 2.0 ** -14   # f16 has its full 11 bits
    tol = (U16 + (D / 32 + 40) * U32 * 16) * np.abs(want)
    worst = np.abs(got["dW"] - want) / tol
    assert worst.max() <= 1.0, worst.max()


# rows, features, classes, and pieces of how many MiB: tiles of 64 features and more, either sum split, few rows of unaligned W, pieces
LABELLED = [(130, 64, 1000, 0), (777, 96, 3003, 0), (2, 41, 300, 0), (100, 65, 2049, 0), (2500, 64, 200, 0), (150, 264, 20011, 0), (900, 130, 2100, 1),
            (3000, 520, 5003, 0)]


@pytest.mark.parametrize("labels", ["uniform", "few", "one"])
@pytest.mark.parametrize("shape", LABELLED, ids=lambda s: "%dx%dx%d_%d" % s)
def test_f16_gradients_keep_p_at_the_label(dev, shape, labels):
    """P at the label is the largest entry of most rows. It takes part with 22 bits, as f16 and what that leaves, so a gradient is off
    by its own rounding, by U16 of the other entries' share, and by f32 sums: with P at the label in f16 alone it is up to twice as far."""
    N, D, V, mb = shape
    r = np.random.default_rng([N, D])
    y = {"uniform": r.integers(0, V, N), "few": np.exp(r.uniform(0, np.log(V), N)).astype(int) - 1, "one": np.full(N, V // 2)}[labels]
    if N > 2:
        y[r.random(N) < 0.2] = -1
    c = TL.Case(N, D, V, dtype=L.AH_F16, grad_dtype=L.AH_F16, labels=y, bias=False)
    s = 2.0 ** 10
    got = TL.run(dev, c, want=("loss", "dX", "dW"), mean=False, grad_scale=s, piece_mb=mb)
    X, W, on = c.X.astype(np.float64), c.W.astype(np.float64), np.flatnonzero(y >= 0)
    X = X[on]
    z = X @ W.T
    p = np.exp(z - z.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    at = np.arange(len(on)), y[on]
    dz = (np.abs(X) @ np.abs(W).T).max(1, keepdims=True) * (D / 32 + 32) * U32
    dP = p * (3 * dz + (V / 64 + 40) * U32 + 2.0 ** -20) + U16 * p   # the logits, the statistics, exp; f16
    P = p.copy()
    P[at] -= 1.0
    dP[at] = p[at] * (3 * dz[:, 0] + (V / 64 + 40) * U32 + 2.0 ** -20) + 2.0 ** -21 * np.abs(P[at])
    dP += 2.0 ** -39
    pieces = 4 if mb else 1
    for name, a, da, b in (("dX", P, dP, W), ("dW", P.T, dP.T, X)):
        want = a @ b * s
        tol = s * (da @ np.abs(b) + (a.shape[1] / 32 + 32 * pieces) * U32 * (np.abs(a) @ np.abs(b))) + U16 * 1.01 * np.abs(want) + 2.0 ** -25
        g = got[name][on] if name == "dX" else got[name]
        over = np.abs(want) > 65504 - tol   # past f16's range (many rows of one label): infinite, or the largest value
        assert np.all(np.sign(g[over]) == np.sign(want[over])) and np.all(np.abs(g[over]) >= np.minimum(np.abs(want), 65504)[over] - tol[over])
        worst = np.where(over, 0.0, np.abs(np.where(over, 0.0, g) - want) / tol)
        assert worst.max() <= 1.0, (name, worst.max(), np.argwhere(worst > 1)[:4].tolist())
