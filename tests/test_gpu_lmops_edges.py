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
