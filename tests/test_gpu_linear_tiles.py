"""Every kind of tile loop of ah_linear and ah_linear_grad (GPU): the shapes of tile_plans.py, which test_tile_plans.py holds to their tiles. A row of each 64
(for dW, a feature) and the last ones are compared, in all their columns, with 64-bit values under the bounds of block_oracle.py."""
import numpy as np
import pytest

import block_oracle as O
import tile_plans as T
from anneal_amd import _lib as L
from test_gpu_linear import Case

pytestmark = pytest.mark.gpu
DTYPES = {0: L.AH_F32, 1: L.AH_F16}


def sample(n, seed):
    """One of each 64, and the last two."""
    r = np.random.default_rng(seed)
    return np.unique(np.concatenate([np.minimum(np.arange(0, n, 64) + r.integers(0, 64, -(-n // 64)), n - 1), [max(0, n - 2), n - 1]]))


def rows_of(v, rows):
    return None if v is None else v[rows]


@pytest.mark.parametrize("case", T.FORWARD_SHAPES, ids=lambda c: "f%d_%dx%dx%d" % ((16 if c[0] else 32,) + c[1:]))
def test_forward(dev, case):
    dtype, N, D, F = case
    c = Case(N, D, F, dtype=DTYPES[dtype], kind=L.ACT_SILU)
    got, rows = c.forward(dev), sample(N, D)
    want = O.linear(c.X[rows], c.W, c.b, rows_of(c.U, rows), rows_of(c.R, rows), c.kind, c.scale, c.dtype)
    O.compare({k: v[rows] for k, v in got.items()}, want)


@pytest.mark.parametrize("case", T.BACKWARD_SHAPES, ids=lambda c: "f%df%d_%dx%dx%d" % ((16 if c[0] else 32, 16 if c[1] else 32) + c[2:]))
def test_backward(dev, case):
    dtype, grad, N, D, F = case
    c = Case(N, D, F, dtype=DTYPES[dtype], grad_dtype=DTYPES[grad], kind=L.ACT_SILU)
    got = c.backward(dev)
    # the row and the feature of the largest dZ are among those compared: its planes' smallest steps go by that one
    _, slope = O.act(c.kind, c.Z.astype(np.float64))
    at = np.unravel_index(np.argmax(np.abs(c.dY * slope * c.U)), c.dY.shape)
    rows, feats = np.union1d(sample(N, D), at[0]), np.union1d(sample(F, D), at[1])
    args = (c.kind, c.scale, c.dtype, c.grad_dtype)
    want = O.linear_grad(c.X[rows], c.W, c.Z[rows], c.dY[rows], c.U[rows], *args)
    O.compare({"dX": got["dX"][rows], "dU": got["dU"][rows]}, {k: want[k] for k in ("dX", "dU")})
    want = O.linear_grad(c.X, c.W[feats], c.Z[:, feats], c.dY[:, feats], c.U[:, feats], *args)
    O.compare({"dW": got["dW"][feats], "dbias": got["dbias"][0][feats]}, {k: want[k] for k in ("dW", "dbias")})
