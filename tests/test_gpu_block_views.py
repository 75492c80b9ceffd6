"""Arrays that lie side by side in one (GPU): the halves of a gated unit's [N, 2 F], and the like. Bounds as derived in block_oracle.py."""
import numpy as np
import pytest

import block_oracle as O
from anneal_amd import _lib as L
from test_gpu_linear import IDS, TYPES, Case
from test_gpu_residual_norm import RMS
from test_gpu_residual_norm import Case as NormCase

pytestmark = pytest.mark.gpu


class Beside:
    """Arrays of as many rows in one, `gap` marked elements after each."""

    def __init__(self, dev, arrays, dtype, gap=0):
        self.dtype, self.gap, self.at, c = dtype, gap, [], 0
        for a in arrays:
            self.at.append((c, a.shape[1]))
            c += a.shape[1] + gap
        self.full = np.full((arrays[0].shape[0], c), 777.0, O.NP[dtype])
        for a, (k, w) in zip(arrays, self.at):
            self.full[:, k: k + w] = a
        self.b, self.ld = dev.buffer(self.full, dtype), c

    def view(self, i):
        class View:
            ptr = self.b.ptr + self.at[i][0] * np.dtype(O.NP[self.dtype]).itemsize
        return View

    def read(self, outputs):
        """The arrays `outputs`; all others are as they were."""
        got, rest = self.b.read().reshape(self.full.shape), self.full.copy()
        for i in outputs:
            k, w = self.at[i]
            rest[:, k: k + w] = got[:, k: k + w]
        np.testing.assert_array_equal(got, rest)
        return [got[:, self.at[i][0]: self.at[i][0] + self.at[i][1]] for i in outputs]


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("gap", [0, 1])
@pytest.mark.parametrize("shape", [(1, 64, 96), (5, 40, 33), (40, 100, 65), (200, 72, 131), (8400, 16, 64)], ids=lambda s: "%dx%dx%d" % s)
def test_a_gated_unit_in_one_array(dev, shape, gap, types):
    """Z, U and Y side by side going forward; Z, U, dU and dY going back."""
    N, D, F = shape
    c = Case(N, D, F, dtype=types[0], grad_dtype=types[1], kind=L.ACT_SILU, res=False)
    t = types[0]
    empty = np.full((N, F), np.nan)
    X, W, b = (dev.buffer(v, t) for v in (c.X, c.W, c.b))
    a = Beside(dev, [empty, c.U, empty], t, gap)
    kw = dict(dtype=t, N=N, D=D, F=F, act=c.kind, scale=c.scale, X=X, W=W, bias=b, Z=a.view(0), U=a.view(1), Y=a.view(2), ldz=a.ld, ldu=a.ld, ldy=a.ld)
    ws = dev.buffer(dev.linear_workspace(**kw) // 4 + 4)
    dev.linear(ws=ws, **kw)
    dev.sync()
    z, y = a.read([0, 2])
    O.compare({"Z": z, "Y": y}, c.expected())

    a = Beside(dev, [c.Z, c.U, empty, c.dY], t, gap)
    dX, dW, db = (dev.buffer(np.full(s, np.nan), k) for s, k in (((N, D), types[1]), ((F, D), types[1]), ((1, F), L.AH_F32)))
    kw = dict(dtype=t, grad_dtype=types[1], N=N, D=D, F=F, act=c.kind, scale=c.scale, X=X, W=W, Z=a.view(0), U=a.view(1), dU=a.view(2), dY=a.view(3), ldz=a.ld,
              ldu=a.ld, lddu=a.ld, lddy=a.ld, dX=dX, dW=dW, dbias=db)
    ws = dev.buffer(dev.linear_grad_workspace(**kw) // 4 + 4)
    dev.linear_grad(ws=ws, **kw)
    dev.sync()
    O.compare({"dU": a.read([2])[0], "dX": dX.read().reshape(N, D), "dW": dW.read().reshape(F, D), "dbias": db.read()}, c.gradients())


@pytest.mark.parametrize("gap", [0, 3])
@pytest.mark.parametrize("shape", [(7, 24), (30, 200), (9, 1001), (3, 9000), (2, 17001)], ids=lambda s: "%dx%d" % s)
def test_norms_in_one_array(dev, shape, gap):
    """H, Y, H_out and O side by side, then all that the gradients read and write."""
    N, D = shape
    c = NormCase(N, D, post=RMS, pre=RMS, gate=False)
    empty = np.full((N, D), np.nan)
    w = {k: dev.buffer(v, L.AH_F32) for k, v in c.w.items()}
    a = Beside(dev, [c.H, empty, c.Y, empty], L.AH_F32, gap)
    dev.residual_norm(**c.common(), **w, H=a.view(0), H_out=a.view(1), Y=a.view(2), O=a.view(3), ldh=a.ld, ldh_out=a.ld, ldy=a.ld, ldo=a.ld)
    dev.sync()
    h, o = a.read([1, 3])
    O.compare({"H_out": h, "O": o}, c.expected())
    a = Beside(dev, [c.H, empty, c.Y, c.dH_out, empty, c.dO], L.AH_F32, gap)
    kw = dict(**c.common(), **w, H_out=a.view(0), dH=a.view(1), Y=a.view(2), dH_out=a.view(3), dY=a.view(4), dO=a.view(5), ldh_out=a.ld, lddh=a.ld, ldy=a.ld,
              lddh_out=a.ld, lddy=a.ld, lddo=a.ld)
    ws = dev.buffer(dev.residual_norm_grad_workspace(**kw) // 4 + 4)
    dev.residual_norm_grad(ws=ws, **kw)
    dev.sync()
    dh, dy = a.read([1, 4])
    O.compare({"dH": dh, "dY": dy}, c.gradients())
