"""The block operators on arrays of more than 2^31 elements and at their largest numbers of rows (GPU). Large arrays are made on the device by linear
layers; gradients are zeros in all but some rows or features, so that 64-bit values of what is compared come from those. Bounds of block_oracle.py."""
import numpy as np
import pytest

import block_oracle as O
from anneal_amd import _lib as L
from anneal_amd.backend import DeviceBuffer

pytestmark = pytest.mark.gpu
N, D, F = 1 << 21, 40, 1032   # N F is 2.16e9
TYPES = [(L.AH_F16, L.AH_F16), (L.AH_F16, L.AH_F32), (L.AH_F32, L.AH_F32)]
IDS = ["f16", "f16_f32grad", "f32"]
LIVE = np.unique(np.concatenate([np.arange(3), [1000, N // 2, (1 << 31) // F, (1 << 31) // F + 1, (1 << 32) // F // 2 + 2], np.arange(N - 5, N)]))


class Rows:
    """Rows of a large array on the device, read a few at a time."""

    def __init__(self, dev, rows, cols, dtype):
        self.b, self.cols, self.dtype = dev.buffer(rows * cols, dtype), cols, dtype
        self.ptr = self.b.ptr

    def __getitem__(self, rows):
        part = DeviceBuffer.__new__(DeviceBuffer)
        part.dev, part.n, part.dtype = self.b.dev, self.cols, self.dtype
        out = np.empty((len(rows), self.cols), O.NP[self.dtype])
        for i, r in enumerate(rows):
            part.ptr = self.b.ptr + int(r) * self.cols * (2 if self.dtype == L.AH_F16 else 4)
            out[i] = part.read()
        return out


class Kept(list):
    def __call__(self, b):
        self.append(b)
        return b


@pytest.fixture
def keep():
    k = Kept()
    yield k
    for b in k:
        (b.b if isinstance(b, Rows) else b).free()


def linear(dev, keep, **kw):
    dev.linear(ws=keep(dev.buffer(dev.linear_workspace(**kw) // 4 + 4)), **kw)


def sparse(dev, keep, dtype, seed, rows=N, live=LIVE, cols=F):
    """[rows, cols]: zeros but in the rows `live`."""
    r = np.random.default_rng(seed)
    x = np.zeros((rows, 8), O.NP[dtype])
    x[live] = r.standard_normal((len(live), 8))
    out = keep(Rows(dev, rows, cols, dtype))
    linear(dev, keep, dtype=dtype, N=rows, D=8, F=cols, X=keep(dev.buffer(x, dtype)), W=keep(dev.buffer(r.standard_normal((cols, 8)), dtype)), Y=out)
    return out


@pytest.mark.parametrize("types", TYPES, ids=IDS)
def test_linear(dev, keep, types):
    t, g = types
    r = np.random.default_rng(1)
    X, W, b = r.standard_normal((N, D)).astype(O.NP[t]), (D ** -0.5 * r.standard_normal((F, D))).astype(O.NP[t]), r.standard_normal(F).astype(O.NP[t])
    dX, dW, db = keep(Rows(dev, N, D, g)), keep(Rows(dev, F, D, g)), keep(dev.buffer(F))
    x, w = keep(dev.buffer(X, t)), keep(dev.buffer(W, t))
    Y, Z = (keep(Rows(dev, N, F, t)) for _ in range(2))
    linear(dev, keep, dtype=t, N=N, D=D, F=F, act=L.ACT_SILU, X=x, W=w, bias=keep(dev.buffer(b, t)), Y=Y, Z=Z)
    dev.sync()
    z = Z[LIVE]
    O.compare({"Y": Y[LIVE], "Z": z}, O.linear(X[LIVE], W, b, kind=L.ACT_SILU, dtype=t))
    dY = sparse(dev, keep, t, 2)
    kw = dict(dtype=t, grad_dtype=g, N=N, D=D, F=F, act=L.ACT_SILU, X=x, W=w, Z=Z, dY=dY, dX=dX, dW=dW, dbias=db)
    dev.linear_grad(ws=keep(dev.buffer(dev.linear_grad_workspace(**kw) // 4 + 4)), **kw)
    dev.sync()
    want = O.linear_grad(X[LIVE], W, z, dY[LIVE], kind=L.ACT_SILU, dtype=t, grad_dtype=g)
    O.compare({"dX": dX[LIVE], "dW": dW[range(F)], "dbias": db.read()}, {k: want[k] for k in ("dX", "dW", "dbias")})
    assert not dX[[5, N // 2 - 1, N - 6]].any()


@pytest.mark.parametrize("types", TYPES, ids=IDS)
def test_few_rows_of_large_weights(dev, keep, types):
    """W of 2.16e9 elements, read as it lies going forward and back."""
    t, g = types
    n, d, f = 3, 54000, 40001
    r = np.random.default_rng(3)
    X, A, B = r.standard_normal((n, d)).astype(O.NP[t]), r.standard_normal((f, 8)), (8 * d) ** -0.5 * r.standard_normal((d, 8))
    W = keep(Rows(dev, f, d, t))
    linear(dev, keep, dtype=t, N=f, D=8, F=d, X=keep(dev.buffer(A, t)), W=keep(dev.buffer(B, t)), Y=W)
    x, Y, Z = keep(dev.buffer(X, t)), keep(Rows(dev, n, f, t)), keep(Rows(dev, n, f, t))
    linear(dev, keep, dtype=t, N=n, D=d, F=f, act=L.ACT_GELU, X=x, W=W, Y=Y, Z=Z)
    dev.sync()
    live = np.array([0, 1, 7777, 39767, 39768, f - 2, f - 1])
    w, z = W[live], Z[range(n)]
    O.compare({"Y": Y[range(n)][:, live], "Z": z[:, live]}, O.linear(X, w, kind=L.ACT_GELU, dtype=t))
    dY = np.zeros((n, f), O.NP[t])
    dY[:, live] = r.standard_normal((n, len(live)))
    dX, dW, db = keep(Rows(dev, n, d, g)), keep(Rows(dev, f, d, g)), keep(dev.buffer(f))
    kw = dict(dtype=t, grad_dtype=g, N=n, D=d, F=f, act=L.ACT_GELU, X=x, W=W, Z=Z, dY=keep(dev.buffer(dY, t)), dX=dX, dW=dW, dbias=db)
    dev.linear_grad(ws=keep(dev.buffer(dev.linear_grad_workspace(**kw) // 4 + 4)), **kw)
    dev.sync()
    want = O.linear_grad(X, w, z[:, live], dY[:, live], kind=L.ACT_GELU, dtype=t, grad_dtype=g)
    O.compare({"dX": dX[range(n)], "dW": dW[live], "dbias": db.read()[live]}, {k: want[k] for k in ("dX", "dW", "dbias")})
    assert not dW[[2, 20000, f - 3]].any()


@pytest.mark.parametrize("types", TYPES, ids=["f16", "f16_f32res", "f32"])
def test_norms(dev, keep, types):
    t, tr = types
    r = np.random.default_rng(4)
    gate, pw, nw = (1 + 0.25 * r.standard_normal((1, F))).astype(O.NP[t]), (1 + 0.25 * r.standard_normal(F)).astype(O.NP[t]), (1 + 0.25 * r.standard_normal(F)).astype(O.NP[t])
    X = r.standard_normal((N, 8)).astype(O.NP[t])
    x = keep(dev.buffer(X, t))
    Y = keep(Rows(dev, N, F, t))
    linear(dev, keep, dtype=t, N=N, D=8, F=F, X=x, W=keep(dev.buffer(r.standard_normal((F, 8)), t)), Y=Y)
    g, p, n = (keep(dev.buffer(v, t)) for v in (gate, pw, nw))
    H, out = keep(Rows(dev, N, F, tr)), keep(Rows(dev, N, F, t))
    common = dict(dtype=t, res_dtype=tr, N=N, D=F, post=L.NORM_RMS, pre=L.NORM_RMS, Y=Y, gate=g, post_w=p, pre_w=n)
    dev.residual_norm(**common, H_out=H, O=out)
    dev.sync()
    y, h = Y[LIVE], H[LIVE]
    O.compare({"H_out": h, "O": out[LIVE]}, O.residual_norm(None, y, gate, 0, L.NORM_RMS, L.NORM_RMS, post_w=pw, pre_w=nw, dtype=t, res_dtype=tr))
    dO = sparse(dev, keep, t, 5)
    dH, dY = keep(Rows(dev, N, F, tr)), out   # (over the norm's output, which is not needed any more)
    sums = {k: keep(dev.buffer(F, t if k == "dgate" else L.AH_F32)) for k in ("dgate", "dpost_w", "dpre_w")}
    kw = dict(**common, H_out=H, dO=dO, dH=dH, dY=dY, **sums)
    dev.residual_norm_grad(ws=keep(dev.buffer(dev.residual_norm_grad_workspace(**kw) // 4 + 4)), **kw)
    dev.sync()
    want = O.residual_norm_grad(h, y, None, dO[LIVE], gate, 0, L.NORM_RMS, L.NORM_RMS, pw, pre_w=nw, dtype=t, res_dtype=tr)
    O.compare({"dH": dH[LIVE], "dY": dY[LIVE], **{k: b.read() for k, b in sums.items()}}, {k: want[k] for k in ("dH", "dY", *sums)})
    assert not dY[[5, N - 6]].any()


def test_clipping(dev, keep):
    """A tensor of 2.16e9 entries among small ones."""
    big, small = sparse(dev, keep, L.AH_F16, 6), keep(dev.buffer(np.full(100, 0.5)))
    out = keep(Rows(dev, N, F, L.AH_F16))
    norm, coef = keep(dev.buffer(1)), keep(dev.buffer(1))
    kw = dict(tensors=dev.tensor_list([(small, small, 100, L.AH_F32, L.AH_F32), (big, out, N * F, L.AH_F16, L.AH_F16)]), max_norm=2.0, norm=norm, coef=coef)
    dev.clip_norm(ws=keep(dev.buffer(dev.clip_norm_workspace(**kw) // 4 + 4)), **kw)
    dev.sync()
    v = big[LIVE].astype(np.float64)
    want = np.sqrt((v * v).sum() + 25.0)
    assert abs(norm.read()[0] - want) <= 8 * O.U32 * want
    c = 2.0 / (want + 1e-6)
    assert np.all(np.abs(out[LIVE] - c * v) <= O.rounded(c * v, L.AH_F16) + 8 * O.U32 * np.abs(c * v))
    assert not out[[5, N - 6]].any() and np.all(np.abs(small.read() - 0.5 * c) <= 8 * O.U32 * c)
