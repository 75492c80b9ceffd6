"""ah_orthogonalize and ah_muon_step against the iteration in 64 bits (GPU).

Bound on the error of the last iterate in the Frobenius norm: a step multiplies what is already wrong by at most L = |a| + 3|b| s^2 +
5|c| s^4 for singular values up to s, taken at the values that occur (the polynomial's slope is at most 3.4445, at 0, where the
small values are, and at most 4 in size up to s = 1.21), and adds the roundings of three products: each loses 3 * 2^-22 (planes of
both operands, lo*lo) and (K/32 + 32) 2^-24 (f32 sums over K/32 steps) of |left| |right| per element, whose Frobenius norm is at
most |left|_F |right|_F.
"""
import numpy as np
import pytest

from anneal_amd import _lib as L

pytestmark = pytest.mark.gpu
U16, U32, PLANES = 2.0 ** -11, 2.0 ** -24, 2.0 ** -22
NP = {L.AH_F16: np.float16, L.AH_F32: np.float32}
COEF = (3.4445, -4.7750, 2.0315)


def iterate(U, steps=5, coef=COEF, eps=1e-7):
    """The iterate and the bound on its Frobenius error."""
    a, b, c = (float(np.float32(v)) for v in coef)
    T = U.shape[0] > U.shape[1]
    X = U.T if T else U
    X = X / (np.linalg.norm(X) + float(np.float32(eps)))
    K = X.shape[1]
    u = 3 * PLANES + (K / 32 + 32) * U32
    err = np.linalg.norm(X) * 2 * PLANES
    for _ in range(steps):
        A = X @ X.T
        B = a * np.eye(len(A)) + b * A + c * A @ A
        nx, na = np.linalg.norm(X), np.linalg.norm(A)
        s = np.linalg.norm(X, 2)
        slope = max(abs(a + 3 * b * t * t + 5 * c * t ** 4) for t in np.linspace(0, s, 200))
        dA = u * nx * nx
        dB = (abs(b) + 2 * abs(c) * s * s) * dA + abs(c) * u * na * na + PLANES * np.linalg.norm(B)
        err = slope * err + dB * s + u * np.linalg.norm(B) * nx
        X = B @ X
    return (X.T if T else X), err


def gradient(r, rows, cols, dtype):
    k = min(rows, cols, 16)
    g = (r.standard_normal((rows, k)) * 0.7 ** np.arange(k)) @ r.standard_normal((k, cols)) + 0.3 * r.standard_normal((rows, cols))
    return (1e-3 * g).astype(NP[dtype])


def ortho(dev, G, dtype, out_dtype=L.AH_F32, **kw):
    G = G if G.ndim == 3 else G[None]
    batch, rows, cols = G.shape
    g, o = dev.buffer(G, dtype), dev.buffer(np.full(G.shape, 777, NP[out_dtype]), out_dtype)
    args = dict(dtype=dtype, out_dtype=out_dtype, rows=rows, cols=cols, batch=batch, G=g, O=o, **kw)
    ws = dev.buffer(dev.orthogonalize_workspace(**args) // 4 + 4)
    dev.orthogonalize(ws=ws, **args)
    dev.sync()
    out = o.read().reshape(G.shape).astype(np.float64)
    for b in (g, o, ws):
        b.free()
    return out


SHAPES = [(1, 1), (1, 50), (50, 1), (3, 3), (64, 64), (65, 63), (128, 200), (200, 128), (33, 1000), (1000, 33), (257, 300), (513, 512)]


@pytest.mark.parametrize("types", [(L.AH_F32, L.AH_F32), (L.AH_F16, L.AH_F16), (L.AH_F16, L.AH_F32), (L.AH_F32, L.AH_F16)],
                         ids=["f32", "f16", "f16_f32", "f32_f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_orthogonalize(dev, shape, types):
    G = gradient(np.random.default_rng(shape), *shape, types[0])
    want, err = iterate(G.astype(np.float64))
    got = ortho(dev, G, types[0], types[1])[0]
    tol = err + (U16 * 1.01 * np.linalg.norm(want) + 2.0 ** -25 * want.size ** 0.5 if types[1] == L.AH_F16 else U32 * np.linalg.norm(want))
    assert np.linalg.norm(got - want) <= tol, (np.linalg.norm(got - want), tol)
    # and near what 32-bit products leave (the first step's 485-fold slope at 0 is met by few values)
    if types[1] == L.AH_F32:
        assert np.linalg.norm(got - want) <= 2e-5 * np.linalg.norm(want)


@pytest.mark.parametrize("steps,coef", [(1, COEF), (2, (2.0, -1.5, 0.5)), (12, (1.875, -1.25, 0.375))])
def test_other_polynomials(dev, steps, coef):
    G = gradient(np.random.default_rng(steps), 96, 160, L.AH_F32)
    want, err = iterate(G.astype(np.float64), steps, coef)
    got = ortho(dev, G, L.AH_F32, steps=steps, coef=coef)[0]
    assert np.linalg.norm(got - want) <= err + U32 * np.linalg.norm(want)


@pytest.mark.parametrize("shape", [(70, 130), (130, 70)])
def test_batch_and_strides(dev, shape):
    """Matrices of one call are as they are alone; what lies between rows and matrices stays; a batch may repeat one matrix."""
    rows, cols = shape
    r = np.random.default_rng(8)
    Gs = [gradient(r, rows, cols, L.AH_F32) for _ in range(3)]
    alone = [ortho(dev, g, L.AH_F32)[0] for g in Gs]
    ld, stride = cols + 3, rows * (cols + 3) + 5
    flat = np.full(3 * stride, np.nan, np.float32)
    at = [z * stride + i * ld + np.arange(cols) for z in range(3) for i in range(rows)]
    flat[np.array(at).ravel()] = np.concatenate([g.ravel() for g in Gs])
    g, o = dev.buffer(flat), dev.buffer(np.full(3 * stride, 777, np.float32))
    args = dict(dtype=L.AH_F32, rows=rows, cols=cols, batch=3, G=g, O=o, ldg=ld, ldo=ld, stride_o=stride)
    ws = dev.buffer(dev.orthogonalize_workspace(stride_g=stride, **args) // 4 + 4)
    for sg, want in ((stride, alone), (0, [alone[0]] * 3)):
        dev.orthogonalize(ws=ws, stride_g=sg, **args)
        dev.sync()
        out = o.read()
        np.testing.assert_array_equal(out[np.array(at).ravel()], np.concatenate([a.ravel() for a in want]).astype(np.float32))
        keep = np.ones(len(out), bool)
        keep[np.array(at).ravel()] = False
        assert np.all(out[keep] == 777)
    for b in (g, o, ws):
        b.free()


def test_zero_tiny_huge_and_nonfinite(dev):
    assert not ortho(dev, np.zeros((40, 70), np.float32), L.AH_F32).any()
    base = gradient(np.random.default_rng(2), 40, 70, L.AH_F32) * 1000
    want, err = iterate(base.astype(np.float64), eps=0.0)
    for s in (2.0 ** -100, 2.0 ** 100):   # the norm's squares pass f32's range
        got = ortho(dev, base * np.float32(s), L.AH_F32, eps=0.0)[0]
        assert np.linalg.norm(got - want) <= err + U32 * np.linalg.norm(want), s
    base[3, 4] = np.nan
    assert np.isnan(ortho(dev, base, L.AH_F32)).any()


def test_in_place(dev):
    G = gradient(np.random.default_rng(4), 100, 90, L.AH_F32)
    want = ortho(dev, G, L.AH_F32)[0].astype(np.float32)
    b = dev.buffer(G)
    args = dict(dtype=L.AH_F32, rows=100, cols=90, G=b, O=b)
    ws = dev.buffer(dev.orthogonalize_workspace(**args) // 4 + 4)
    dev.orthogonalize(ws=ws, **args)
    dev.sync()
    np.testing.assert_array_equal(b.read().reshape(100, 90), want)
    b.free()
    ws.free()


@pytest.mark.parametrize("rows,cols", [(150, 5003), (5003, 150)])
def test_long_sides_of_a_batch(dev, rows, cols):
    """More tiles than the chip takes at once, each summed in pieces: every matrix is the one alone to its last bits' rounding."""
    batch = 60
    G = gradient(np.random.default_rng(rows), rows, cols, L.AH_F32)
    want, err = iterate(G.astype(np.float64))
    g, o = dev.buffer(G), dev.buffer(batch * G.size)
    args = dict(dtype=L.AH_F32, rows=rows, cols=cols, batch=batch, G=g, O=o, stride_g=0)
    dev.orthogonalize(ws=dev.buffer(dev.orthogonalize_workspace(**args) // 4 + 4), **args)
    got = o.read().reshape(batch, rows, cols)
    for z in range(batch):
        assert np.array_equal(got[z], got[0])
    assert np.linalg.norm(got[0] - want) <= min(err + U32 * np.linalg.norm(want), 2e-5 * np.linalg.norm(want))


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("batch,rows,cols", [(1, 128, 784), (1, 100, 33), (2, 65, 130)])
def test_muon_step(dev, batch, rows, cols, dtype, nesterov):
    """Three steps in place against 64 bits, step by step on the state that the device holds."""
    r = np.random.default_rng([rows, cols])
    shape = (batch, rows, cols)
    M, W = 1e-2 * r.standard_normal(shape).astype(np.float32), r.standard_normal(shape).astype(np.float32)
    bM, bW, b16 = dev.buffer(M), dev.buffer(W), dev.buffer(np.zeros(shape, np.float16), L.AH_F16)
    bG = dev.buffer(np.zeros(shape, NP[dtype]), dtype)
    lr, mu, wd, sc = (float(np.float32(v)) for v in (0.02, 0.95, 0.1, 1.5))
    args = dict(dtype=dtype, rows=rows, cols=cols, batch=batch, G=bG, M=bM, W=bW, W16_out=b16, lr=lr, momentum=mu, decay=wd, scale=sc, nesterov=nesterov)
    ws = dev.buffer(dev.muon_step_workspace(**args) // 4 + 4)
    for _ in range(3):
        G = np.stack([gradient(r, rows, cols, dtype) for _ in range(batch)])
        bG.write(G)
        dev.muon_step(ws=ws, **args)
        dev.sync()
        gM, gW, g16 = bM.read().reshape(shape), bW.read().reshape(shape), b16.read().reshape(shape)
        M1 = mu * M.astype(np.float64) + G
        assert np.all(np.abs(gM - M1) <= 2 * U32 * (np.abs(mu * M) + np.abs(M1)))
        for z in range(batch):
            U = G[z] + mu * gM[z].astype(np.float64) if nesterov else gM[z].astype(np.float64)
            O, err = iterate(U)
            err += 2 * U32 * 485 / np.linalg.norm(U) * np.linalg.norm(np.abs(mu * gM[z]) + np.abs(U))   # U's own rounding
            want = (1 - lr * wd) * W[z].astype(np.float64) - lr * sc * O
            tol = lr * sc * err + 4 * U32 * (np.linalg.norm(W[z]) + lr * sc * np.linalg.norm(O))
            assert np.linalg.norm(gW[z] - want) <= tol
        np.testing.assert_array_equal(g16, gW.astype(np.float16))
        M, W = gM, gW
    for b in (bM, bW, b16, bG, ws):
        b.free()


def test_out_of_place_leaves_the_inputs(dev):
    r = np.random.default_rng(6)
    G, M, W = (r.standard_normal((50, 80)).astype(np.float32) for _ in range(3))
    bG, bM, bW, oM, oW = dev.buffer(G), dev.buffer(M), dev.buffer(W), dev.buffer(4000), dev.buffer(4000)
    args = dict(dtype=L.AH_F32, rows=50, cols=80, G=bG, M=bM, W=bW, lr=0.1, decay=0.01)
    ws = dev.buffer(dev.muon_step_workspace(**args) // 4 + 4)
    dev.muon_step(ws=ws, M_out=oM, W_out=oW, **args)
    dev.sync()
    for b, a in ((bG, G), (bM, M), (bW, W)):
        np.testing.assert_array_equal(b.read(), a.ravel())
    dev.muon_step(ws=ws, **args)
    dev.sync()
    np.testing.assert_array_equal(bM.read(), oM.read())
    np.testing.assert_array_equal(bW.read(), oW.read())
    for b in (bG, bM, bW, oM, oW, ws):
        b.free()


@pytest.mark.parametrize("shape", [(96, 160), (160, 96), (300, 520)])
def test_repeats_bit_for_bit_in_a_graph(dev, shape):
    from anneal_amd.backend import C as ct
    rows, cols = shape
    r = np.random.default_rng(shape)
    G, M, W = (r.standard_normal(shape).astype(np.float32) for _ in range(3))
    bG, bM, bW, oM, oW = dev.buffer(G), dev.buffer(M), dev.buffer(W), dev.buffer(G.size), dev.buffer(G.size)
    args = dict(dtype=L.AH_F32, rows=rows, cols=cols, G=bG, M=bM, M_out=oM, W=bW, W_out=oW, lr=0.1)
    ws = dev.buffer(dev.muon_step_workspace(**args) // 4 + 4)
    dev.muon_step(ws=ws, **args)
    dev.sync()
    first = oM.read(), oW.read()
    g = ct.c_void_p()
    L.check(dev.lib.ah_graph_begin(dev.h))
    dev.muon_step(ws=ws, **args)
    L.check(dev.lib.ah_graph_end(dev.h, ct.byref(g)))
    for _ in range(4):
        ws.write(np.full(ws.n, np.nan, np.float32))
        oM.write(np.zeros(G.size, np.float32))
        oW.write(np.zeros(G.size, np.float32))
        L.check(dev.lib.ah_graph_replay(dev.h, g))
        dev.sync()
        np.testing.assert_array_equal(oM.read(), first[0])
        np.testing.assert_array_equal(oW.read(), first[1])
        dev.muon_step(ws=ws, **args)
        dev.sync()
        np.testing.assert_array_equal(oW.read(), first[1])
    dev.lib.ah_graph_destroy(g)
    for b in (bG, bM, bW, oM, oW, ws):
        b.free()
