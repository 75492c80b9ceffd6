"""ah_linear_ce against its definition in 64 bits (GPU).

Tolerances are bounds, element by element, from the roundings on the way. u16 = 2^-11 and u32 = 2^-24 are half steps of f16 and
f32 relative to the value; a pair of f16 planes leaves 2^-22 of a value.
  logit:   dz = sum_d |x||w| (3 * 2^-22 + (D/32 + 32) u32) + u32 |z|: three plane roundings (f32 operands; none for f16) and the
           sums of 32 products (exact inside an MFMA up to its f32 adds) over D/32 steps
  P:       p (2 dz + 2^-21 + |z - lse| 2^-22) (z and lse move p by e^dz each; the exponent's product rounds by |z - lse| u32 and
           exp2 by an ulp or two), and per f16 rounding of it u16 p, per pair of planes 2^-22 p; below the planes' range 2^-39
  gradient: (error of P) @ |W| + 2^-22 |P| @ |W| for planes + (K/32 + 32) u32 |P| @ |W|, times s, and the output's own rounding
"""
import numpy as np
import pytest

from anneal_amd import _lib as L

pytestmark = pytest.mark.gpu
U16, U32, PLANES = 2.0 ** -11, 2.0 ** -24, 2.0 ** -22
NP = {L.AH_F16: np.float16, L.AH_F32: np.float32}


class Case:
    """Inputs in numpy and their values in 64 bits."""

    def __init__(self, N, D, V, dtype=L.AH_F32, grad_dtype=None, bias=True, labels=None, seed=0, std=1.0, wstd=None):
        r = np.random.default_rng([seed, N, D, V])
        self.N, self.D, self.V, self.dtype = N, D, V, dtype
        self.grad_dtype = L.AH_F32 if grad_dtype is None else grad_dtype
        t = NP[dtype]
        self.X = (std * r.standard_normal((N, D))).astype(t)
        self.W = ((D ** -0.5 if wstd is None else wstd) * r.standard_normal((V, D))).astype(t)
        self.b = (0.5 * r.standard_normal(V)).astype(t) if bias else None
        self.labels = (r.integers(0, V, N) if labels is None else np.asarray(labels)).astype(np.int32)

    def exact(self, mean=True, grad_scale=1.0):
        """Values and bounds: {name: (value, tolerance)}."""
        X, W = self.X.astype(np.float64), self.W.astype(np.float64)
        y = self.labels
        on = (y >= 0) & (y < self.V)
        c = int(on.sum())
        with np.errstate(all="ignore"):
            X = np.where(on[:, None], X, 0.0)
            z = X @ W.T + (0.0 if self.b is None else self.b.astype(np.float64))
            mag = np.abs(X) @ np.abs(W).T
            fin = np.where(np.isfinite(z), z, 0.0)
            dz = mag * ((3 * PLANES if self.dtype == L.AH_F32 else 0.0) + (self.D / 32 + 32) * U32) + U32 * np.abs(fin)
            m = z.max(1, keepdims=True)
            lse = m + np.log(np.exp(z - m).sum(1, keepdims=True))
            p = np.exp(z - lse)
        at = np.where(on, y, 0)
        rows = np.arange(self.N)
        dzm = dz.max(1)
        dlse = dzm + (self.V / 64 + 40) * U32 + 2 * U32 * np.abs(lse[:, 0])
        out = {"lse": (np.where(on, lse[:, 0], 0.0), np.where(on, dlse, 0.0))}
        rl, drl = np.where(on, lse[:, 0] - z[rows, at], 0.0), np.where(on, dlse + dzm + U32 * np.abs(fin[rows, at]), 0.0)
        out["rowloss"] = (rl, drl)
        n = max(c, 1) if mean else 1
        out["loss"] = (rl.sum() / n, drl.sum() / n + 2 * U32 * abs(rl.sum()) / n)
        f16 = self.grad_dtype == L.AH_F16
        with np.errstate(all="ignore"):
            dP = p * (dzm[:, None] + dlse[:, None] + 2.0 ** -21 + np.where(np.isfinite(z), np.abs(z - lse), 0.0) * 2.0 ** -22)
        P = p.copy()
        P[rows, at] -= 1.0
        dbP = dP.copy()
        if f16:   # exp(z - tile maximum) is kept in f16, then P is
            dP = dP + U16 * p + U16 * np.abs(P)
            dbP = dbP + U16 * p
        else:
            dP = dP + PLANES * np.abs(P)
        dP, P, dbP = (np.where(on[:, None], v, 0.0) for v in (dP + 2.0 ** -39, P, dbP + 2.0 ** -39))
        s = grad_scale / n

        def product(P, dP, B, K):
            Ba = np.abs(B)
            lost = (2 * PLANES if self.dtype == L.AH_F32 else 0.0) + (K / 32 + 32) * U32
            g = P @ B * s
            return g, abs(s) * (dP @ Ba + lost * (np.abs(P) @ Ba)) + (U16 if f16 else 4 * U32) * np.abs(g) * 1.01 + (2.0 ** -25 if f16 else 1e-37)
        out["dX"] = product(P, dP, W, self.V)
        out["dW"] = product(P.T, dP.T, X, self.N)
        db = P.sum(0) * s
        out["dbias"] = (db, abs(s) * (dbP.sum(0) + (self.N + 8) * U32 * np.abs(P).sum(0)) + 4 * U32 * np.abs(db) + 1e-37)
        return out


def buffers(dev, c, want, fill=None):
    """Device buffers of the inputs and of the wanted outputs; outputs start at fill."""
    shapes = {"loss": 1, "rowloss": c.N, "lse": c.N, "dX": c.N * c.D, "dW": c.V * c.D, "dbias": c.V}
    b = {"X": dev.buffer(c.X, c.dtype), "W": dev.buffer(c.W, c.dtype), "labels": dev.buffer(c.labels, L.AH_I32)}
    if c.b is not None:
        b["bias"] = dev.buffer(c.b, c.dtype)
    for k in want:
        t = c.grad_dtype if k in ("dX", "dW") else L.AH_F32
        b[k] = dev.buffer(np.full(shapes[k], 777.0 if fill is None else fill, NP[t]), t)
    return b


def run(dev, c, want=("loss", "rowloss", "lse", "dX", "dW", "dbias"), **kw):
    b = buffers(dev, c, want)
    args = dict(dtype=c.dtype, grad_dtype=c.grad_dtype, N=c.N, D=c.D, V=c.V, **b, **kw)
    ws = dev.buffer(dev.linear_ce_workspace(**args) // 4 + 4)
    dev.linear_ce(ws=ws, **args)
    dev.sync()
    shapes = {"dX": (c.N, c.D), "dW": (c.V, c.D)}
    got = {k: b[k].read().astype(np.float64).reshape(shapes.get(k, -1)) for k in want}
    for v in list(b.values()) + [ws]:
        v.free()
    return got


def compare(got, exact):
    for k, g in got.items():
        v, tol = exact[k]
        d = np.abs(g - v)
        bad = ~(d <= tol)
        assert not bad.any(), (k, "worst ratio", float(np.max(d / np.maximum(tol, 1e-300))), "at", np.argwhere(bad)[:4].tolist(), int(bad.sum()))


SHAPES = [(1, 1, 1), (1, 64, 7), (3, 5, 2), (7, 33, 65), (64, 64, 64), (65, 128, 257), (130, 72, 1000), (257, 200, 515), (300, 65, 2049)]
TYPES = [(L.AH_F32, L.AH_F32), (L.AH_F16, L.AH_F16), (L.AH_F16, L.AH_F32)]


@pytest.mark.parametrize("types", TYPES, ids=["f32", "f16", "f16_f32grad"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%dx%d" % s)
def test_loss_and_gradients(dev, shape, types):
    c = Case(*shape, dtype=types[0], grad_dtype=types[1])
    scale = 256.0 if types[1] == L.AH_F16 else 1.0
    compare(run(dev, c, grad_scale=scale), c.exact(grad_scale=scale))


@pytest.mark.parametrize("types", TYPES, ids=["f32", "f16", "f16_f32grad"])
def test_rows_that_do_not_count(dev, types):
    """Labels outside [0, V): what those rows hold is not used, their outputs are zero."""
    N, V = 150, 300
    y = np.random.default_rng(5).integers(0, V, N)
    y[:40], y[60], y[61], y[140:] = -100, V, 2 ** 31 - 1, -1
    c = Case(N, 96, V, dtype=types[0], grad_dtype=types[1], labels=y)
    c.X[:40], c.X[140:] = np.nan, np.inf
    exact = c.exact()
    got = run(dev, c)
    compare(got, exact)
    off = (y < 0) | (y >= V)
    assert not got["dX"][off].any() and not got["rowloss"][off].any() and not got["lse"][off].any()


@pytest.mark.parametrize("types", TYPES, ids=["f32", "f16", "f16_f32grad"])
def test_no_row_counts(dev, types):
    c = Case(70, 40, 90, dtype=types[0], grad_dtype=types[1], labels=np.full(70, -1))
    c.X[:] = np.nan
    for k, v in run(dev, c).items():
        assert not v.any(), k


@pytest.mark.parametrize("want", [("loss",), ("loss", "rowloss"), ("loss", "dX"), ("loss", "dW"), ("loss", "dbias"), ("loss", "lse", "dX", "dbias")], ids="_".join)
@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
def test_each_output_alone(dev, dtype, want):
    c = Case(100, 80, 700, dtype=dtype, grad_dtype=dtype)
    compare(run(dev, c, want=want), c.exact())


def test_sum_and_scale(dev):
    c = Case(90, 64, 333, dtype=L.AH_F16, grad_dtype=L.AH_F32, bias=False)
    compare(run(dev, c, want=("loss", "rowloss", "dX", "dW"), mean=False, grad_scale=-0.125), c.exact(mean=False, grad_scale=-0.125))


@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
def test_classes_ruled_out(dev, dtype):
    """A bias of -inf over whole stretches of the vocabulary, a tile's width and more."""
    V = 1100
    y = np.random.default_rng(1).integers(600, 700, 66)
    c = Case(66, 64, V, dtype=dtype, grad_dtype=dtype, labels=y)
    c.b[:600], c.b[800:] = -np.inf, -np.inf
    got = run(dev, c)
    compare(got, c.exact())
    assert not got["dW"][:600].any() and not got["dbias"][800:].any()


@pytest.mark.parametrize("types", TYPES, ids=["f32", "f16", "f16_f32grad"])
def test_confident_and_far_rows(dev, types):
    """Logits of several hundred: rows that are all but certain, right and wrong."""
    c = Case(64, 128, 256, dtype=types[0], grad_dtype=types[1], std=8.0, wstd=4.0)
    X, W = c.X.astype(np.float64), c.W.astype(np.float64)
    best = (X @ W.T + c.b.astype(np.float64)).argmax(1)
    c.labels[::2] = best[::2]
    compare(run(dev, c), c.exact())


def test_operand_scales(dev):
    """f32 operands far from 1: the planes' power of two follows them."""
    for xs, ws in ((1e-20, 1e18), (1e15, 1e-17), (1.0, 1e-30), (3e-38, 3e-38)):
        c = Case(40, 48, 100, std=xs, wstd=ws)
        e = c.exact()
        got = run(dev, c)
        compare({k: got[k] for k in ("loss", "rowloss", "dX", "dbias")}, e)
        v, tol = e["dW"]   # the P floor of 2^-40 and the planes' relative to the operand's largest value
        assert np.all(np.abs(got["dW"] - v) <= tol + 2.0 ** -38 * np.abs(c.X).max())


def test_nonfinite_logits_show(dev):
    c = Case(70, 64, 200, dtype=L.AH_F16, grad_dtype=L.AH_F16)
    c.X[9, 3] = np.nan
    got = run(dev, c)
    assert np.isnan(got["rowloss"][9]) and np.isnan(got["loss"][0]) and np.isnan(got["dX"][9]).all()
    keep = np.arange(70) != 9
    assert np.isfinite(got["rowloss"][keep]).all() and np.isfinite(got["dX"][keep]).all()


@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("pad", [1, 8])
def test_strides(dev, dtype, pad):
    """Rows further apart than they are long; what lies between them stays."""
    c = Case(75, 64, 130, dtype=dtype, grad_dtype=dtype)
    t, ld = NP[dtype], c.D + pad
    wide = lambda a: np.pad(a, ((0, 0), (0, pad)), constant_values=np.nan)   # noqa: E731
    b = {"X": dev.buffer(wide(c.X), dtype), "W": dev.buffer(wide(c.W), dtype), "labels": dev.buffer(c.labels, L.AH_I32), "bias": dev.buffer(c.b, dtype),
         "loss": dev.buffer(1), "dX": dev.buffer(np.full((c.N, ld), 777, t), dtype), "dW": dev.buffer(np.full((c.V, ld), 777, t), dtype)}
    args = dict(dtype=dtype, grad_dtype=dtype, N=c.N, D=c.D, V=c.V, ldx=ld, ldw=ld, lddx=ld, lddw=ld, **b)
    ws = dev.buffer(dev.linear_ce_workspace(**args) // 4 + 4)
    dev.linear_ce(ws=ws, **args)
    dev.sync()
    dX, dW = b["dX"].read().reshape(c.N, ld), b["dW"].read().reshape(c.V, ld)
    e = c.exact()
    compare({"loss": b["loss"].read(), "dX": dX[:, :c.D].astype(np.float64), "dW": dW[:, :c.D].astype(np.float64)}, e)
    assert np.all(dX[:, c.D:] == 777) and np.all(dW[:, c.D:] == 777)
    for v in list(b.values()) + [ws]:
        v.free()


# Around the forms' limits (16, 64, 128 rows; 8 features) and a stage's and a tile's (64 or 128 of either sum, 128 classes, 256 features);
# long sums are split.
FEW = [(1, 8, 3), (5, 7, 40), (16, 70, 300), (17, 65, 129), (64, 131, 260), (65, 261, 97), (128, 333, 1030), (129, 333, 1030), (33, 4099, 70), (9, 41, 20011)]


@pytest.mark.parametrize("types", TYPES, ids=["f32", "f16", "f16_f32grad"])
@pytest.mark.parametrize("shape", FEW, ids=lambda s: "%dx%dx%d" % s)
@pytest.mark.parametrize("pad", [3, 8])
def test_few_rows_of_any_stride(dev, types, shape, pad):
    """Few rows and W as it lies: rows that end anywhere, NaN between them and behind the last."""
    dtype, gdtype = types
    c = Case(*shape, dtype=dtype, grad_dtype=gdtype, labels=np.where(np.arange(shape[0]) % 5 == 3, -1, np.arange(shape[0]) * 7 % shape[2]))
    t, ld = NP[gdtype], c.D + pad
    wide = lambda a: np.concatenate([np.pad(a, ((0, 0), (0, pad)), constant_values=np.nan).ravel(), np.full(64, np.nan, a.dtype)])   # noqa: E731
    b = {"X": dev.buffer(wide(c.X), dtype), "W": dev.buffer(wide(c.W), dtype), "labels": dev.buffer(c.labels, L.AH_I32), "bias": dev.buffer(c.b, dtype),
         "loss": dev.buffer(1), "rowloss": dev.buffer(c.N), "dX": dev.buffer(np.full((c.N, ld), 777, t), gdtype),
         "dW": dev.buffer(np.full((c.V, ld), 777, t), gdtype)}
    args = dict(dtype=dtype, grad_dtype=gdtype, N=c.N, D=c.D, V=c.V, ldx=ld, ldw=ld, lddx=ld, lddw=ld, grad_scale=256.0 if gdtype == L.AH_F16 else 1.0, **b)
    ws = dev.buffer(np.full(dev.linear_ce_workspace(**args) // 4 + 4, np.nan, np.float32))
    dev.linear_ce(ws=ws, **args)
    dev.sync()
    dX, dW = b["dX"].read().reshape(c.N, ld), b["dW"].read().reshape(c.V, ld)
    got = {"loss": b["loss"].read(), "rowloss": b["rowloss"].read(), "dX": dX[:, :c.D].astype(np.float64), "dW": dW[:, :c.D].astype(np.float64)}
    compare(got, c.exact(grad_scale=args["grad_scale"]))
    assert np.all(dX[:, c.D:] == 777) and np.all(dW[:, c.D:] == 777)
    loss = {"loss": dev.buffer(1)}   # and the loss alone
    for k in ("dX", "dW", "rowloss", "loss"):
        args.pop(k)
    dev.linear_ce(ws=ws, **args, **loss)
    dev.sync()
    compare({"loss": loss["loss"].read()}, c.exact())
    for v in list(b.values()) + list(loss.values()) + [ws]:
        v.free()


@pytest.mark.parametrize("shape", [(200, 96, 1500), (70, 203, 3001)], ids=lambda s: "%dx%dx%d" % s)
@pytest.mark.parametrize("types", TYPES, ids=["f32", "f16", "f16_f32grad"])
def test_repeats_bit_for_bit_in_a_graph(dev, types, shape):
    """Captured, then replayed between other work: the eager call's bits each time, also after new inputs."""
    from anneal_amd.backend import C as ct
    c = Case(*shape, dtype=types[0], grad_dtype=types[1])
    want = ("loss", "rowloss", "dX", "dW", "dbias")
    b = buffers(dev, c, want)
    args = dict(dtype=c.dtype, grad_dtype=c.grad_dtype, N=c.N, D=c.D, V=c.V, **b)
    ws = dev.buffer(dev.linear_ce_workspace(**args) // 4 + 4)
    dev.linear_ce(ws=ws, **args)
    dev.sync()
    first = {k: b[k].read() for k in want}
    g = ct.c_void_p()
    L.check(dev.lib.ah_graph_begin(dev.h))
    dev.linear_ce(ws=ws, **args)
    L.check(dev.lib.ah_graph_end(dev.h, ct.byref(g)))
    labels = np.where(np.arange(shape[0]) % 3 == 0, 5, -1)   # fewer rows count on the graph's replay
    other = Case(*shape, labels=labels, dtype=types[0], grad_dtype=types[1], seed=3)
    for step in range(4):
        src = other if step == 2 else c
        for k, a in (("X", src.X), ("W", src.W), ("bias", src.b), ("labels", src.labels)):
            b[k].write(a)
        ws.write(np.full(ws.n, np.nan, np.float32))
        L.check(dev.lib.ah_graph_replay(dev.h, g))
        dev.sync()
        got = {k: b[k].read() for k in want}
        if step != 2:
            for k in want:
                np.testing.assert_array_equal(got[k].view(np.uint8), first[k].view(np.uint8), err_msg=k)
        dev.linear_ce(ws=ws, **args)
        dev.sync()
        for k in want:
            np.testing.assert_array_equal(got[k].view(np.uint8), b[k].read().view(np.uint8), err_msg=k)
    dev.lib.ah_graph_destroy(g)
    for v in list(b.values()) + [ws]:
        v.free()
