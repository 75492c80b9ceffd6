"""ah_linear and ah_linear_grad against their formulas in 64 bits (GPU). Bounds as derived in block_oracle.py."""
import numpy as np
import pytest

import block_oracle as O
from anneal_amd import _lib as L

pytestmark = pytest.mark.gpu
TYPES = [(L.AH_F32, L.AH_F32), (L.AH_F16, L.AH_F16), (L.AH_F16, L.AH_F32)]
IDS = ["f32", "f16", "f16_f32grad"]
# rows, features in, features out: one row, few rows, single tiles and ragged ones, more rows than features and the other way round
SHAPES = [(1, 1, 1), (1, 7, 3), (1, 64, 65), (3, 8, 33), (5, 100, 260), (16, 128, 128), (17, 9, 129), (63, 264, 72), (64, 64, 64), (65, 200, 130), (128, 72, 257),
          (129, 65, 300), (200, 513, 136), (300, 7, 1000), (257, 1001, 515)]


class Strided:
    """A 2-D array on the device with `gap` elements between rows, which hold a mark."""
    MARK = 777.0

    def __init__(self, dev, a, dtype, gap=0):
        a = np.atleast_2d(a)
        self.shape, self.dtype, self.ld = a.shape, dtype, a.shape[1] + gap
        full = np.full((a.shape[0], self.ld), self.MARK, O.NP[dtype])
        full[:, : a.shape[1]] = a
        self.b = dev.buffer(full, dtype)
        self.ptr = self.b.ptr

    def read(self):
        full = self.b.read().reshape(self.shape[0], self.ld)
        assert np.all(full[:, self.shape[1]:] == self.MARK), "written between the rows"
        return full[:, : self.shape[1]]

    def free(self):
        self.b.free()


class Case:
    def __init__(self, N, D, F, dtype=L.AH_F32, grad_dtype=None, kind=L.ACT_GELU, bias=True, factor=True, res=True, scale=0.75, seed=0):
        r = np.random.default_rng([seed, N, D, F, kind])
        t = O.NP[dtype]
        self.N, self.D, self.F, self.dtype, self.kind, self.scale = N, D, F, dtype, kind, scale
        self.grad_dtype = L.AH_F32 if grad_dtype is None else grad_dtype
        self.X, self.W = r.standard_normal((N, D)).astype(t), (D ** -0.5 * r.standard_normal((F, D))).astype(t)
        self.b = (0.5 * r.standard_normal(F)).astype(t) if bias else None
        self.U = r.standard_normal((N, F)).astype(t) if factor else None
        self.R = (2 * r.standard_normal((N, F))).astype(t) if res else None
        self.Z = (1.5 * r.standard_normal((N, F))).astype(t)
        self.dY = r.standard_normal((N, F)).astype(t)

    def forward(self, dev, keep=True, gap=0, in_place=False):
        a = {k: Strided(dev, v, self.dtype, gap if v.ndim == 2 else 0) for k, v in (("X", self.X), ("W", self.W), ("bias", self.b), ("U", self.U), ("R", self.R)) if v is not None}
        out = {"Y": a["R"] if in_place else Strided(dev, np.full((self.N, self.F), np.nan), self.dtype, gap)}
        if keep:
            out["Z"] = Strided(dev, np.full((self.N, self.F), np.nan), self.dtype, gap)
        kw = dict(dtype=self.dtype, N=self.N, D=self.D, F=self.F, act=self.kind, scale=self.scale, **a, **out)
        kw.update({"ld" + k.lower(): v.ld for k, v in {**a, **out}.items() if k != "bias"})
        ws = dev.buffer(dev.linear_workspace(**kw) // 4 + 4)
        dev.linear(ws=ws, **kw)
        dev.sync()
        got = {k: v.read() for k, v in out.items()}
        for v in {id(v): v for v in [*a.values(), *out.values(), ws]}.values():
            v.free()
        return got

    def expected(self):
        return O.linear(self.X, self.W, self.b, self.U, self.R, self.kind, self.scale, self.dtype)

    def backward(self, dev, want=("dX", "dW", "dbias", "dU"), gap=0):
        if self.U is None:
            want = [k for k in want if k != "dU"]
        inputs = {"X": self.X, "W": self.W, "Z": self.Z, "U": self.U, "dY": self.dY}
        a = {k: Strided(dev, v, self.dtype, gap) for k, v in inputs.items() if v is not None}
        shapes = {"dX": (self.N, self.D, self.grad_dtype), "dW": (self.F, self.D, self.grad_dtype), "dbias": (1, self.F, L.AH_F32), "dU": (self.N, self.F, self.dtype)}
        out = {k: Strided(dev, np.full(shapes[k][:2], np.nan), shapes[k][2], gap if k != "dbias" else 0) for k in want}
        kw = dict(dtype=self.dtype, grad_dtype=self.grad_dtype, N=self.N, D=self.D, F=self.F, act=self.kind, scale=self.scale, **a, **out)
        kw.update({"ld" + k.lower(): v.ld for k, v in {**a, **out}.items() if k != "dbias"})
        ws = dev.buffer(dev.linear_grad_workspace(**kw) // 4 + 4)
        dev.linear_grad(ws=ws, **kw)
        dev.sync()
        got = {k: v.read() for k, v in out.items()}
        for v in [*a.values(), *out.values(), ws]:
            v.free()
        return got

    def gradients(self):
        return O.linear_grad(self.X, self.W, self.Z, self.dY, self.U, self.kind, self.scale, self.dtype, self.grad_dtype)


@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%dx%d" % s)
def test_forward(dev, shape, dtype):
    c = Case(*shape, dtype=dtype)
    O.compare(c.forward(dev), c.expected())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%dx%d" % s)
def test_gradients(dev, shape, types):
    c = Case(*shape, dtype=types[0], grad_dtype=types[1])
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("kind", O.ACTS)
@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("N", [2, 70, 140])
def test_activations(dev, N, types, kind):
    """Without bias, factor and residual, with values out to where the activations are flat; zeros exactly."""
    c = Case(N, 40, 96, dtype=types[0], grad_dtype=types[1], kind=kind, bias=False, factor=False, res=False, scale=1.0)
    c.W = (c.W * 16).astype(c.W.dtype)
    c.X[0] = 0
    c.Z = (6 * c.Z).astype(c.Z.dtype)
    c.Z[:, 5] = 0
    O.compare(c.forward(dev), c.expected())
    O.compare(c.forward(dev, keep=False), c.expected())
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("kind", O.ACTS)
@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
def test_activations_at_their_ends(dev, dtype, kind):
    """z from the smallest to the largest values of the type: act and slope go to 0 or to z and 1, and nothing becomes NaN on the way."""
    v = np.array([0.0, 1e-40, 1e-7, 1.0, 5.0, 9.5, 13.0, 20.0, 89.0, 104.0, 1e4, 6e4, 1e10, 2e19, 3e38])
    v = v[v <= 6e4] if dtype == L.AH_F16 else v
    z = np.concatenate([v, -v]).astype(O.NP[dtype])
    n = len(z)
    c = Case(n, 1, 1, dtype=dtype, grad_dtype=dtype, kind=kind, bias=False, factor=True, res=False, scale=1.0)
    c.X, c.W, c.U, c.Z, c.dY = z[:, None], np.ones_like(c.W), np.ones_like(c.U), z[:, None], np.ones_like(c.dY)
    got, want = c.forward(dev), c.expected()
    got.update(c.backward(dev, want=("dU", "dX")))
    want.update(c.gradients())
    for k, g in got.items():
        assert np.all(np.isfinite(g)), k
    # the planes' products may leave the last 2^-21 of a value as it is
    np.testing.assert_allclose(got["Y"].astype(np.float64), want["Y"][0], rtol=2.0 ** -10 if dtype == L.AH_F16 else 2.0 ** -18, atol=3e-6)
    np.testing.assert_allclose(got["dU"].astype(np.float64), want["dU"][0], rtol=2.0 ** -10 if dtype == L.AH_F16 else 2.0 ** -20, atol=3e-6)
    np.testing.assert_allclose(got["dX"].astype(np.float64), want["dX"][0], rtol=2.0 ** -9 if dtype == L.AH_F16 else 2.0 ** -18, atol=3e-6)


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("factor", [True, False])
@pytest.mark.parametrize("res", [True, False])
@pytest.mark.parametrize("N", [1, 200])
def test_parts(dev, N, bias, factor, res):
    c = Case(N, 72, 136, dtype=L.AH_F16, grad_dtype=L.AH_F16, kind=L.ACT_SILU, bias=bias, factor=factor, res=res)
    O.compare(c.forward(dev, keep=res), c.expected())
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("gap", [1, 8])
@pytest.mark.parametrize("N", [6, 150])
def test_strides(dev, N, gap, types):
    """Rows that are further apart, at offsets of any alignment; what lies between them stays."""
    c = Case(N, 64, 200, dtype=types[0], grad_dtype=types[1])
    O.compare(c.forward(dev, gap=gap), c.expected())
    O.compare(c.backward(dev, gap=gap), c.gradients())


@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("shape", [(4, 64, 200), (150, 100, 130), (4, 4096, 130)], ids=lambda s: "%dx%dx%d" % s)
def test_onto_the_residual_stream(dev, shape, dtype):
    """Y may be R."""
    c = Case(*shape, dtype=dtype)
    O.compare(c.forward(dev, in_place=True), c.expected())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("N", [3, 100])
@pytest.mark.parametrize("want", ["dX", "dW", "dbias", "dU"])
def test_single_outputs(dev, want, N, types):
    """Each alone, with the inputs that it does not need left out: the bits of the call with all."""
    c = Case(N, 96, 130, dtype=types[0], grad_dtype=types[1])
    full = c.backward(dev)
    if want != "dX":
        c.W = None
    if want != "dW":
        c.X = None
    np.testing.assert_array_equal(c.backward(dev, want=(want,))[want], full[want])


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1500, 700, 1111), (40, 3000, 500), (2100, 130, 520), (96, 2048, 4100), (1, 8192, 777)], ids=lambda s: "%dx%dx%d" % s)
def test_large(dev, shape, types):
    """256-, 128- and 64-wide tiles, whole and split over K, and long rows read as they lie."""
    c = Case(*shape, dtype=types[0], grad_dtype=types[1], kind=L.ACT_GELU_TANH)
    if types[1] == types[0]:
        O.compare(c.forward(dev), c.expected())
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
def test_rows_without_a_gradient(dev, types):
    """dY of zeros in some rows, and in all."""
    c = Case(150, 64, 200, dtype=types[0], grad_dtype=types[1])
    c.dY[20:90] = 0
    got = c.backward(dev)
    O.compare(got, c.gradients())
    assert not got["dX"][20:90].any() and not got["dU"][20:90].any()
    c.dY[:] = 0
    assert all(not v.any() for v in c.backward(dev).values())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 10])
@pytest.mark.parametrize("N", [30, 150])
def test_sizes_of_values(dev, N, size, types):
    """Operands and gradients far from 1, and rows of very different sizes (f32: each row of X and W has its own scale)."""
    c = Case(N, 96, 200, dtype=types[0], grad_dtype=types[1], kind=L.ACT_RELU, bias=False, factor=False, res=False, scale=1.0)
    c.X, c.W, c.dY = (c.X * size).astype(c.X.dtype), (c.W / size).astype(c.W.dtype), (c.dY * size).astype(c.dY.dtype)
    if types[0] == L.AH_F32:
        c.X *= np.float32(2.0) ** np.random.default_rng(1).integers(-40, 40, N)[:, None]
        c.dY *= np.float32(2.0) ** -30
    O.compare(c.forward(dev), c.expected())
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf], ids=str)
@pytest.mark.parametrize("N", [10, 100, 200])
def test_what_is_not_finite_stays_in_its_row_or_column(dev, N, bad, types):
    clean = Case(N, 96, 200, dtype=types[0], grad_dtype=types[1], kind=L.ACT_SILU)
    c = Case(N, 96, 200, dtype=types[0], grad_dtype=types[1], kind=L.ACT_SILU)
    c.X[3, 5], c.W[7, 2] = bad, bad
    rows, cols = np.arange(N) != 3, np.arange(200) != 7
    want, got = clean.expected(), c.forward(dev)
    for k, g in got.items():
        O.compare({k: g[rows][:, cols]}, {k: tuple(v[rows][:, cols] for v in want[k])})
    assert not np.isfinite(got["Z"][3]).any() and not np.isfinite(got["Z"][:, 7]).any()
    c = Case(N, 96, 200, dtype=types[0], grad_dtype=types[1], kind=L.ACT_SILU)
    c.dY[4, 9] = bad
    got, want = c.backward(dev), clean.gradients()
    rows, cols = np.arange(N) != 4, np.arange(200) != 9
    O.compare({"dX": got["dX"][rows], "dW": got["dW"][cols], "dbias": got["dbias"][0][cols], "dU": got["dU"][rows]},
              {"dX": tuple(v[rows] for v in want["dX"]), "dW": tuple(v[cols] for v in want["dW"]), "dbias": tuple(v[cols] for v in want["dbias"]),
               "dU": tuple(v[rows] for v in want["dU"])})
    assert not np.isfinite(got["dX"][4]).any() and not np.isfinite(got["dW"][9]).any() and not np.isfinite(got["dbias"][0, 9])


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("N", [30, 300])
def test_results_repeat(dev, N, types):
    c = Case(N, 520, 260, dtype=types[0], grad_dtype=types[1])
    for run in (c.forward, c.backward):
        a, b = run(dev), run(dev)
        for k in a:
            np.testing.assert_array_equal(a[k], b[k])


def test_gradients_against_differences(dev):
    """Central differences of the call's own forward pass along random directions: an f32 Y is off by 2^-20 or so of its terms, and a
    difference over 2 h by h^2 / 6 times the third derivative (below 2 along unit directions here)."""
    c = Case(64, 48, 80, kind=L.ACT_GELU, scale=0.5)
    z = c.forward(dev)["Z"]
    c.Z = z.astype(np.float32)
    g = c.backward(dev)
    r = np.random.default_rng(0)
    h = 2.0 ** -6
    for name, grad in (("X", "dX"), ("W", "dW"), ("b", "dbias"), ("U", "dU")):
        base = getattr(c, name).copy()
        d = r.standard_normal(base.shape).astype(np.float32)
        d /= np.float32(np.linalg.norm(d))
        y = []
        for s in (h, -h):
            setattr(c, name, (base + np.float32(s) * d).astype(np.float32))
            y.append(c.forward(dev)["Y"].astype(np.float64))
        setattr(c, name, base)
        want = float(((y[0] - y[1]) * c.dY).sum()) / (2 * h)
        noise = 2.0 ** -20 * np.linalg.norm(c.dY) * np.abs(y[0]).max() / h
        assert abs(float((g[grad].reshape(base.shape) * d).sum()) - want) <= noise + h * h * np.linalg.norm(c.dY), name


@pytest.mark.parametrize("gap", [0, 3])
@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("shape", [(1, 8, 1), (2, 9, 33), (5, 31, 16), (17, 100, 70), (33, 776, 333), (64, 1001, 131), (16, 8192, 2000), (64, 4096, 1000), (48, 4100, 2050),
                                   (16, 1000, 16400)], ids=lambda s: "%dx%dx%d" % s)
def test_few_rows(dev, shape, dtype, gap):
    """W read as it lies: K over 4, 8 and 16 waves with ends inside a lane's load, a chunk and a wave's turn, and tiles of 128 columns."""
    c = Case(*shape, dtype=dtype, kind=L.ACT_SILU)
    O.compare(c.forward(dev, gap=gap), c.expected())


@pytest.mark.parametrize("dtype", [L.AH_F32, L.AH_F16], ids=["f32", "f16"])
@pytest.mark.parametrize("D", [9, 33, 130])
def test_few_rows_read_twice_at_the_end(dev, D, dtype):
    """An infinity among the columns that two lanes read: it counts once, and where X is positive Z is infinite, not NaN."""
    c = Case(5, D, 40, dtype=dtype, kind=L.ACT_NONE, bias=False, factor=False, res=False)
    c.X = np.abs(c.X)
    c.W[3, D - 2] = np.inf
    z = c.forward(dev)["Z"]
    assert np.all(z[:, 3] == np.inf) and np.isfinite(np.delete(z, 3, axis=1)).all()
