"""ah_linear and ah_linear_grad where values of one array differ in size by far more than a plane's bits (GPU). Bounds as derived in
block_oracle.py, taken as they stand."""
import numpy as np
import pytest
from scipy.special import erfc

import block_oracle as O
from anneal_amd import _lib as L
from block_oracle import U32
from test_gpu_linear import IDS, TYPES, Case

pytestmark = pytest.mark.gpu
KINDS = [L.ACT_RELU, L.ACT_GELU, L.ACT_GELU_TANH, L.ACT_SILU]
OFF = 11   # a feature that is off for every row
BIG = {(L.AH_F32, L.AH_F32): 1e4, (L.AH_F16, L.AH_F16): 3e4, (L.AH_F16, L.AH_F32): 4e3}
SMALL = {(L.AH_F32, L.AH_F32): 1e-3, (L.AH_F16, L.AH_F16): 1e-2, (L.AH_F16, L.AH_F32): 1e-2}


def inactive(N, types, kind, z, factor=True, D=96, F=64):
    """dY and U are large where the activation is off, and nowhere else."""
    c = Case(N, D, F, dtype=types[0], grad_dtype=types[1], kind=kind, bias=False, factor=factor, res=False)
    c.dY = (c.dY * SMALL[types]).astype(c.dY.dtype)
    c.dY[:, OFF], c.Z[:, OFF] = BIG[types], z
    if factor:
        c.U[:, OFF] = BIG[types]
    return c


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N", [1, 30, 200, 8400])   # 8400: dZ is bounded first, and stored again where the bound is loose
@pytest.mark.parametrize("factor", [True, False])
def test_what_is_off_does_not_set_the_scale(dev, N, kind, types, factor):
    """At z = -200 every slope but ReLU's is under 2^-280, in f32 as in f16 0: the gradients are those of a call whose dY is 0 there."""
    c = inactive(N, types, kind, -200.0, factor)
    got = c.backward(dev)
    c.dY[:, OFF] = 0
    O.compare(got, c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("z", [-4.0, -9.0, -30.0])
@pytest.mark.parametrize("N", [30, 200, 8400])
def test_what_is_nearly_off(dev, N, z, kind, types):
    c = inactive(N, types, kind, z)
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("N", [30, 200, 8400])
def test_one_entry_that_is_off(dev, N, types):
    """One large entry under ReLU, in a row and a column whose other entries are live."""
    c = Case(N, 96, 64, dtype=types[0], grad_dtype=types[1], kind=L.ACT_RELU, factor=False)
    c.dY[5, 7], c.Z[5, 7] = 2.0 ** 30 if types[0] == L.AH_F32 else 6e4, -1.0
    c.dY[np.arange(N) != 5] *= c.dY.dtype.type(2.0 ** -10)
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", [L.ACT_NONE, L.ACT_RELU, L.ACT_SILU])
@pytest.mark.parametrize("apart", [20, 30])
@pytest.mark.parametrize("N", [30, 200, 8400])
def test_rows_far_apart(dev, N, apart, kind, types):
    """Rows of dY 2^20 and 2^30 apart (f16: what its range has): what is under 2^-39 of the largest dZ may go."""
    c = Case(N, 96, 64, dtype=types[0], grad_dtype=types[1], kind=kind, factor=False)
    size = np.float32(2.0) ** -np.linspace(0, apart, N).astype(np.float32)[:, None]
    c.dY = (c.dY.astype(np.float32) * size).astype(c.dY.dtype)
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N", [30, 200, 8400])
def test_a_gradient_near_the_end_of_f32(dev, N, kind):
    """dZ fits f32 where dY times the largest slope of the GELUs does not."""
    c = Case(N, 96, 64, kind=kind, bias=False, factor=False, res=False, scale=1.0)
    c.W = (c.W * 2.0 ** -6).astype(np.float32)
    c.X = (c.X * 2.0 ** -20).astype(np.float32)
    c.dY[3, 4], c.Z[3, 4] = 3.3e38, 0.25
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [64.0, 2.0 ** -6])
def test_the_largest_in_any_place(dev, size, kind, types):
    """The largest dZ early and late, with larger ones that are off before it and after it, in more rows and columns than the scan's waves see
    at once; and the same bits again."""
    for at in (0, 701, 2999):
        c = Case(3000, 8, 2100, dtype=types[0], grad_dtype=types[1], kind=kind, factor=False)
        c.dY = (c.dY * 2.0 ** -8).astype(c.dY.dtype)
        c.Z[at, 2050], c.dY[at, 2050] = 3.0, size
        for off in (17, 1500, 2700):
            c.Z[off, ::5], c.dY[off, ::5] = -200.0, 3e4
        got, again = c.backward(dev), c.backward(dev)
        for off in (17, 1500, 2700):
            c.dY[off, ::5] = 0
        O.compare(got, c.gradients())
        for k in got:
            np.testing.assert_array_equal(got[k], again[k], err_msg=k)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf], ids=str)
@pytest.mark.parametrize("kind", [L.ACT_NONE, L.ACT_RELU, L.ACT_GELU])
@pytest.mark.parametrize("N", [30, 8400])
def test_what_is_not_finite_does_not_set_the_scale(dev, N, kind, bad, types):
    clean = Case(N, 96, 64, dtype=types[0], grad_dtype=types[1], kind=kind)
    clean.dY = (clean.dY * clean.dY.dtype.type(2.0 ** -8)).astype(clean.dY.dtype)
    c = Case(N, 96, 64, dtype=types[0], grad_dtype=types[1], kind=kind)
    c.dY = clean.dY.copy()
    c.dY[4, 9] = bad
    got, want = c.backward(dev), clean.gradients()
    rows, cols = np.arange(N) != 4, np.arange(64) != 9
    O.compare({"dX": got["dX"][rows], "dW": got["dW"][cols], "dU": got["dU"][rows]},
              {"dX": tuple(v[rows] for v in want["dX"]), "dW": tuple(v[cols] for v in want["dW"]), "dU": tuple(v[rows] for v in want["dU"])})
    assert not np.isfinite(got["dX"][4]).any() and not np.isfinite(got["dW"][9]).any()


@pytest.mark.parametrize("kind", [L.ACT_GELU, L.ACT_GELU_TANH, L.ACT_SILU])
@pytest.mark.parametrize("N", [1, 8400])
def test_f32_gradients_of_f16_operands_have_f32_slopes(dev, N, kind):
    """dbias of one live row is dZ itself. With e = 2^-24: e^x is off by 2^-22 of its value and 4 e |x| for its argument's roundings, 1 / (1 + e^x) by
    2^-22 of its value, s (1 - s) by 2^-21 and erfc by 2^-21 of theirs, and the last product and sum by 2 e of the slope. e^x may be 0 below 2^-126, the
    smallest normal f32: that times what it is multiplied with. (GELU's slope is p + z g with p from erfc: 1 + erf(z) is off by 2^-53 in f64, more than all
    of it at z = -12.)"""
    z = np.linspace(-12, 12, 4801).astype(np.float16)
    c = Case(N, 1, len(z), dtype=L.AH_F16, kind=kind, bias=False, factor=False, res=False, scale=1.0)
    c.dY[:], c.dY[0], c.Z[:] = 0, 1, z
    got = c.backward(dev, want=("dbias",))["dbias"][0].astype(np.float64)
    x, e = z.astype(np.float64), U32
    _, slope = O.act(kind, x)
    flushed = 2.0 ** -126
    if kind == L.ACT_GELU:
        p, g = 0.5 * erfc(-x / np.sqrt(2)), np.exp(-0.5 * x * x) / np.sqrt(2 * np.pi)
        slope = p + x * g
        flushed *= 1 + np.abs(x)
        tol = 2 ** -21 * p + 2 * e * g * np.abs(x) + np.abs(x * g) * (e * x * x + 2 ** -21)
    else:
        a, b = (1.0, 0.0) if kind == L.ACT_SILU else (2 * O._C, 2 * O._C * 0.044715)
        t = x * (a + b * x * x)
        s, s1 = 1 / (1 + np.exp(-t)), np.exp(-np.abs(t)) / (1 + np.exp(-np.abs(t))) ** 2
        arg = 4 * e * np.abs(t) if b else 0.0
        flushed *= 1 + np.abs(x) * (a + 3 * b * x * x)
        tol = np.abs(x) * s1 * (a + 3 * b * x * x) * (arg + 2 ** -21) + s1 * arg + 2 ** -22 * s
    tol = tol + 2 * e * np.abs(slope) + flushed
    assert np.all(np.abs(got - slope) <= tol), float(np.max(np.abs(got - slope) / tol))


@pytest.mark.parametrize("power", [-110, -126, -135])
@pytest.mark.parametrize("which", ["X", "W", "rows of X", "rows of W"])
def test_operands_near_the_beginning_of_f32(dev, which, power):
    """f32 operands down to f32's subnormals beside large ones: their planes hold what they have."""
    c = Case(200, 96, 64, kind=L.ACT_NONE, bias=False, factor=False, res=False, scale=1.0)
    small, other = (c.X, c.W) if "X" in which else (c.W, c.X)
    other *= np.float32(2.0 ** 100)
    rows = slice(3, 20) if "rows" in which else slice(None)
    small[rows] *= np.float32(2.0 ** power)
    O.compare(c.forward(dev), c.expected())
    if "rows" not in which:
        c.dY *= np.float32(2.0 ** 20)
        O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("power", [-110, -126, -135])
def test_gradients_near_the_beginning_of_f32(dev, power):
    c = Case(200, 96, 64, kind=L.ACT_RELU, bias=False, factor=False, res=False, scale=1.0)
    c.dY *= np.float32(2.0 ** power)
    c.X, c.W = c.X * np.float32(2.0 ** 100), c.W * np.float32(2.0 ** 100)
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("kind", [L.ACT_RELU, L.ACT_GELU])
def test_few_rows_of_many_features(dev, kind, types):
    """Few rows, whose dX reads W as it lies, with more features than are scanned for dZ's magnitude."""
    N, F = (60, 72000) if types[0] == L.AH_F16 else (100, 43008)
    c = inactive(N, types, kind, -200.0, D=16, F=F)
    got = c.backward(dev)
    c.dY[:, OFF] = 0
    O.compare(got, c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("N", [200, 8400])
def test_captured_with_other_gradients(dev, N, types):
    """A captured call, replayed on gradients whose largest is live, off, and live again: what one replay found is nothing to the next."""
    import ctypes as C
    a, b = inactive(N, types, L.ACT_GELU, -200.0), inactive(N, types, L.ACT_GELU, -200.0)
    a.dY[:, OFF] = 0
    arrays = {k: dev.buffer(getattr(a, k), types[0]) for k in ("X", "W", "Z", "U", "dY")}
    shapes = {"dX": (N, 96, types[1]), "dW": (64, 96, types[1]), "dbias": (1, 64, L.AH_F32), "dU": (N, 64, types[0])}
    out = {k: dev.buffer(np.full(s[:2], np.nan), s[2]) for k, s in shapes.items()}
    kw = dict(dtype=types[0], grad_dtype=types[1], N=N, D=96, F=64, act=a.kind, scale=a.scale, **arrays, **out)
    ws = dev.buffer(dev.linear_grad_workspace(**kw) // 4 + 4)
    g = C.c_void_p()
    L.check(dev.lib.ah_graph_begin(dev.h))
    dev.linear_grad(ws=ws, **kw)
    L.check(dev.lib.ah_graph_end(dev.h, C.byref(g)))
    want = {k: v for k, v in a.gradients().items()}   # of both: what is off adds nothing
    first = None
    for c in (a, b, a, b, b, a):
        arrays["dY"].write(c.dY)
        for k, s in shapes.items():
            out[k].write(np.full(s[:2], np.nan).astype(O.NP[s[2]]))
        L.check(dev.lib.ah_graph_replay(dev.h, g))
        dev.sync()
        got = {k: v.read().reshape(shapes[k][:2]) for k, v in out.items()}
        O.compare(got, want)
        first = first or got
        for k in got if c is a else ():
            np.testing.assert_array_equal(got[k], first[k], err_msg=k)
        dev.linear_grad(ws=ws, **kw)   # eager between the replays
    dev.sync()
    dev.lib.ah_graph_destroy(g)
