"""ah_residual_norm and ah_residual_norm_grad against their formulas in 64 bits (GPU). Bounds as derived in block_oracle.py."""
import numpy as np
import pytest

import block_oracle as O
from anneal_amd import _lib as L
from test_gpu_linear import Strided

pytestmark = pytest.mark.gpu
TYPES = [(L.AH_F32, L.AH_F32), (L.AH_F16, L.AH_F16), (L.AH_F16, L.AH_F32)]
IDS = ["f32", "f16", "f16_f32res"]
NONE, RMS, LAYER = L.NORM_NONE, L.NORM_RMS, L.NORM_LAYER
# rows and columns: one of each, every number of threads a row, ragged and past a workgroup's registers
SHAPES = [(1, 1), (1, 8), (3, 5), (7, 64), (33, 65), (1, 200), (40, 256), (9, 511), (130, 513), (2, 1001), (50, 2048), (6, 4095), (20, 4100), (3, 8192), (5, 8200), (2, 20001)]


class Case:
    def __init__(self, N, D, types=(L.AH_F32, L.AH_F32), post=RMS, pre=RMS, per=0, gate=True, H=True, Y=True, weights=True, eps=1e-6, seed=0):
        r = np.random.default_rng([seed, N, D, post, pre, per])
        self.N, self.D, self.types = N, D, types
        t, tr = O.NP[types[0]], O.NP[types[1]]
        self.kw = dict(per=per, post=post, pre=pre, eps=eps, skip=0.9375, scale=0.5)
        self.H = (3 * r.standard_normal((N, D)) + 0.5).astype(tr) if H else None
        self.Y = (r.standard_normal((N, D)) + 0.25).astype(t) if Y else None
        self.gate = r.standard_normal((-(-N // per) if per else 1, D)).astype(t) if gate and Y else None
        self.w = {}
        for k, kind in (("post", post if Y else NONE), ("pre", pre)):
            if weights and kind != NONE:
                self.w[k + "_w"] = (1 + 0.25 * r.standard_normal(D)).astype(t)
            if weights and kind == LAYER:
                self.w[k + "_b"] = (0.25 * r.standard_normal(D)).astype(t)
        self.dH_out, self.dO = r.standard_normal((N, D)).astype(tr), (r.standard_normal((N, D)).astype(t) if pre != NONE else None)

    def args(self, arrays, dev, gap):
        """Device arrays with their strides."""
        a = {k: Strided(dev, v, t, gap if k not in ("post_w", "post_b", "pre_w", "pre_b") else 0) for k, (v, t) in arrays.items() if v is not None}
        names = {"H": "ldh", "Y": "ldy", "gate": "ldgate", "H_out": "ldh_out", "O": "ldo", "dH_out": "lddh_out", "dO": "lddo", "dH": "lddh", "dY": "lddy",
                 "dgate": "lddgate"}
        return a, {names[k]: v.ld for k, v in a.items() if k in names}

    def common(self):
        k = self.kw
        return dict(dtype=self.types[0], res_dtype=self.types[1], N=self.N, D=self.D, post=k["post"], pre=k["pre"], rows_per_gate=k["per"], eps=k["eps"],
                    skip=k["skip"], scale=k["scale"])

    def forward(self, dev, gap=0, in_place=False, want=("H_out", "O")):
        t, tr = self.types
        a, ld = self.args({"H": (self.H, tr), "Y": (self.Y, t), "gate": (self.gate, t), **{k: (v, t) for k, v in self.w.items()}}, dev, gap)
        empty = np.full((self.N, self.D), np.nan)
        o, ldo = self.args({k: (empty, tr if k == "H_out" else t) for k in want if k != "O" or self.kw["pre"] != NONE}, dev, gap)
        if in_place:
            o["H_out"].free()
            o["H_out"] = a["H"]
        dev.residual_norm(**self.common(), **a, **o, **ld, **ldo)
        dev.sync()
        got = {k: v.read() for k, v in o.items()}
        for v in {id(v): v for v in [*a.values(), *o.values()]}.values():
            v.free()
        return got

    def expected(self):
        return O.residual_norm(self.H, self.Y, self.gate, **self.kw, **self.w, dtype=self.types[0], res_dtype=self.types[1])

    def outputs(self):
        kinds = {"post": self.kw["post"], "pre": self.kw["pre"]}
        out = ["dH"] + (["dY"] if self.Y is not None else []) + (["dgate"] if self.gate is not None else [])
        for k, kind in kinds.items():
            out += (["d" + k + "_w"] if kind != NONE else []) + (["d" + k + "_b"] if kind == LAYER else [])
        return out

    def backward(self, dev, gap=0, in_place=False, want=None):
        t, tr = self.types
        w = {k: (v, t) for k, v in self.w.items() if k != "pre_b"}
        a, ld = self.args({"H_out": (self.H if self.kw["pre"] != NONE else None, tr), "Y": (self.Y, t), "gate": (self.gate, t), "dH_out": (self.dH_out, tr),
                           "dO": (self.dO, t), **w}, dev, gap)
        shapes = {"dH": (self.N, self.D), "dY": (self.N, self.D), "dgate": None if self.gate is None else self.gate.shape}
        kind = {"dH": tr, "dY": t, "dgate": t}
        o, ldo = self.args({k: (np.full(shapes.get(k, (1, self.D)), np.nan), kind.get(k, L.AH_F32)) for k in (want or self.outputs())}, dev, 0)
        if in_place:
            o["dH"].free()
            o["dH"], ldo["lddh"] = a["dH_out"], a["dH_out"].ld
        kw = dict(**self.common(), **a, **o, **ld, **ldo)
        ws = dev.buffer(dev.residual_norm_grad_workspace(**kw) // 4 + 4)
        dev.residual_norm_grad(ws=ws, **kw)
        dev.sync()
        got = {k: v.read() for k, v in o.items()}
        for v in {id(v): v for v in [*a.values(), *o.values(), ws]}.values():
            v.free()
        return got

    def gradients(self):
        w = {k: v for k, v in self.w.items() if k != "pre_b"}
        return O.residual_norm_grad(self.H, self.Y, self.dH_out, self.dO, self.gate, **self.kw, **w, dtype=self.types[0], res_dtype=self.types[1])


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("kinds", [(RMS, RMS), (LAYER, LAYER)], ids=["rms", "layer"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_shapes(dev, shape, kinds, types):
    c = Case(*shape, types=types, post=kinds[0], pre=kinds[1], eps=1e-2 if shape[1] == 1 else 1e-6)
    O.compare(c.forward(dev), c.expected())
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("post", [NONE, RMS, LAYER])
@pytest.mark.parametrize("pre", [NONE, RMS, LAYER])
@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("shape", [(37, 72), (11, 1000), (3, 8300)], ids=lambda s: "%dx%d" % s)
def test_kinds(dev, shape, post, pre, weights):
    c = Case(*shape, types=TYPES[2], post=post, pre=pre, weights=weights, per=4)
    O.compare(c.forward(dev), c.expected())
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("per", [0, 1, 2, 3, 7, 64, 250, 999, 1000, 5000])
@pytest.mark.parametrize("shape", [(1000, 40), (1000, 520), (300, 8200), (1, 64)], ids=lambda s: "%dx%d" % s)
def test_gates(dev, shape, per):
    """A gate for all rows, for runs of any length (whole in one worker, shared by two or by many, the last one short) and for each row."""
    c = Case(*shape, types=TYPES[1], per=per)
    O.compare(c.forward(dev), c.expected())
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(20, 100), (20, 1000), (5, 9000)], ids=lambda s: "%dx%d" % s)
def test_parts(dev, shape, types):
    """No residual stream, no branch, no gate; one output of the two; no gradient of H_out."""
    for kw in (dict(H=False), dict(Y=False, post=NONE), dict(gate=False)):
        c = Case(*shape, types=types, **kw)
        O.compare(c.forward(dev), c.expected())
    for want in ("H_out",), ("O",):
        c = Case(*shape, types=types)
        if want == ("H_out",):
            c = Case(*shape, types=types, pre=NONE)
        O.compare(c.forward(dev, want=want), c.expected())
    c = Case(*shape, types=types, Y=False, post=NONE)
    O.compare(c.backward(dev), c.gradients())
    c = Case(*shape, types=types)
    c.dH_out = None
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("shape", [(30, 200), (30, 700), (4, 8200)], ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("types", TYPES, ids=IDS)
def test_single_outputs(dev, shape, types):
    """Each alone: the bits of the call with all."""
    c = Case(*shape, types=types, post=LAYER, pre=LAYER, per=8)
    full = c.backward(dev)
    for k in c.outputs():
        np.testing.assert_array_equal(c.backward(dev, want=(k,))[k], full[k], err_msg=k)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("gap", [1, 8])
@pytest.mark.parametrize("shape", [(19, 64), (19, 1500), (3, 8201)], ids=lambda s: "%dx%d" % s)
def test_strides_and_in_place(dev, shape, gap, types):
    """Rows further apart at any alignment, what lies between them left; H_out over H, dH over dH_out."""
    c = Case(*shape, types=types, post=LAYER, pre=RMS, per=5)
    O.compare(c.forward(dev, gap=gap), c.expected())
    O.compare(c.forward(dev, gap=gap, in_place=True), c.expected())
    O.compare(c.backward(dev, gap=gap), c.gradients())
    O.compare(c.backward(dev, gap=gap, in_place=True), c.gradients())


@pytest.mark.parametrize("kind", [RMS, LAYER])
@pytest.mark.parametrize("D", [64, 1000, 9000])
def test_rows_of_zeros_and_constants(dev, D, kind):
    """eps alone divides them: a zero row gives zeros and finite gradients, and a constant one is nothing to a layer norm."""
    c = Case(6, D, post=kind, pre=kind, gate=False, weights=False, eps=1e-3)
    c.H[1], c.Y[1], c.H[2], c.Y[3] = 0, 0, 4.0, 2.0
    got = c.forward(dev)
    O.compare(got, c.expected())
    assert not got["O"][1].any() and not got["H_out"][1].any()
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("bad", [np.nan, np.inf], ids=str)
@pytest.mark.parametrize("shape", [(30, 24), (30, 200), (30, 600), (6, 9000)], ids=lambda s: "%dx%d" % s)
def test_a_row_that_is_not_finite_leaves_the_others(dev, shape, bad):
    clean, c = Case(*shape, per=1), Case(*shape, per=1)
    c.H[4, 3] = bad
    keep = np.arange(shape[0]) != 4
    got, want = c.forward(dev), clean.expected()
    O.compare({k: v[keep] for k, v in got.items()}, {k: tuple(x[keep] for x in v) for k, v in want.items()})
    assert not np.isfinite(got["O"][4]).all() and not np.isfinite(got["H_out"][4, 3])
    got, want = c.backward(dev), clean.gradients()
    rows = ("dH", "dY", "dgate")
    O.compare({k: got[k][keep] for k in rows}, {k: tuple(x[keep] for x in want[k]) for k in rows})
    assert not np.isfinite(got["dH"][4]).all()


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(5000, 96), (3000, 768), (1500, 4096), (700, 6000)], ids=lambda s: "%dx%d" % s)
def test_many_rows(dev, shape, types):
    """Runs of many rows, a gate that several share; results repeat."""
    c = Case(*shape, types=types, post=RMS, pre=LAYER, per=700)
    O.compare(c.forward(dev), c.expected())
    got, again = c.backward(dev), c.backward(dev)
    O.compare(got, c.gradients())
    for k in got:
        np.testing.assert_array_equal(got[k], again[k], err_msg=k)


def test_gradients_against_differences(dev):
    """Central differences of the call's own forward pass along random directions (f32 results off by 2^-21 or so of their terms)."""
    c = Case(32, 72, post=LAYER, pre=RMS, per=5)
    stream = c.H.copy()
    c.H = c.forward(dev)["H_out"].astype(np.float32)
    g = c.backward(dev)
    c.H = stream
    r = np.random.default_rng(0)
    h = 2.0 ** -6
    for name, grad in (("H", "dH"), ("Y", "dY"), ("gate", "dgate"), ("post_w", "dpost_w"), ("post_b", "dpost_b"), ("pre_w", "dpre_w")):
        home = c.w if name in c.w else c.__dict__
        base = home[name].copy()
        d = r.standard_normal(base.shape).astype(np.float32)
        d /= np.float32(np.linalg.norm(d))
        values = []
        for s in (h, -h):
            home[name] = (base + np.float32(s) * d).astype(np.float32)
            y = c.forward(dev)
            values.append((y["H_out"].astype(np.float64) * c.dH_out).sum() + (y["O"].astype(np.float64) * c.dO).sum())
        home[name] = base
        want = (values[0] - values[1]) / (2 * h)
        noise = 2.0 ** -21 * 8 * (np.linalg.norm(c.dH_out) + np.linalg.norm(c.dO)) / h
        assert abs(float((g[grad].reshape(base.shape) * d).sum()) - want) <= noise + h * h * 16, name


@pytest.mark.parametrize("kinds", [(RMS, RMS), (LAYER, LAYER), (NONE, RMS), (LAYER, NONE)], ids=lambda k: "%d_%d" % k)
@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** 40])
@pytest.mark.parametrize("shape", [(9, 100), (9, 1001), (3, 5000)], ids=lambda s: "%dx%d" % s)
def test_sizes_of_gradients(dev, shape, size, kinds):
    """Gradients far from 1 beside a stream and a branch of 2^10 (f32): a row's sums of products keep to the bounds of one norm after the other."""
    c = Case(*shape, post=kinds[0], pre=kinds[1], per=2)
    c.H, c.Y = c.H * np.float32(2.0 ** 10), c.Y * np.float32(2.0 ** 10)
    c.dH_out = c.dH_out * np.float32(size)
    if c.dO is not None:
        c.dO = c.dO * np.float32(size)
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("D", [8193, 12000, 16384, 16385])
def test_two_groups_of_columns(dev, D, types):
    """Rows past 8192 columns, held in registers up to 16384, and the first that is not."""
    c = Case(3, D, types=types, post=RMS, pre=LAYER, per=2)
    O.compare(c.forward(dev, gap=1), c.expected())
    O.compare(c.forward(dev, gap=1, in_place=True), c.expected())
    O.compare(c.backward(dev, gap=1, in_place=True), c.gradients())
