"""ah_residual_norm and ah_residual_norm_grad on rows far from 1 (GPU). Bounds as derived in block_oracle.py."""
import numpy as np
import pytest

import block_oracle as O
from anneal_amd import _lib as L
from test_gpu_residual_norm import LAYER, NONE, RMS, Case

pytestmark = pytest.mark.gpu
SHAPES = [(9, 64), (9, 1001), (3, 5000)]


@pytest.mark.parametrize("kinds", [(RMS, RMS), (LAYER, LAYER), (RMS, NONE), (LAYER, NONE), (NONE, RMS), (NONE, LAYER)], ids=lambda k: "%d_%d" % k)
@pytest.mark.parametrize("power", [-55, -46, -30, 30, 46, 50, 55])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_gradients_of_far_rows(dev, shape, power, kinds):
    """Branch and stream far from 1, where r^3 leaves f32's range and nothing that is needed does; small ones without eps, which would hide
    them."""
    c = Case(*shape, post=kinds[0], pre=kinds[1], per=2, eps=0.0 if power < 0 else 1e-6)
    c.H, c.Y = (v * np.float32(2.0 ** power) for v in (c.H, c.Y))
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("kinds", [(RMS, RMS), (LAYER, LAYER)], ids=["rms", "layer"])
@pytest.mark.parametrize("powers", [(50, -40), (-46, 40), (55, 0), (0, 55)], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
def test_branch_and_stream_apart(dev, shape, powers, kinds):
    c = Case(*shape, post=kinds[0], pre=kinds[1], eps=0.0)
    c.Y, c.H = c.Y * np.float32(2.0 ** powers[0]), c.H * np.float32(2.0 ** powers[1])
    O.compare(c.backward(dev), c.gradients())


@pytest.mark.parametrize("kinds", [(RMS, RMS), (LAYER, LAYER), (RMS, NONE), (NONE, LAYER)], ids=lambda k: "%d_%d" % k)
@pytest.mark.parametrize("power", [-118, -100, -75, -60, 60, 64, 67, 90, 110])
@pytest.mark.parametrize("shape", [(9, 7), (9, 64), (9, 200), (9, 1001), (3, 5000), (3, 12000), (2, 20001)], ids=lambda s: "%dx%d" % s)
def test_squares_past_the_range(dev, shape, power, kinds):
    """Some rows whose squares are past f32's range, or with a tiny eps below it, beside ordinary ones."""
    c = Case(*shape, post=kinds[0], pre=kinds[1], per=1, eps=2.0 ** -300 if power < 0 else 1e-6)
    for v, rows in ((c.H, (0, 2)), (c.Y, (0, 1))):
        for r in rows:
            if r < shape[0]:
                v[r] *= np.float32(2.0 ** power)
    if kinds[0] == NONE:   # the branch is not normed: what goes into the stream's sum stays far below it
        c.Y[1] = 0
    O.compare(c.forward(dev), c.expected())
    O.compare(c.forward(dev, in_place=True, gap=1), c.expected())


@pytest.mark.parametrize("kind", [RMS, LAYER])
@pytest.mark.parametrize("D", [40, 777, 4099, 9000, 20001])
def test_one_large_entry(dev, D, kind):
    """One entry of 1e20 leaves a row that is almost nothing beside it; under RMS also the largest that f32 has."""
    for big in (1e20, 3e38) if kind == RMS else (1e20,):
        c = Case(5, D, post=kind, pre=kind, gate=False)
        c.H[1, 3], c.Y[2, D - 1] = big, -big
        O.compare(c.forward(dev), c.expected())


@pytest.mark.parametrize("kinds", [(RMS, RMS), (LAYER, LAYER)], ids=["rms", "layer"])
@pytest.mark.parametrize("types", [0, 1], ids=["f32", "f16_f32res"])
def test_zeros_without_eps(dev, types, kinds):
    """0 / 0 is NaN in its own row, as a row that is not finite has it, and the others are as ever."""
    c = Case(6, 300, types=[(L.AH_F32, L.AH_F32), (L.AH_F16, L.AH_F32)][types], post=kinds[0], pre=kinds[1], gate=False, weights=False, eps=0.0)
    c.Y[2] = 0
    keep = np.arange(6) != 2
    with np.errstate(all="ignore"):
        got, want = c.forward(dev), c.expected()
    O.compare({k: v[keep] for k, v in got.items()}, {k: tuple(x[keep] for x in v) for k, v in want.items()})
    assert np.isnan(got["H_out"][2]).all() and np.isnan(got["O"][2]).all()


@pytest.mark.parametrize("kind", [RMS, LAYER])
@pytest.mark.parametrize("which", ["Y", "H"])
@pytest.mark.parametrize("D", [40, 777, 9000])
def test_gradients_past_the_range_are_not_zeros(dev, D, which, kind):
    """A row whose squares are past f32's range has gradients of NaN, not of 0, and leaves the others."""
    clean, c = Case(5, D, post=kind, pre=kind, per=1), Case(5, D, post=kind, pre=kind, per=1)
    getattr(c, which)[3, 2:6] = 1e20
    keep = np.arange(5) != 3
    got, want = c.backward(dev), clean.gradients()
    rows = ("dH", "dY", "dgate")
    O.compare({k: got[k][keep] for k in rows}, {k: tuple(x[keep] for x in want[k]) for k in rows})
    assert np.isnan(got["dY"][3]).all() and (which == "Y" or np.isnan(got["dH"][3]).all())


@pytest.mark.parametrize("kind", [RMS, LAYER])
@pytest.mark.parametrize("D", [40, 1000, 9000])
def test_gradients_of_zeros_under_a_tiny_eps(dev, D, kind):
    """eps is a subnormal f32 and divides a row of zeros: its gradients are large and finite."""
    c = Case(4, D, post=kind, pre=kind, gate=False, weights=False, eps=2.0 ** -130)
    c.H[:], c.Y[:] = 0, 0
    c.dH_out, c.dO = c.dH_out * np.float32(2.0 ** -20), c.dO * np.float32(2.0 ** -90)
    O.compare(c.forward(dev), c.expected())
    O.compare(c.backward(dev), c.gradients())
