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
