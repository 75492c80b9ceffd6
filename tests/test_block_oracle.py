"""The oracles of tests/block_oracle.py against differences of their own forward values (CPU)."""
import numpy as np
import pytest

import block_oracle as O
from anneal_amd import _lib as L


def differences(f, x, h=1e-6):
    """The gradient of f by central differences."""
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        v = x[i]
        x[i] = v + h
        a = f()
        x[i] = v - h
        g[i] = (a - f()) / (2 * h)
        x[i] = v
    return g


@pytest.mark.parametrize("kind", O.ACTS)
@pytest.mark.parametrize("factor", [True, False])
def test_linear(kind, factor):
    r = np.random.default_rng(kind)
    X, W, b, dY = r.standard_normal((5, 4)), r.standard_normal((3, 4)), r.standard_normal(3), r.standard_normal((5, 3))
    U, R = (r.standard_normal((5, 3)) if factor else None), r.standard_normal((5, 3))
    f = lambda: float((O.linear(X, W, b, U, R, kind, 0.5)["Y"][0] * dY).sum())   # noqa: E731
    g = O.linear_grad(X, W, O.linear(X, W, b)["Z"][0], dY, U, kind, 0.5)
    for k, v in {"dX": X, "dW": W, "dbias": b, **({"dU": U} if factor else {})}.items():
        np.testing.assert_allclose(g[k][0], differences(f, v), rtol=1e-6, atol=1e-7)


@pytest.mark.parametrize("post", range(3))
@pytest.mark.parametrize("pre", range(3))
@pytest.mark.parametrize("per", [0, 1, 2])
def test_norms(post, pre, per):
    r = np.random.default_rng([post, pre, per])
    N, D = 5, 4
    H, Y = r.standard_normal((N, D)), r.standard_normal((N, D))
    gate = r.standard_normal((-(-N // per) if per else 1, D))
    w = {k: r.standard_normal(D) for k in ("post_w", "post_b", "pre_w", "pre_b")}
    dH, dO = r.standard_normal((N, D)), r.standard_normal((N, D)) if pre else None
    kw = dict(gate=gate, per=per, post=post, pre=pre, eps=1e-2, skip=0.75, scale=0.5)

    def f():
        o = O.residual_norm(H, Y, **kw, **w)
        return float((o["H_out"][0] * dH).sum() + ((o["O"][0] * dO).sum() if pre else 0.0))

    args = {k: v for k, v in w.items() if k != "pre_b"}
    g = O.residual_norm_grad(O.residual_norm(H, Y, **kw, **w)["H_out"][0], Y, dH, dO, **kw, **args)
    leaves = {"dH": H, "dY": Y, "dgate": gate, **({"dpost_w": w["post_w"]} if post else {}), **({"dpost_b": w["post_b"]} if post == L.NORM_LAYER else {}),
              **({"dpre_w": w["pre_w"]} if pre else {}), **({"dpre_b": w["pre_b"]} if pre == L.NORM_LAYER else {})}
    for k, v in leaves.items():
        np.testing.assert_allclose(g[k][0], differences(f, v), rtol=1e-6, atol=1e-7, err_msg=k)
