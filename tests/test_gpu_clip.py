"""ah_clip_norm against its formula in 64 bits (GPU).

norm is a sum of exact squares in f64 (f16 ones eight at a time in f32, 8 U32 of their sum), a root and one rounding to f32; an output is
its input times a factor with one rounding, and its own rounding."""
import numpy as np
import pytest

from anneal_amd import _lib as L

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
NP = {L.AH_F16: np.float16, L.AH_F32: np.float32}
PAIRS = [(L.AH_F32, L.AH_F32), (L.AH_F16, L.AH_F16), (L.AH_F16, L.AH_F32)]
SIZES = [1, 2, 3, 7, 8, 9, 63, 64, 1000, 2047, 2048, 2049, 4096, 8191, 8192, 8193, 20000, 100003]


def run(dev, arrays, types, max_norm=1.0, eps=1e-6, unscale=1.0, in_place=False, count_only=(), offset=0):
    """arrays lie one after the other in one buffer a type, from `offset` elements on. Returns outputs (None: not written), norm, coef."""
    src, dst, rows = [], [], []
    for a, (t, to) in zip(arrays, types):
        src.append(dev.buffer(np.concatenate([np.zeros(offset, NP[t]), a.astype(NP[t])]), t))
        dst.append(src[-1] if in_place else dev.buffer(np.full(a.size + offset + 3, 777.0, NP[to]), to))

    class At:
        def __init__(self, b, t):
            self.ptr = b.ptr + offset * np.dtype(NP[t]).itemsize
    for i, (a, (t, to)) in enumerate(zip(arrays, types)):
        rows.append((At(src[i], t), None if i in count_only else At(dst[i], to), a.size, t, to))
    tensors = dev.tensor_list(rows)
    norm, coef = dev.buffer(1), dev.buffer(1)
    kw = dict(tensors=tensors, max_norm=max_norm, eps=eps, unscale=unscale, norm=norm, coef=coef)
    ws = dev.buffer(dev.clip_norm_workspace(**kw) // 4 + 4)
    dev.clip_norm(ws=ws, **kw)
    dev.sync()
    out = []
    for i, a in enumerate(arrays):
        got = dst[i].read()
        if not in_place:
            assert np.all(got[:offset] == 777.0) and np.all(got[offset + a.size:] == 777.0), "written beside the tensor"
            if i in count_only:
                assert np.all(got == 777.0)
        out.append(None if i in count_only else got[offset: offset + a.size])
    n, c = float(norm.read()[0]), float(coef.read()[0])
    for b in {id(b): b for b in [*src, *dst, norm, coef, ws]}.values():
        b.free()
    return out, n, c


def check(arrays, types, got, max_norm=1.0, eps=1e-6, unscale=1.0, count_only=()):
    out, n, c = got
    eps, unscale, max_norm = float(np.float32(eps)), float(np.float32(unscale)), float(np.float32(max_norm))
    exact = [a.astype(NP[t]).astype(np.float64) for a, (t, _) in zip(arrays, types)]
    norm = unscale * np.sqrt(sum(float((a * a).sum()) for a in exact))
    coef = min(1.0, max_norm / (norm + eps)) if norm + eps > 0 else 1.0
    if norm > np.finfo(np.float32).max:   # its rounding to f32 is an infinity
        assert np.isposinf(n)
    else:
        assert abs(n - norm) <= 6 * U32 * norm + 2.0 ** -149
    assert abs(c - coef) <= 6 * U32 * coef + 2.0 ** -149
    for i, (a, o, (_, to)) in enumerate(zip(exact, out, types)):
        if i in count_only:
            continue
        want = unscale * coef * a
        tol = 8 * U32 * np.abs(want) + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if to == L.AH_F16 else 2.0 ** -149)
        assert np.all(np.abs(o.astype(np.float64) - want) <= tol), i


@pytest.mark.parametrize("types", PAIRS, ids=["f32", "f16", "f16_f32"])
@pytest.mark.parametrize("n", SIZES)
@pytest.mark.parametrize("offset", [0, 1])
def test_one_tensor(dev, n, types, offset):
    a = [np.random.default_rng(n).standard_normal(n)]
    for max_norm in (1e6, 0.5 * n ** 0.5):
        check(a, [types], run(dev, a, [types], max_norm, offset=offset), max_norm)
        if types[0] == types[1]:
            check(a, [types], run(dev, a, [types], max_norm, in_place=True, offset=offset), max_norm)


@pytest.mark.parametrize("n", [1, 5, 89, 90, 91, 180, 181, 1000])
def test_many_tensors(dev, n):
    """As many as travel with the launch, and more; empty ones first, last and between; types mixed; some only counted."""
    r = np.random.default_rng(n)
    arrays = [r.standard_normal(0 if i % 5 == 0 else int(r.integers(1, 6000))) * 10.0 ** r.uniform(-3, 1) for i in range(n)]
    types = [PAIRS[i % 3] for i in range(n)]
    only = [i for i in range(n) if i % 7 == 3]
    check(arrays, types, run(dev, arrays, types, 2.0, count_only=only), 2.0, count_only=only)


def test_a_large_tensor_among_small_ones(dev):
    r = np.random.default_rng(0)
    arrays = [r.standard_normal(10), r.standard_normal(20_000_001), r.standard_normal(3), r.standard_normal(5_000_000)]
    types = [PAIRS[0], PAIRS[0], PAIRS[1], PAIRS[2]]
    a, b = (run(dev, arrays, types, 1.0, offset=1) for _ in range(2))
    check(arrays, types, a)
    assert a[1:] == b[1:] and all(np.array_equal(x, y) for x, y in zip(a[0], b[0]))


def test_only_empty_tensors(dev):
    out, n, c = run(dev, [np.zeros(0)] * 3, [PAIRS[0]] * 3)
    assert n == 0.0 and c == 1.0


@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e19, 1e37])
def test_squares_past_the_range_of_f32(dev, size):
    a = [np.random.default_rng(3).standard_normal(5000) * size]
    check(a, [PAIRS[0]], run(dev, a, [PAIRS[0]], size, eps=0.0), size, 0.0)


def test_a_norm_past_the_range_of_f32(dev):
    a = [np.full(1000, 3e38)]
    out, n, c = run(dev, a, [PAIRS[0]], 1.0)
    assert np.isposinf(n) and 0.0 < c < 2.0 ** -126   # a subnormal, but the outputs have all of f32's bits
    np.testing.assert_allclose(out[0], 1000 ** -0.5, rtol=1e-6)


@pytest.mark.parametrize("unscale", [2.0 ** -10, 3.0])
def test_loss_scales(dev, unscale):
    r = np.random.default_rng(1)
    arrays = [100 * r.standard_normal(3000), 100 * r.standard_normal(50)]
    for max_norm in (1.0, 1e9, float("inf")):
        types = [PAIRS[1], PAIRS[2]]
        check(arrays, types, run(dev, arrays, types, max_norm, unscale=unscale), max_norm, unscale=unscale)


@pytest.mark.parametrize("max_norm,eps", [(0.0, 1e-6), (0.0, 0.0), (1.0, 0.0)])
def test_limits(dev, max_norm, eps):
    for a in ([np.zeros(100)], [np.ones(100)]):
        check(a, [PAIRS[0]], run(dev, a, [PAIRS[0]], max_norm, eps), max_norm, eps)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf], ids=str)
@pytest.mark.parametrize("n", [3, 200])
@pytest.mark.parametrize("in_place", [False, True])
def test_what_is_not_finite_stops_the_update(dev, n, bad, in_place):
    """norm says so, coef is 0 and every output 0."""
    r = np.random.default_rng(2)
    arrays, types = [r.standard_normal(500) for _ in range(n)], [PAIRS[i % 2] for i in range(n)]
    arrays[n // 2][77] = bad
    out, norm, c = run(dev, arrays, types, 1.0, in_place=in_place)
    assert not np.isfinite(norm) and c == 0.0 and all(not o.any() for o in out)
    assert np.isnan(norm) == np.isnan(bad)


def test_tensors_within_the_norm_stay_as_they_are(dev):
    """In place with unscale coef = 1: the bits of the inputs, NaN-free or not touched at all."""
    a = [np.random.default_rng(5).standard_normal(3000)]
    out, _, c = run(dev, a, [PAIRS[0]], 1e9, in_place=True)
    assert c == 1.0
    np.testing.assert_array_equal(out[0], a[0].astype(np.float32))
