"""ah_clip_norm with factors below f32's normal numbers (GPU). Bounds as in test_gpu_clip.py."""
import numpy as np
import pytest

from test_gpu_clip import PAIRS, check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-40, -60, -70, -100, -126])
@pytest.mark.parametrize("unscale", [1.0, 2.0 ** -20])
@pytest.mark.parametrize("n", [5, 9001])
def test_a_factor_of_few_bits(dev, n, unscale, power):
    """Entries near f32's largest and a norm that they are to be brought to near its smallest: the factor is below 2^-126 and the outputs are not."""
    a = [3e38 * np.random.default_rng(n).uniform(-1, 1, n)]
    max_norm = 2.0 ** power
    check(a, [PAIRS[0]], run(dev, a, [PAIRS[0]], max_norm, eps=0.0, unscale=unscale), max_norm, eps=0.0, unscale=unscale)
    check(a, [PAIRS[0]], run(dev, a, [PAIRS[0]], max_norm, eps=0.0, unscale=unscale, in_place=True), max_norm, eps=0.0, unscale=unscale)


@pytest.mark.parametrize("power", [-30, -60, -66, -90, -130])
def test_small_entries_beside_large_ones(dev, power):
    """What the factor brings below f32's normal numbers is off by its own rounding and one in its last place."""
    a = [np.concatenate([[3e38], 2.0 ** np.linspace(-149, 127, 500) * np.random.default_rng(1).uniform(1, 2, 500) * 0.49])]
    check(a, [PAIRS[0]], run(dev, a, [PAIRS[0]], 2.0 ** power, eps=0.0), 2.0 ** power, eps=0.0)
