"""YaRN frequencies against their definition, over original contexts from short to long."""
import math

import pytest


@pytest.mark.parametrize("dim,base", [(32, 10000.0), (64, 10000.0), (64, 500000.0), (96, 10000.0), (128, 10000.0),
                                      (128, 1000000.0), (256, 10000.0)])
@pytest.mark.parametrize("original", [2 ** n for n in range(8, 19)])
def test_yarn_over_original_lengths(fa, dim, base, original):
    """Pair j turns original * base^(-2j / dim) / 2 pi times.  The ramp begins at the last whole j that
    turns 32 times or more and ends at the first that turns once or less, which may lie behind the
    last pair (the method bounds it by dim - 1); between them it is linear in j."""
    factor = 4.0
    plain, _ = fa.rotary_frequencies(dim, base)
    got, table_factor = fa.rotary_frequencies(dim, base, scaling="yarn", factor=factor, original_positions=original)
    assert table_factor == pytest.approx(0.1 * math.log(factor) + 1.0, rel=1e-15)

    def turns(j):
        return original * base ** (-2.0 * j / dim) / (2 * math.pi)

    low = max(j for j in range(-1, dim) if turns(j) >= 32.0 or j == -1)
    high = min(j for j in range(dim) if turns(j) <= 1.0 or j == dim - 1)
    low = max(low, 0)
    for j, (f, g) in enumerate(zip(plain, got)):
        share = min(1.0, max(0.0, (j - low) / (high - low))) if high > low else float(j > low)
        assert g == pytest.approx(f * (1 - share) + f / factor * share, rel=1e-12), (j, low, high)
        if turns(j) >= 32.0:
            assert g == f
        assert (g <= f / factor * (1 + 1e-12)) == (turns(j) <= 1.0), (j, turns(j), g / f)
