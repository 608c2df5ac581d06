"""The paged operators at the ends of their arguments' ranges, without a GPU."""
import math

import pytest

from ancha_amd import paged


@pytest.mark.parametrize("how", [(4, 1e4, "ntk", 1e200), (4, 1e300, "ntk", 1e5), (64, 10.0, "ntk", 1e308),
                                 (64, 1e4, "yarn", 2.0, 2 ** 2000), (64, 1e4, "yarn", 2.0, 2 ** 53 + 1)])
def test_frequencies_beyond_64_bits_are_refused(how):
    with pytest.raises(ValueError, match="beyond 64-bit|original"):
        paged.frequencies(*how)


def test_frequencies_of_the_largest_bases():
    f, _ = paged.frequencies(4, 1e100, "ntk", 1e100)
    assert f[0] == 1 and math.isclose(f[1], 1e-150, rel_tol=1e-12)
    f, _ = paged.frequencies(64, 1e4, "yarn", 1e300, 2 ** 53)
    assert f[0] == 1 and all(0 < x <= 1 for x in f)
