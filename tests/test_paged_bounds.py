"""The yardsticks of the paged attention's and the scoring's precision tests
see the mistakes that they are for (numpy only)."""
import numpy as np
import pytest

import precision_np as P


@pytest.mark.parametrize("dtype,parts", [("f16", 2), ("bf16", 3)])
@pytest.mark.parametrize("scene", list(P.SCENES))
def test_a_lost_part_is_seen(dtype, parts, scene):
    """Queries and weights in all of their parts are far inside what is allowed,
    with one part less far outside, in every scene that a kernel is held to."""
    sc = P.SCENES[scene](dtype)
    at = P.sample(sc, 60)
    ref = P.exact(sc, at)
    allowed = P.allowed(sc, at, ref)
    off = lambda q, w: P.rms(P.in_parts(sc, at, dtype, q, w) - ref)
    assert off(parts, parts) <= allowed / 4
    assert off(parts - 1, parts) >= 3 * allowed and off(parts, parts - 1) >= 3 * allowed
