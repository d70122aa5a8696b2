"""The yardsticks of the paged attention's and the scoring's precision tests
see the mistakes that they are for (numpy only)."""
import numpy as np
import pytest

import precision_np as P
from paged_np import logprobs


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


@pytest.mark.parametrize("vocab", [7, 8195, 16387, 49157])
def test_a_lost_or_doubled_logit_is_seen(vocab):
    """A log Z without one logit, or with one twice, is outside the bound."""
    x, who = P.edge_rows(1, vocab)
    x = x.astype(np.float64)
    lp, ent, _, _ = logprobs(x, who, 1)
    bound, ebound = P.logprob_bounds(x, lp[:, None])
    m = x.max(1)
    p = np.exp(x[np.arange(len(x)), who] - m)
    z = np.exp(x - m[:, None]).sum(1)
    for weight in (0.0, 2.0):
        off = np.log(z + (weight - 1.0) * p) - np.log(z)
        assert (np.abs(off) > 1000 * bound[:, 0]).all()


def test_the_end_of_a_random_row_is_seen():
    """The last 7 of 128256 logits."""
    x = np.random.default_rng(0).standard_normal((4, 128256)).astype(np.float32).astype(np.float64)
    tokens = np.arange(4)
    lp = logprobs(x, tokens, 1)[0]
    short = logprobs(x[:, :-7], tokens, 1)[0]
    assert (np.abs(short - lp) > P.logprob_bounds(x, lp[:, None])[0][:, 0]).all()
