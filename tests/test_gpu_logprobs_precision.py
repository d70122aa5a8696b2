"""How exact yl_token_logprobs is, against 64-bit numpy."""
import numpy as np
import pytest

from paged_np import U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [40, 16384, 20000, 40000])
@pytest.mark.parametrize("other", ["near", "far"])
def test_exponentials_of_far_logits(gpu, vocab, other):
    """Two tokens that count, whose logits differ by an exact d: 1 - p of the
    first is e^d / (1 + e^d), however far d is.

    Relative bound: exp2 is right to an ulp (2 U), its argument's rounding is taken
    back but for log(2)'s own rounding (0.05 U |d|), one rounding of the product
    and one where stretches are joined (the same again where the two lie on
    different stretches); log1p has 2 ulp (4 U).  2 (3 + 0.05 |d|) + 4; the entropy
    adds a product, a sum, a quotient and a difference: 4 more."""
    from yallma3_mini_inference_amd import ops
    d = -np.arange(0.75, 80.0, 0.71875).astype(np.float32)
    x = np.full((len(d), vocab), -np.inf, np.float32)
    at = 5 if other == "near" else vocab - 1
    x[:, 3] = 2.0
    x[:, at] = 2.0 + d
    assert (x[:, at].astype(np.float64) - 2.0 == d).all()
    lp, ent, ids, tlp = ops.token_logprobs(x, np.full(len(d), 3), 2)
    e = np.exp(d.astype(np.float64))
    ref, rent = -np.log1p(e), np.log1p(e) - d * e / (1 + e)
    bound = (10 + 0.1 * np.abs(d)) * U
    err, eent = np.abs(lp / ref - 1), np.abs(ent / rent - 1)
    assert (err <= bound).all(), f"{(err / U).max():.1f} U"
    assert (eent <= bound + 4 * U).all(), f"{(eent / U).max():.1f} U"
    assert np.array_equal(tlp[:, 0], lp) and (ids[:, 0] == 3).all() and (ids[:, 1] == at).all()
