"""How exact yl_token_logprobs is, against 64-bit numpy."""
import numpy as np
import pytest

from paged_np import U, bf16_bits, logprobs, widened
from precision_np import edge_rows, logprob_bounds

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


def _check(x, tokens, top, dtype):
    from yallma3_mini_inference_amd import ops
    y = x.astype(np.float32) if dtype == "f32" else x.astype(np.float16) if dtype == "f16" else bf16_bits(x)
    w = widened(y)
    lp, ent, ids, tlp = ops.token_logprobs(y, tokens, top)
    rlp, rent, rids, rtlp = logprobs(w, tokens, top)
    assert np.array_equal(ids, rids)
    both, rboth = np.concatenate([lp[:, None], tlp], 1), np.concatenate([rlp[:, None], rtlp], 1)
    bl, be = logprob_bounds(w, rboth)
    assert (np.abs(both - rboth) <= bl).all(), f"{(np.abs(both - rboth) / bl).max():.3g} of the bound"
    assert (np.abs(ent - rent) <= be).all(), f"{(np.abs(ent - rent) / be).max():.3g} of the bound"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 65, 257, 4097, 8192, 8193, 16384, 16385, 49152, 128256])
@pytest.mark.parametrize("size", [0.5, 3.0, 9.0])
def test_random_rows(gpu, dtype, vocab, size):
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((4, vocab)) * size).astype(np.float32)
    _check(x, rng.integers(0, vocab, 4), min(5, vocab), dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("vocab", [7, 1000, 8191, 8195, 16384, 16387, 24583, 49157, 128256])
def test_no_logit_is_left_out_or_counted_twice(gpu, dtype, rows, vocab):
    """A row for each of the last 7 ids, and for the ids on both sides of the
    places where a thread's, a wavefront's or a stretch's share ends: that id
    and one other hold all of the weight, so a log Z without it (or with it
    twice) is off by 0.3 or more.  Few rows and many: both stretch lengths."""
    x, who = edge_rows(rows, vocab)
    if rows == 1:
        for r in range(0, len(x), 9):
            _check(x[r:r + 1], who[r:r + 1], min(2, vocab), dtype)
    _check(x, who, min(2, vocab), dtype)


@pytest.mark.parametrize("vocab", [50, 16390])
def test_more_rows_than_a_grid_has(gpu, vocab):
    """Beyond 65535 rows a call is several launches: rows of one stretch and of two."""
    from yallma3_mini_inference_amd import ops
    rows, kinds = 65535 + 70, 7
    rng = np.random.default_rng(vocab)
    x = bf16_bits((rng.standard_normal((kinds, vocab)) * 3).astype(np.float32))
    tokens = rng.integers(0, vocab, rows)
    kind = np.arange(rows) % kinds
    lp, ent, ids, tlp = ops.token_logprobs(x[kind], tokens, 3)
    w = widened(x)
    _, rent, rids, rtlp = logprobs(w, None, 3)
    logp = w - w.max(1, keepdims=True)
    logp -= np.log(np.exp(logp).sum(1, keepdims=True))
    rlp = logp[kind, tokens]
    bl, be = logprob_bounds(w, rtlp)
    z = (bl - 4 * U * np.abs(rtlp))[:, 0]          # log Z's part of the bound
    assert (np.abs(lp - rlp) <= z[kind] + 4 * U * np.abs(rlp)).all()
    assert (np.abs(ent - rent[kind]) <= be[kind]).all()
    assert np.array_equal(ids, rids[kind]) and (np.abs(tlp - rtlp[kind]) <= bl[kind]).all()
