"""How exact yl_paged_attention's weights and references are, in both kernels
(160 heads of their own kv head put a prompt on the tile kernel)."""
import numpy as np
import pytest

import precision_np as P
from paged_np import Scene, U, widened

pytestmark = pytest.mark.gpu

ROWS, TILE = (1, 4, 1), (40, 160, 160)       # rows of the sequence, heads, kv heads


def _attend(sc):
    from yallma3_mini_inference_amd import ops
    k, v = sc.pools()
    return ops.paged_attention(k, v, sc.batch(ops), sc.q, sc.heads, sc.scale)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout,hd,prefix", [(ROWS, 64, 0), (ROWS, 64, 300), (TILE, 32, 0), (TILE, 128, 0)])
@pytest.mark.parametrize("power", [20, 24, 28, 40, 80])
def test_scores_far_from_zero(gpu, dtype, layout, hd, prefix, power):
    """Scores of 2^power and more: the one that is largest by more than scores
    are rounded takes all of the weight.

    A score is off by at most (hd + 4) U sum |q k| scale: where the largest one
    leads by four times that, which at these sizes is also more than the 110
    powers of two that an f32 weight reaches, the result is its value but for the roundings
    of the weight's parts, the sum and the quotient, 4 U."""
    rows, heads, kvh = layout
    n = 650
    sc = Scene([rows, 1], [n, prefix + 1], heads, kvh, hd, 16, dtype, prefix=prefix, seed=power)
    sc.q *= np.float32(2.0 ** power)
    out = _attend(sc).reshape(sc.total, heads, hd)
    assert np.isfinite(out).all()
    k, v = (widened(x) for x in sc.pools())
    looked_at = 0
    for s in range(2):
        for r in range(sc.starts[s], sc.starts[s + 1]):
            pg, sl = np.array(sc.places(s, sc.lens[s] - (int(sc.starts[s + 1]) - r) + 1)).T
            for h in range(0, heads, max(1, heads // 8)):
                kk, vv = k[pg, h // (heads // kvh), sl], v[pg, h // (heads // kvh), sl]
                q = sc.q[r, h * hd:(h + 1) * hd].astype(np.float64)
                score = kk @ q * sc.scale
                off = 4 * (hd + 4) * U * (np.abs(kk) @ np.abs(q)).max() * sc.scale
                first = int(score.argmax())
                if len(score) > 1 and np.partition(score, -2)[-2] > score[first] - max(off, 80.0):
                    continue
                looked_at += 1
                assert (np.abs(out[r, h] - vv[first]) <= 4 * U * np.abs(vv[first])).all(), (r, h)
    assert looked_at >= 5


def _sink(dtype, rows, heads, kvh, hd, n, at, gap, prefix=0):
    """Position `at` has e^(gap ln 2) times every other position's weight and values of 0."""
    sc = Scene([rows], [n], heads, kvh, hd, 16, dtype, prefix=prefix, seed=int(gap))
    sc.scale = 0.125
    held = ~np.isnan(sc.k32[:, :, :, :1])
    sc.k32 = np.where(held, np.float32(0.0), np.float32(np.nan)) + np.zeros_like(sc.k32)
    sc.v32 = np.where(held, sc.rng.uniform(0.5, 1.5, sc.v32.shape).astype(np.float32), np.float32(np.nan))
    page, slot = sc.places(0, n)[at]
    sc.k32[page, :, slot, 0] = 8.0
    sc.v32[page, :, slot] = 0.0
    sc.q = np.zeros_like(sc.q)
    sc.q[:, ::hd] = gap * np.log(2.0)        # times 8, times the scale
    return sc


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout,hd,n,prefix", [(ROWS, 64, 3000, 0), (ROWS, 128, 3000, 1500), (TILE, 32, 1500, 0), (TILE, 64, 700, 0)])
@pytest.mark.parametrize("gap", [13.9, 21.3, 24.4, 31.0, 36.0])
def test_small_weights_beside_a_large_one(gpu, dtype, layout, hd, n, prefix, gap):
    """One position takes nearly all of the weight and adds nothing (its values
    are 0): the result is made of weights of 2^-gap.

    Bound, relative to the result: the exponent gap is rounded as the scale,
    the scale times log2(e), the product and the difference (4 U gap ln 2 <=
    3 U gap), exp2 (2 U), the parts of a weight (2 U, 2^-23), and the sums of equal
    terms, up to n / 64 of them in a row and 64 in a product; twice for the
    quotient.  Beside it, the positions of the large one's own step (at most 64)
    may be off by 2^-36 of it each."""
    rows, heads, kvh = layout
    for at in (0, n // 2 + 3):
        sc = _sink(dtype, rows, heads, kvh, hd, n, at, gap, prefix)
        ref, _ = sc.attention()
        assert 0 < ref.max() < 2 * n * 2.0 ** -gap
        err = np.abs(_attend(sc) - ref)
        bound = 2 * (3 * gap + 4 + n / 64 + 64) * U * ref + 64 * 2.0 ** -36 * 1.5
        assert (err <= bound).all(), f"sink at {at}: off by {np.max(err / ref):.3g} of the result, {np.max(err / bound):.3g} of the bound"


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout,hd", [((16, 2, 1), 32), ((16, 2, 1), 64), ((16, 2, 1), 128), (TILE, 64)])
def test_small_elements_of_a_query(gpu, dtype, layout, hd):
    """Equal elements of q some 2^-24 of its largest decide between two
    positions, whose keys are 2^14 and -2^14 there (and 0 at the largest element,
    which keeps every other position out).

    An element may be off by 2^-38 of the largest, 1.5, and by U of itself, all
    of a row to the same side; a score by that times hd 2^14 and by its sum's
    roundings, (hd + 8) U of its size; the result by a quarter of the two
    scores' errors times the values' difference, and 14 U of the values."""
    rows, heads, kvh = layout
    sc = Scene([rows], [rows + 2], heads, kvh, hd, 16, dtype, seed=hd)
    sc.scale = 1.0
    small = (np.linspace(0.6, 1.7, sc.total * heads) * 2.0 ** -24).astype(np.float32).reshape(sc.total, heads)
    q = np.repeat(small[..., None], hd, 2)
    q[..., 0] = 1.5
    sc.q = q.reshape(sc.total, heads * hd)
    sc.k32[..., 1:] = 0.0
    sc.k32[..., 0] = -1024.0
    (pa, sa), (pb, sb) = sc.places(0, 2)
    for page, slot, key in ((pa, sa, 2.0 ** 14), (pb, sb, -2.0 ** 14)):
        sc.k32[page, :, slot] = key
        sc.k32[page, :, slot, 0] = 0.0
    ref, _ = sc.attention()
    v = np.nan_to_num(widened(sc.pools()[1]))
    va, vb = (np.repeat(v[page, :, slot], heads // kvh, 0)[None] for page, slot in ((pa, sa), (pb, sb)))
    score = hd * 2.0 ** 14 * (2.0 ** -38 * 1.5 + (hd + 9) * U * small.astype(np.float64))[..., None]
    bound = 0.5 * score * np.abs(va - vb) + 14 * U * np.maximum(np.abs(va), np.abs(vb))
    err = np.abs(_attend(sc) - ref).reshape(sc.total, heads, hd)
    assert (err <= bound).all(), f"off by {err.max():.3g}, {(err / bound).max():.3g} of the bound"


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("scene", list(P.SCENES))
def test_no_less_exact_than_f32_loops(gpu, dtype, scene):
    """The RMS error over rows and heads is that of an f32 evaluation: a lost
    part of the queries or weights is 5 times that and more (test_paged_bounds.py)."""
    sc = P.SCENES[scene](dtype)
    at = P.sample(sc, 150)
    ref = P.exact(sc, at)
    out = _attend(sc).reshape(sc.total, sc.heads, sc.hd)
    err = P.rms(np.array([out[a] for a in at]) - ref)
    assert err <= P.allowed(sc, at, ref), f"{err / P.allowed(sc, at, ref):.3g} of what is allowed"


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("layout", [ROWS, (40, 8, 2), TILE])
@pytest.mark.parametrize("size", [2.0, 5.0, 12.0])
def test_scores_far_apart(gpu, dtype, layout, size):
    """Scores of a deviation of 2 to 12: what the weights are taken against rises
    and falls from step to step; the RMS error stays that of an f32 evaluation."""
    rows, heads, kvh = layout
    sc = Scene([rows, 1], [640, 900], heads, kvh, 64, 16, dtype, seed=int(size))
    sc.q *= np.float32(size)
    for at in (5, 130, 131, 400):            # and single positions far above the others
        page, slot = sc.places(0, 600)[at]
        sc.k32[page, :, slot] *= 2.5
    at = P.sample(sc, 150)
    ref = P.exact(sc, at)
    out = _attend(sc).reshape(sc.total, sc.heads, sc.hd)
    err = P.rms(np.array([out[a] for a in at]) - ref)
    assert err <= P.allowed(sc, at, ref), f"{err / P.allowed(sc, at, ref):.3g} of what is allowed"
