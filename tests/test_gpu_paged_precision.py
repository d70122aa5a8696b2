"""How exact yl_paged_attention's weights and references are, in both kernels
(160 heads of their own kv head put a prompt on the tile kernel)."""
import numpy as np
import pytest

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
