"""What f32 evaluations of attention and of log probabilities are off by, in
numpy: yardsticks that are tight enough to miss a lost part of a number, or a
lost logit."""
import numpy as np

from paged_np import Scene, U, widened

# name -> scene of a cache type: decoded rows, long contexts, prompts
# of the row kernel and of the tile kernel (160 workgroups of 128 stacked rows),
# prefixes of both (the tile kernel's from 2^23 stacked rows times positions on)
SCENES = {
    "decode_64": lambda d: Scene([1] * 6, [33, 64, 127, 200, 257, 600], 32, 8, 64, 16, d, seed=1),
    "decode_128": lambda d: Scene([1] * 6, [33, 64, 127, 200, 257, 600], 8, 1, 128, 16, d, seed=1),
    "long_64": lambda d: Scene([1, 1, 1, 2], [3001, 40, 1777, 2050], 4, 1, 64, 64, d, seed=2),
    "long_128": lambda d: Scene([1, 1, 1, 2], [3001, 40, 1777, 2050], 4, 1, 128, 64, d, seed=2),
    "prompt_32": lambda d: Scene([70, 3], [90, 300], 8, 2, 32, 16, d, seed=3),
    "short": lambda d: Scene([16], [16], 8, 2, 64, 16, d, seed=3),
    "prefix_64": lambda d: Scene([1, 5, 1, 2, 40, 1, 3], [334, 342, 383, 333, 393, 330, 334], 8, 2, 64, 16, d, prefix=333, seed=4),
    "tile_32": lambda d: Scene([40, 0, 33, 70], [40, 7, 130, 75], 160, 160, 32, 16, d, seed=5),
    "tile_64": lambda d: Scene([40, 0, 33, 70], [40, 7, 530, 75], 160, 160, 64, 16, d, seed=5),
    "tile_128": lambda d: Scene([40, 0, 33, 70], [77, 44, 167, 112], 160, 160, 128, 16, d, prefix=37, seed=5),
    "tile_prefix_64": lambda d: Scene([1] * 35 + [9], [1011 + 7 * i for i in range(36)], 192, 32, 64, 32, d, prefix=1010, seed=6),
    "tile_prefix_128": lambda d: Scene([1] * 35 + [9], [1011 + 7 * i for i in range(36)], 192, 32, 128, 32, d, prefix=1010, seed=6),
}


def _of(sc, row, head):
    """q, keys and values (f64) of a row and head of the scene."""
    s = int(np.searchsorted(sc.starts, row, side="right")) - 1
    k, v = sc._widened
    pg, sl = np.array(sc.places(s, sc.lens[s] - (int(sc.starts[s + 1]) - row) + 1)).T
    g = head // (sc.heads // sc.kvh)
    return sc.q[row, head * sc.hd:(head + 1) * sc.hd].astype(np.float64), k[pg, g, sl], v[pg, g, sl]


def sample(sc, count, seed=0):
    """Up to `count` (row, head) that attend to something, from all of the batch."""
    sc._widened = tuple(widened(x) for x in sc.pools())
    rng = np.random.default_rng(seed)
    rows = [r for s, n in enumerate(sc.lens) for r in range(sc.starts[s], sc.starts[s + 1])
            if sc.places(s, max(0, n - (int(sc.starts[s + 1]) - r) + 1))]
    return [(int(rng.choice(rows)), int(rng.integers(sc.heads))) for _ in range(count)]


def exact(sc, at):
    out = []
    for q, k, v in (_of(sc, *a) for a in at):
        s = k @ q * float(sc.scale)
        e = np.exp(s - s.max())
        out.append(e @ v / e.sum())
    return np.array(out)


def serial_f32(sc, at):
    """The plain loop in f32: every product and every sum rounded, one after another."""
    out = []
    f = np.float32
    for q, k, v in (_of(sc, *a) for a in at):
        q, k, v = q.astype(f), k.astype(f), v.astype(f)
        s = np.cumsum(q * k, axis=1, dtype=f)[:, -1] * f(sc.scale)
        e = np.exp(s - s.max())
        out.append(np.cumsum(e[:, None] * v, axis=0, dtype=f)[-1] / np.cumsum(e, dtype=f)[-1])
    return np.array(out, np.float64)


def cut(x, dtype, parts):
    """f64 values as the sum of `parts` values of f16 (rounded, the largest of
    the array brought to 2^13) or bf16 (cut off)."""
    left, got = x.copy(), np.zeros_like(x)
    unit = 2.0 ** (13 - np.floor(np.log2(np.abs(x).max())))
    for _ in range(parts):
        if dtype == "f16":
            p = (left * unit).astype(np.float16).astype(np.float64) / unit
        else:
            p = (left.astype(np.float32).view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32).astype(np.float64)
        got, left = got + p, left - p
    return got


def in_parts(sc, at, dtype, q_parts, weight_parts):
    """64-bit sums of queries and weights that are held in so many parts."""
    out = []
    for q, k, v in (_of(sc, *a) for a in at):
        s = k @ cut(q * float(sc.scale), dtype, q_parts)
        e = np.exp(s - s.max())
        out.append(cut(e, dtype, weight_parts) @ v / cut(e, dtype, weight_parts).sum())
    return np.array(out)


def rms(x):
    return float(np.sqrt(np.mean(np.square(x))))


def allowed(sc, at, ref):
    """RMS error that a kernel may have: twice the serial loop's, which rounds
    more sums than any kernel here, and 2 U of the results for the parts (U / 2
    rms each at most) and the quotient."""
    return 2 * rms(serial_f32(sc, at) - ref) + 2 * U * rms(ref)


def logprob_bounds(x, lp):
    """Bounds of log probabilities and entropies of f64 rows.

    A weight is off by the rounding of d = x - m (U |d|), its exponential
    (exp2 to an ulp, the product's rounding, 0.05 U |d|) and that of its
    stretch where it is joined (again).  Sums: a thread adds up to 32 terms, a wavefront its threads in 6 steps, a workgroup its 8
    wavefronts, the join up to one stretch per thread of 256 (these vocabularies) and
    8 steps: 55 roundings.  With E1 = sum p |d| and E2 = sum p d^2, log Z is off
    by U (61 + 2.1 E1), sum d e / Z by U (61 E1 + 2.1 E2) and |sum d e / Z| = E1
    times Z's; the logarithm and the differences add 4 U times their sizes."""
    m = x.max(1, keepdims=True)
    d = np.where(np.isneginf(x), -1e4, x - m)
    p = np.exp(d)
    p /= p.sum(1, keepdims=True)
    e1, e2 = (p * -d).sum(1), (p * d * d).sum(1)
    z = U * (61 + 2.1 * e1)
    return z[:, None] + 4 * U * np.abs(lp), z + U * (61 * e1 + 2.1 * e2) + e1 * z + 4 * U * (e1 + np.log(1 / p.max(1)))


def edge_rows(rows, vocab):
    """(logits, ids): a row for each of the last 7 ids and of those beside the
    ends of threads', wavefronts' and stretches' shares, at least `rows` of them;
    that id and one other hold all of the weight."""
    edges = {e for n in (1, 4, 8, 64, 512, 2048, 4096, 8192, 16384, 32768, 65536, 122880, vocab) for e in range(n - 7, n + 8)}
    ids = np.array(sorted(i for i in edges if 0 <= i < vocab))
    who = np.resize(ids, max(rows, len(ids)))
    x = np.full((len(who), vocab), -40.0, np.float32)
    x[np.arange(len(x)), (who + vocab // 2 + 1) % vocab] = 0.0
    x[np.arange(len(x)), who] = 0.5
    return x, who
