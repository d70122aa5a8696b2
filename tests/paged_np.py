"""Paged caches, their attention and the scoring of logits in numpy, in 64 bits."""
import numpy as np

U = 2.0 ** -24    # half a step of f32, relative to the value


def bf16_bits(x):
    """f32 -> bfloat16 bits, to nearest, ties to even (finite values)."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def to_cache(x, dtype):
    x = np.asarray(x, np.float32)
    return x if dtype == "f32" else x.astype(np.float16) if dtype == "f16" else bf16_bits(x)


def widened(a):
    """Cache values as f64."""
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if a.dtype == np.uint16 else a.astype(np.float64)


class Scene:
    """A pool of pages and a batch over it.  Every slot that no sequence holds is NaN."""

    def __init__(self, rows, lens, heads, kvh, hd, page, dtype, prefix=0, seed=0, spare=2, extra_entries=0, behind=0):
        self.rng = r = np.random.default_rng(seed)
        self.rows, self.lens, self.heads, self.kvh, self.hd, self.page = list(rows), list(lens), heads, kvh, hd, page
        self.dtype, self.prefix = dtype, prefix
        held = [max(0, n - prefix) for n in lens]
        need = [-(-n // page) for n in held]
        shared = -(-prefix // page)
        self.n_pages = sum(need) + shared + spare
        order = r.permutation(self.n_pages)
        self.prefix_pages = order[:shared].astype(np.int32)
        self.table = np.full((len(lens), max(need + [0]) + extra_entries), -1, np.int32)
        at = shared
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (self.n_pages, kvh, page, hd)
        self.k32, self.v32 = np.full(shape, np.nan, np.float32), np.full(shape, np.nan, np.float32)
        for pages, n in [(self.prefix_pages, prefix)] + [(self.table[i, :m], h) for i, (m, h) in enumerate(zip(need, held))]:
            for j in range(n):
                self.k32[pages[j // page], :, j % page] = r.standard_normal((kvh, hd), np.float32)
                self.v32[pages[j // page], :, j % page] = r.standard_normal((kvh, hd), np.float32)
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
        self.total = int(self.starts[-1]) + behind
        self.q = r.standard_normal((self.total, heads * hd), np.float32)
        self.scale = 1.0 / np.sqrt(hd)

    def pools(self):
        out = []
        for x in (self.k32, self.v32):
            with np.errstate(all="ignore"):
                y = to_cache(np.nan_to_num(x, nan=0.0, posinf=np.inf, neginf=-np.inf), self.dtype)
            # (NaN bits of the type: 0x7fc0 for bf16)
            y = y.copy()
            y[np.isnan(x)] = 0x7FC0 if self.dtype == "bf16" else np.nan
            out.append(y)
        return out

    def batch(self, ops, single=False, max_len=0):
        return ops.PagedBatch(self.table, np.array(self.lens, np.uint32), None if single else self.starts, self.prefix,
                             self.prefix_pages if self.prefix else None, max_len)

    def places(self, s, limit):
        """Pages and slots of the positions below `limit` that sequence s holds."""
        out = []
        for p in range(limit):
            i = p if p < self.prefix else p - self.prefix
            pages = self.prefix_pages if p < self.prefix else self.table[s]
            if i // self.page < len(pages) and 0 <= pages[i // self.page] < self.n_pages:
                out.append((pages[i // self.page], i % self.page))
        return out

    def attention(self):
        """(out, bound): 64-bit results and what f32 arithmetic may be off by.

        The bound, per row and head: a score is a sum of hd f32 products (error
        at most (hd + 4) U sum |q k| scale, the scaling of q included; where q
        or a weight is held as two or three narrower parts, their omitted rest
        is below 2^-21 of the largest, 8 U, for each of the hd terms: counted
        as 8 U hd max|q| max|k| scale).  A weight's relative error is that, its
        own rounding, exp2's (2 U) and the rescalings' (8 U).  The result is a
        quotient of two sums over n weights, whose relative errors add up to at
        most twice (the weights' error + n U), times the largest |v|."""
        k, v = (widened(x) for x in self.pools())
        out = np.zeros((self.total, self.heads, self.hd))
        bound = np.zeros_like(out)
        for s, n in enumerate(self.lens):
            for r in range(self.starts[s], self.starts[s + 1]):
                limit = n - (int(self.starts[s + 1]) - r) + 1
                at = self.places(s, max(0, limit))
                if not at:
                    continue
                pg, sl = np.array(at).T
                for h in range(self.heads):
                    g = h // (self.heads // self.kvh)
                    kk, vv = k[pg, g, sl], v[pg, g, sl]
                    qq = self.q[r, h * self.hd:(h + 1) * self.hd].astype(np.float64)
                    with np.errstate(invalid="ignore"):
                        sc = kk @ qq * self.scale
                    e = np.exp(sc - sc.max())
                    out[r, h] = e @ vv / e.sum()
                    ds = ((self.hd + 4) * U * (np.abs(kk) @ np.abs(qq)).max()
                          + 8 * U * self.hd * np.abs(qq).max() * np.abs(kk).max()) * abs(self.scale)
                    bound[r, h] = 2 * (ds + 12 * U + len(at) * U) * np.abs(vv).max()
        return out.reshape(self.total, -1), bound.reshape(self.total, -1)


def rotated(x, cos, sin, pos, pairs, n, hd):
    """Rows of n heads turned to their positions, in f64 from the f32 tables."""
    x = x.astype(np.float64).reshape(len(x), n, hd)
    if pairs == "none":
        return x
    c, s = cos[pos].astype(np.float64)[:, None], sin[pos].astype(np.float64)[:, None]
    out = np.empty_like(x)
    lo, hi = (slice(0, None, 2), slice(1, None, 2)) if pairs == "adjacent" else (slice(0, hd // 2), slice(hd // 2, None))
    out[..., lo] = x[..., lo] * c - x[..., hi] * s
    out[..., hi] = x[..., lo] * s + x[..., hi] * c
    return out


def logprobs(x, tokens, top):
    """(logprob, entropy, ids, top logprobs) of f64 rows without NaN or +inf."""
    rows, vocab = x.shape
    lp, ent = np.full(rows, -np.inf), np.zeros(rows)
    ids, tlp = np.zeros((rows, top), np.uint32), np.full((rows, top), -np.inf)
    for r in range(rows):
        ids[r] = np.lexsort((np.arange(vocab), -x[r]))[:top]
        m = x[r].max()
        if m == -np.inf:
            continue
        lz = np.log(np.exp(x[r] - m).sum())
        logp = (x[r] - m) - lz
        p = np.exp(logp)
        ent[r] = -(p[p > 0] * logp[p > 0]).sum()
        if tokens is not None and tokens[r] < vocab:
            lp[r] = logp[tokens[r]]
        tlp[r] = logp[ids[r]]
    return lp, ent, ids, tlp
