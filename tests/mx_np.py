"""MXFP4 pages in numpy: blocks of 32 elements of 4 bits under a power-of-two scale byte."""
import copy

import numpy as np

from paged_np import Scene

UNITS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_bytes(x):
    """Of blocks [..., 32]: the exponent of the largest element less 2, one more from a mantissa of 1.75 on; 255 with an
    infinity or NaN."""
    amax = np.abs(np.asarray(x, np.float32)).max(-1).astype(np.float64)
    odd = ~np.isfinite(x).all(-1)
    mantissa, exponent = np.frexp(np.where(odd | (amax == 0), 1.0, amax))      # amax = mantissa 2^exponent, 1/2 <= mantissa < 1
    e = exponent - 1 + (mantissa >= 0.875) + 127 - 2
    return np.where(odd, 255, np.where(amax < 2.0 ** -126, 2, np.clip(e, 2, 252))).astype(np.uint8)


def codes_of(x, scales):
    """Nearest codes [..., 32], ties to even codes; by distances, in 64 bits."""
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.asarray(x, np.float64) * 2.0 ** (127 - scales.astype(np.float64))[..., None]
        d = np.abs(np.minimum(np.abs(y), 6.0)[..., None] - UNITS)
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])          # of two codes as near, the even one
    code = order[np.argmin(d[..., order], -1)]
    return (code + 8 * np.signbit(y)).astype(np.uint8)


def values_of(codes, scales):
    v = UNITS[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    v = v * 2.0 ** (scales.astype(np.float64) - 127)[..., None]
    return np.where(scales[..., None] == 255, np.nan, v).astype(np.float32)


def rounded(x):
    """What MXFP4 holds of x [..., hd]."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    e = scale_bytes(b)
    return values_of(codes_of(b, e), e).reshape(x.shape)


def packed(x):
    """Pages [pages][kv_heads][page][hd] -> bytes [pages][kv_heads][page][17 hd / 32], codes of all slots first."""
    n, kvh, page, hd = x.shape
    b = np.asarray(x, np.float32).reshape(n, kvh, page, hd // 32, 32)
    e = scale_bytes(b)
    c = codes_of(b, e).reshape(n, kvh, page * hd // 2, 2)
    out = np.concatenate([c[..., 0] | c[..., 1] << 4, e.reshape(n, kvh, -1)], -1)
    return np.ascontiguousarray(out.reshape(n, kvh, page, 17 * hd // 32))


def unpacked(raw):
    """The f32 values that such bytes stand for."""
    n, kvh, page, w = raw.shape
    hd = w // 17 * 32
    flat = raw.reshape(n, kvh, -1)
    c = flat[..., :page * hd // 2]
    c = np.stack([c & 15, c >> 4], -1).reshape(n, kvh, page, hd // 32, 32)
    e = flat[..., page * hd // 2:].reshape(n, kvh, page, hd // 32)
    return values_of(c, e).reshape(n, kvh, page, hd)


class MxScene(Scene):
    """A Scene over MXFP4 pages (k32, v32: the values they stand for); slots that nothing holds are NaN blocks."""

    def __init__(self, rows, lens, heads, kvh, hd, page, spread=0.0, **kw):
        super().__init__(rows, lens, heads, kvh, hd, page, "mxfp4", **kw)
        if spread:       # blocks of unlike size
            for x in (self.k32, self.v32):
                x *= np.exp(spread * self.rng.standard_normal(x.shape[:3] + (hd // 32,))).repeat(32, -1).astype(np.float32)
        self.settle()

    def settle(self):
        """Rounds what the pools hold (after a test has changed it)."""
        self.k32, self.v32 = rounded(self.k32), rounded(self.v32)

    def pools(self):
        return [packed(self.k32), packed(self.v32)]

    def plain(self):
        """The same over f32 pages of the same values."""
        sc = copy.copy(self)
        sc.__class__, sc.dtype = Scene, "f32"
        return sc

    def attention(self):
        return self.plain().attention()
