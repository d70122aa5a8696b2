"""yl_token_logprobs against 64-bit numpy.

Bound: with m the row's maximum, a log probability is (x - m) - log Z.  x - m
is rounded once (U |x - m|); each weight is off by its argument's rounding and
exp's error (U |x - m| + 4 U, of which the weights beyond exp(-30) do not
matter: 34 U relative), Z's sum of positive terms by at most that and, in
partial sums of at most 4096 terms a lane and a tree, 4096 U: relative to Z,
so absolute in log Z; the logarithm and the last difference add 4 U times
their sizes.  The entropy log Z - sum d e / Z has the same errors, weighted by
|d| <= 30 where it counts.  In all at most 4200 U (1 + 30) plus 4 U |result|;
the sums' errors are random in sign, and 1 / 16 of it is asked for."""
import numpy as np
import pytest

from hip_rt import Graph, Stream, buffer, bytes_of, filled
from paged_np import U, bf16_bits, logprobs, widened

pytestmark = pytest.mark.gpu


def _as(x, dtype):
    return x.astype(np.float32) if dtype == "f32" else x.astype(np.float16) if dtype == "f16" else bf16_bits(x)


def _close(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    fine = np.isfinite(b)
    assert np.array_equal(a[~fine], b[~fine])
    err = np.abs(a[fine] - b[fine])
    assert (err <= 4200 * U * 31 / 16 + 4 * U * np.abs(b[fine])).all(), err.max()


def _check(x, tokens, top, dtype):
    from yallma3_mini_inference_amd import ops
    y = _as(x, dtype)
    w = np.where(np.isneginf(x), -np.inf, widened(np.where(np.isneginf(x), np.zeros_like(y), y))) if dtype == "bf16" else y.astype(np.float64)
    if dtype == "bf16":
        y = np.where(np.isneginf(x), np.uint16(0xFF80), y)
    got = ops.token_logprobs(y, tokens, top)
    ref = logprobs(w, tokens, top)
    assert np.array_equal(got[2], ref[2])
    _close(got[1], ref[1])
    _close(got[3], ref[3])
    if tokens is not None:
        _close(got[0], ref[0])
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 64, 65, 257, 1000, 4097, 16384, 16385, 49152, 128256])
def test_rows(gpu, dtype, vocab):
    rng = np.random.default_rng(vocab)
    rows = 5
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    tokens = rng.integers(0, vocab, rows)
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(32, vocab)}):
        _check(x, tokens, top, dtype)


@pytest.mark.parametrize("rows", [1, 3, 64, 300, 1500])
def test_many_rows(gpu, rows):
    rng = np.random.default_rng(rows)
    x = (rng.standard_normal((rows, 700)) * 2).astype(np.float32)
    _check(x, rng.integers(0, 700, rows), 7, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(100, 50000, 9), (300, 17000, 3), (300, 10000, 32), (2, 300000, 32), (2, 300000, 5)])
def test_stretches_and_their_joining(gpu, dtype, rows, vocab, top):
    """Both stretch lengths, rows of one stretch and of several, and lists too many for one selection."""
    rng = np.random.default_rng(rows + vocab)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    _check(x, rng.integers(0, vocab, rows), top, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [50, 40000])
def test_equal_values_by_rising_id(gpu, dtype, vocab):
    rng = np.random.default_rng(1)
    x = np.zeros((6, vocab), np.float32)
    x[1] = -5.0
    x[2] = rng.integers(0, 3, vocab)
    x[3, vocab // 2:] = 1.0
    x[4, ::7] = -0.0                       # -0 and +0 are equal
    x[5] = np.arange(vocab) // 9
    _check(x, np.full(6, vocab - 1), 32, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [300, 40000])
def test_rising_and_falling_rows(gpu, dtype, vocab):
    """Orders in which every next value beats, or none beats, those before."""
    x = np.stack([np.linspace(-20, 20, vocab), np.linspace(20, -20, vocab)]).astype(np.float32)
    _check(x, np.array([0, 1]), 20, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [100, 33000])
def test_masked_logits(gpu, dtype, vocab):
    """-inf almost everywhere (a constrained choice), everywhere, nowhere but one; the lowest finite value."""
    x = np.full((5, vocab), -np.inf, np.float32)
    x[0, [3, 50, vocab - 1]] = [1.0, 2.0, 1.5]
    x[2, vocab - 2] = -7.0
    x[3, :] = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3e38}[dtype]
    x[4, :] = x[3, 0]
    x[4, 40] = 2.0
    got = _check(x, np.array([50, 3, vocab - 2, 5, 41]), 12, dtype)
    assert got[0][1] == -np.inf and got[1][1] == 0.0 and got[0][2] == 0.0 and got[1][2] == 0.0


@pytest.mark.parametrize("vocab", [100, 33000])
def test_nan_and_infinity(gpu, vocab):
    from yallma3_mini_inference_amd import ops
    x = np.random.default_rng(0).standard_normal((5, vocab)).astype(np.float32)
    x[0, 17] = np.nan
    x[1, 90] = np.inf
    x[2, [5, 60]] = np.inf
    x[3, :] = np.nan
    lp, ent, ids, tlp = ops.token_logprobs(x, np.array([1, 1, 5, 0, 2]), 4)
    assert np.isnan(lp[:4]).all() and np.isnan(ent[:4]).all() and np.isnan(tlp[:4]).all()
    assert np.isfinite(lp[4]) and np.isfinite(ent[4]) and np.isfinite(tlp[4]).all()
    z = x[0].copy()
    z[17] = -np.inf
    assert np.array_equal(ids[0], np.lexsort((np.arange(vocab), -z))[:4])     # NaN comes last
    assert ids[1][0] == 90 and list(ids[2][:2]) == [5, 60] and list(ids[3]) == [0, 1, 2, 3]


def test_ids_outside_the_vocabulary(gpu):
    from yallma3_mini_inference_amd import ops
    x = np.random.default_rng(0).standard_normal((3, 100)).astype(np.float32)
    lp = ops.token_logprobs(x, np.array([100, 0xFFFFFFFF, 99], np.uint32))[0]
    assert lp[0] == -np.inf and lp[1] == -np.inf and np.isfinite(lp[2])


def test_sharp_rows_keep_small_probabilities(gpu):
    """The most probable id of a sharp row: 1 - p down to 1e-7, in relative precision (U times a few, and the weights' 34 U)."""
    from yallma3_mini_inference_amd import ops
    gaps = np.array([5.0, 10.0, 16.0, 25.0], np.float32)
    x = np.zeros((4, 20000), np.float32)
    x[:] = -60.0
    x[:, 7] = 0.0
    x[:, 1234] = -gaps
    lp, ent, _, tlp = ops.token_logprobs(x, np.full(4, 7), 1)
    d = np.concatenate([-gaps[:, None].astype(np.float64), np.full((4, 19998), -60.0)], 1)
    e = np.exp(d)
    ref = -np.log1p(e.sum(1))
    assert (np.abs(lp - ref) <= 80 * U * np.abs(ref)).all() and np.array_equal(lp, tlp[:, 0])
    rent = np.log1p(e.sum(1)) - (d * e).sum(1) / (1 + e.sum(1))
    assert (np.abs(ent - rent) <= 80 * U * np.abs(rent)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ld,offset", [(1003, 0), (1007, 1), (1024, 3)])
def test_strides_and_alignment(gpu, dtype, ld, offset):
    """Rows at odd strides from an odd element; what lies between them (NaN) takes no part; each output on its own."""
    rows, vocab, top = 4, 1003, 6
    rng = np.random.default_rng(ld)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    y = _as(x, dtype)
    es = y.dtype.itemsize
    buf = np.full(rows * ld + offset, 0x7FC0 if dtype == "bf16" else np.nan, y.dtype)
    buf[offset:].reshape(rows, ld)[:, :vocab] = y
    tokens = rng.integers(0, vocab, rows).astype(np.uint32)
    d, dt = buffer(buf), buffer(tokens)
    L = gpu.lib()
    need = L.yl_token_logprobs_workspace(rows, vocab, top)
    space = bytes_of(need, 255)
    ref = logprobs(widened(y), tokens, top)
    for want in ("all", "logprob", "entropy", "top"):
        lp, ent = filled(rows + 1, 7.0), filled(rows + 1, 7.0)
        ids, tlp = filled(rows * top + 1, 7, np.uint32), filled(rows * top + 1, 7.0)
        w = lambda n, b: b.ptr if want in ("all", n) else None
        gpu.check(L.yl_token_logprobs(d.ptr + offset * es, gpu.DTYPES[dtype], rows, vocab, ld, w("logprob", dt), w("logprob", lp),
                                      w("entropy", ent), top if want in ("all", "top") else 0, w("top", ids), w("top", tlp),
                                      space.ptr, need, None))
        gpu.check(L.yl_synchronize())
        for name, got, r in (("logprob", lp, ref[0]), ("entropy", ent, ref[1]), ("top", ids, ref[2]), ("top", tlp, ref[3])):
            g = got.numpy()
            assert g[-1] == 7
            if want not in ("all", name):
                assert (g == 7).all()
            elif got is ids:
                assert np.array_equal(g[:-1].reshape(rows, top), r)
            else:
                _close(g[:-1].reshape(r.shape), r)


def test_graph_replays(gpu):
    """A captured call replayed over new logits, an eager call on another stream between."""
    rows, vocab, top = 3, 50000, 8
    L = gpu.lib()
    x, tokens = filled((rows, vocab), 0.0), filled(rows, 0, np.uint32)
    need = L.yl_token_logprobs_workspace(rows, vocab, top)

    def outputs():
        return [filled(rows, 0.0), filled(rows, 0.0), filled((rows, top), 0, np.uint32), filled((rows, top), 0.0), bytes_of(need, 255)]

    def call(o, stream):
        gpu.check(L.yl_token_logprobs(x.ptr, 0, rows, vocab, vocab, tokens.ptr, o[0].ptr, o[1].ptr, top, o[2].ptr, o[3].ptr, o[4].ptr,
                                      need, stream))
    a, b, side = outputs(), outputs(), Stream()
    graph = Graph(lambda stream: call(a, stream))
    rng = np.random.default_rng(3)
    for _ in range(4):
        h = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
        t = rng.integers(0, vocab, rows).astype(np.uint32)
        x.upload(h)
        tokens.upload(t)
        graph.replay()
        call(b, side.handle)
        gpu.check(L.yl_synchronize())
        ref = logprobs(h.astype(np.float64), t, top)
        assert np.array_equal(a[2].numpy(), ref[2])
        _close(a[0].numpy(), ref[0])
        assert all(np.array_equal(p.numpy(), q.numpy()) for p, q in zip(a[:4], b[:4]))


def test_rows_beyond_32_bits(gpu):
    """A row whose elements start past 2^31."""
    rows, vocab, ld, top = 3, 70000, 1 << 30, 2
    x = gpu.DeviceBuffer(2 * ((rows - 1) * ld + vocab))
    bits = bf16_bits(np.random.default_rng(2).standard_normal((rows, vocab)).astype(np.float32))
    L = gpu.lib()
    for r in range(rows):
        gpu.check(L.yl_memcpy_h2d(x.ptr + 2 * r * ld, bits[r].ctypes.data, 2 * vocab))
    tokens = buffer(np.array([0, 1, vocab - 1], np.uint32))
    lp, ids, tlp = filled(rows, 0.0), filled((rows, top), 0, np.uint32), filled((rows, top), 0.0)
    need = L.yl_token_logprobs_workspace(rows, vocab, top)
    space = bytes_of(need, 255)
    gpu.check(L.yl_token_logprobs(x.ptr, 2, rows, vocab, ld, tokens.ptr, lp.ptr, None, top, ids.ptr, tlp.ptr, space.ptr, need, None))
    gpu.check(L.yl_synchronize())
    ref = logprobs(widened(bits), [0, 1, vocab - 1], top)
    assert np.array_equal(ids.numpy(), ref[2])
    _close(lp.numpy(), ref[0])
    _close(tlp.numpy(), ref[3])
