"""MXFP4 pages: yl_paged_append's codes against numpy's, exactly; yl_paged_gather;
yl_paged_attention over such pages against 64-bit numpy of the values that they
stand for (bounds derived in paged_np.Scene.attention and precision_np)."""
import ctypes as C

import numpy as np
import pytest

import mx_np as X
import precision_np as P
from hip_rt import Graph, Stream, buffer, filled
from mx_np import MxScene
from paged_np import Scene, widened
from test_gpu_paged import LAYOUTS, Call, _check, _tables

pytestmark = pytest.mark.gpu


def _attend(sc, single=False, max_len=0):
    from yallma3_mini_inference_amd import ops
    return ops.paged_attention(*sc.pools(), sc.batch(ops, single, max_len), sc.q, sc.heads, sc.scale)


# ------------------------------------------------------------------ append


def _rotated32(x, cos, sin, pos, pairs, n, hd):
    """Each product and sum rounded to f32 on its own."""
    x = x.reshape(len(x), n, hd)
    if pairs == "none":
        return x
    c, s = cos[pos][:, None], sin[pos][:, None]
    out = np.empty_like(x)
    lo, hi = (slice(0, None, 2), slice(1, None, 2)) if pairs == "adjacent" else (slice(0, hd // 2), slice(hd // 2, None))
    out[..., lo] = x[..., lo] * c - x[..., hi] * s
    out[..., hi] = x[..., lo] * s + x[..., hi] * c
    return out


@pytest.mark.parametrize("pairs", ["none", "adjacent", "half"])
@pytest.mark.parametrize("heads,kvh,hd,page", [(4, 2, 32, 16), (9, 3, 64, 32), (8, 1, 128, 256), (2, 2, 64, 64), (5, 5, 32, 128), (32, 8, 128, 16)])
def test_append_and_gather(gpu, pairs, heads, kvh, hd, page):
    """Every touched block's bytes, and nothing else, are what numpy makes of the
    rows; gathering reads the values back and passes over what nothing holds."""
    from yallma3_mini_inference_amd import ops
    prefix = 20
    rows, lens = [1, 40, 0, 3, 1, 5, 2, 1], [90, 40, 7, 300, 1, 22, 21, 400]
    sc = MxScene(rows, lens, heads, kvh, hd, page, prefix=prefix, seed=hd)
    sc.table[3, (299 - prefix) // page] = sc.n_pages     # the last page of the fourth sequence is missing
    rope_rows = 350                                      # the last row lies beyond the tables
    cos, sin = _tables(hd, rope_rows) if pairs != "none" else (None, None)
    k, v = (sc.rng.standard_normal((sc.total, kvh * hd), np.float32) * np.float32(s) for s in (3.0, 1e-3))
    k[::3] *= np.exp(4 * sc.rng.standard_normal(k[::3].shape)).astype(np.float32)
    pk, pv = sc.pools()
    q2, k2, v2 = ops.paged_append(pk, pv, sc.batch(ops), sc.q, k, v, heads, pairs, cos, sin)
    want = [X.unpacked(x) for x in (pk, pv)]
    touched, held = np.zeros(want[0].shape[:3], bool), np.zeros(sc.total, bool)
    gk, gv = (np.full((sc.total, kvh, hd), 5.0, np.float32) for _ in range(2))
    for s, n in enumerate(lens):
        places = sc.places(s, n)
        for r in range(sc.starts[s], sc.starts[s + 1]):
            pos = n - (int(sc.starts[s + 1]) - r)
            if pos < 0 or (pairs != "none" and pos >= rope_rows):
                continue
            i = pos - prefix
            if i >= 0 and not 0 <= sc.table[s, i // page] < sc.n_pages:
                continue
            page_id, slot = (sc.table[s, i // page], i % page) if i >= 0 else (sc.prefix_pages[pos // page], pos % page)
            if i >= 0:
                at = np.array([pos])
                want[0][page_id, :, slot] = X.rounded(_rotated32(k[r:r + 1], cos, sin, at, pairs, kvh, hd)[0])
                want[1][page_id, :, slot] = X.rounded(v[r].reshape(kvh, hd))
                touched[page_id, :, slot] = True
            held[r] = True
            gk[r], gv[r] = want[0][page_id, :, slot], want[1][page_id, :, slot]
    assert touched.any() and not touched.all()
    for got, ref, before in ((k2, want[0], pk), (v2, want[1], pv)):
        assert np.array_equal(X.unpacked(got)[touched], ref[touched])
        # scale bytes, and bytes of the slots that no row has
        part = lambda raw: (raw.reshape(sc.n_pages, kvh, -1)[..., :page * hd // 2].reshape(sc.n_pages, kvh, page, -1),
                            raw.reshape(sc.n_pages, kvh, -1)[..., page * hd // 2:].reshape(sc.n_pages, kvh, page, -1))
        for a, b in zip(part(got), part(before)):
            assert np.array_equal(a[~touched], b[~touched])
        assert np.array_equal(part(got)[1], part(X.packed(ref))[1])
    if pairs == "none":
        rows_k, rows_v = ops.paged_gather(k2, v2, sc.batch(ops), sc.total, fill=5.0)
        assert not held.all()
        assert np.array_equal(rows_k.reshape(gk.shape), gk) and np.array_equal(rows_v.reshape(gv.shape), gv)


def test_append_extremes(gpu):
    """Ties, saturation, zeros, the ends of the scale's range, infinities and NaN, a block each."""
    from yallma3_mini_inference_amd import ops
    blocks = np.zeros((16, 32), np.float32)
    blocks[0, :12] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -5.0, 6.99]
    blocks[1, :6] = [7.0, 0.5, 1.5, 2.5, 3.5, -7.0]                      # the next unit
    blocks[2, :4] = [6.999999, 5.0, 4.999999, -6.999999]                 # 6.999999 -> 6
    blocks[3] = 0.0
    blocks[4, :3] = [-0.0, 0.0, 1e-45]
    blocks[5, :4] = [2.0 ** -126, 2.0 ** -127, -2.0 ** -125, 2.0 ** -124]
    blocks[6, :4] = [3.4028235e38, -3.4e38, 1e38, 1e30]                  # 6 * 2^125
    blocks[7, :3] = [1.75 * 2.0 ** 126, 2.0 ** 126, 1.0]
    blocks[8, 5] = np.inf
    blocks[9, 31] = -np.inf
    blocks[10, 0] = np.nan
    blocks[11, :3] = [np.nan, np.inf, 3.0]
    blocks[12] = np.linspace(-6, 6, 32)
    blocks[13] = 2.0 ** -60 * np.linspace(-7, 7, 32)
    blocks[14] = np.float32(2.0 ** 100) * np.linspace(-1, 1, 32)
    blocks[15, 7] = 1e-30
    x = blocks.reshape(4, 128)
    sc = MxScene([4], [9], 1, 1, 128, 16, seed=4)
    pk, pv = sc.pools()
    _, k2, v2 = ops.paged_append(pk, pv, sc.batch(ops), None, -x, x, 1)
    for got, want in ((X.unpacked(v2), X.rounded(x)), (X.unpacked(k2), X.rounded(-x))):
        got = got[sc.table[0, 0], 0, 5:9]
        assert np.array_equal(got, want, equal_nan=True)
        assert np.isnan(got.reshape(16, 32)[8:12]).all() and np.isfinite(np.delete(got.reshape(16, 32), range(8, 12), 0)).all()


def test_append_fused_rows_at_odd_strides(gpu):
    """q, k and v as parts of fused rows whose length and address are odd, on a stream; keys and values only."""
    sc = MxScene([1, 17], [40, 30], 6, 2, 64, 16, seed=5)
    heads, kvh, hd, ld = 6, 2, 64, (6 + 4) * 64 + 3
    x = sc.rng.standard_normal((sc.total, ld), np.float32)
    cos, sin = _tables(hd, 64)
    call, stream = Call(gpu, sc), Stream()
    dx, dc, ds = buffer(np.concatenate([[0], x.ravel()]).astype(np.float32)), buffer(cos), buffer(sin)
    at = dx.ptr + 4
    gpu.check(gpu.lib().yl_synchronize())
    gpu.check(gpu.lib().yl_paged_append(C.byref(call.cache), C.byref(call.batch), heads, None, 0, None, 0, at + 4 * heads * hd, ld,
                                        at + 4 * (heads + kvh) * hd, ld, 0, dc.ptr, ds.ptr, 64, stream.handle))
    out = [filled((sc.total + 1, kvh * hd + 3), 7.0) for _ in range(2)]
    gpu.check(gpu.lib().yl_paged_gather(C.byref(call.cache), C.byref(call.batch), out[0].ptr + 4, kvh * hd + 3, out[1].ptr + 4,
                                        kvh * hd + 3, stream.handle))
    stream.synchronize()
    pos = np.concatenate([np.arange(39, 40), np.arange(13, 30)])
    k = _rotated32(x[:, heads * hd:(heads + kvh) * hd], cos, sin, pos, "adjacent", kvh, hd)
    v = x[:, (heads + kvh) * hd:(heads + 2 * kvh) * hd].reshape(sc.total, kvh, hd)
    for got, want in zip(out, (k, v)):
        rows = got.numpy().ravel()[1:1 + sc.total * (kvh * hd + 3)].reshape(sc.total, -1)
        assert np.array_equal(rows[:, :kvh * hd], X.rounded(want).reshape(sc.total, -1)) and (rows[:, kvh * hd:] == 7.0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("prefix", [0, 21])
def test_gather_of_other_types(gpu, dtype, prefix):
    """Whole conversations, the shared prefix among them, out of pages of every type."""
    from yallma3_mini_inference_amd import ops
    rows = [prefix + 30, prefix + 1, 0, 5]
    sc = Scene(rows, [prefix + 30, prefix + 1, 9, prefix + 40], 2, 2, 32, 16, dtype, prefix=prefix, seed=3, behind=2)
    k, v = sc.pools()
    got = ops.paged_gather(k, v, sc.batch(ops), sc.total, fill=9.0)
    for g, pool in zip(got, (k, v)):
        for s, n in enumerate(sc.lens):
            at = sc.places(s, n)[n - rows[s]:]
            want = np.array([widened(pool)[p, :, i].ravel() for p, i in at]).reshape(rows[s], 64)
            assert np.array_equal(g[sc.starts[s]:sc.starts[s + 1]], want)
        assert (g[sc.starts[-1]:] == 9.0).all()


def test_gather_of_one_side(gpu):
    sc = MxScene([3], [20], 2, 2, 32, 16, seed=3)
    call, out = Call(gpu, sc), filled((3, 64), 7.0)
    gpu.check(gpu.lib().yl_paged_gather(C.byref(call.cache), C.byref(call.batch), None, 0, out.ptr, 64, None))
    gpu.check(gpu.lib().yl_synchronize())
    assert np.array_equal(out.numpy(), np.array([sc.v32[p, :, i].ravel() for p, i in sc.places(0, 20)[17:]]))


# --------------------------------------------------------------- attention


@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
def test_decode_rows(gpu, heads, kvh, hd):
    """One row per sequence, lengths around page and tile ends; blocks of unlike size."""
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 257]
    sc = MxScene([1] * len(lens), lens, heads, kvh, hd, 16, spread=1.0, seed=heads + hd)
    _check(sc, _attend(sc, single=True))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_ragged_rows(gpu, page, hd):
    rows, lens = [1, 70, 0, 5, 33, 1, 0, 130, 16], [300, 70, 12, 90, 34, 1, 0, 199, 16]
    sc = MxScene(rows, lens, 8, 2, hd, page, seed=page)
    _check(sc, _attend(sc))


@pytest.mark.parametrize("prefix", [1, 16, 37, 333])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 32), (8, 2, 64), (8, 1, 128)])
def test_shared_prefix(gpu, prefix, heads, kvh, hd):
    rows = [1, 5, 1, 2, 40, 1, 3]
    lens = [prefix + 1, prefix + 9, prefix + 50, prefix, prefix + 60, max(1, prefix - 3), prefix + 1]
    sc = MxScene(rows, lens, heads, kvh, hd, 16, prefix=prefix, seed=prefix)
    _check(sc, _attend(sc))


@pytest.mark.parametrize("heads,kvh,hd", [(160, 160, 32), (160, 160, 64), (160, 160, 128), (160, 80, 64)])
@pytest.mark.parametrize("prefix,page", [(0, 16), (37, 16), (0, 256)])
def test_many_prompt_rows(gpu, heads, kvh, hd, prefix, page):
    """Rows enough for the tile kernel (160 workgroups of 128 stacked rows)."""
    rows = [1, 40, 0, 33, 2, 70] if kvh == 160 else [1, 70, 0, 17, 2, 60]
    lens = [prefix + n for n in (90, 40, 7, 130, 20, 75)]
    lens[1] -= prefix // 2
    sc = MxScene(rows, lens, heads, kvh, hd, page, spread=1.0, prefix=prefix, seed=hd)
    _check(sc, _attend(sc))


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_long_prefix_under_a_batch(gpu, hd):
    """A prefix long enough, under rows enough, for the tile kernel (2^23 stacked rows times positions)."""
    prefix, seqs = 1010, 36
    sc = MxScene([1] * (seqs - 1) + [9], [prefix + 1 + 7 * i for i in range(seqs)], 192, 32, hd, 32, prefix=prefix, seed=hd)
    _check(sc, _attend(sc))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("max_len", [0, 100, 5000])
def test_long_contexts_in_chunks(gpu, hd, max_len):
    sc = MxScene([1, 1, 1, 2], [3001, 40, 1777, 2050], 4, 1, hd, 64, seed=hd)
    _check(sc, _attend(sc, max_len=max_len))


def test_positions_nobody_holds(gpu):
    rows, lens = [1, 30, 3, 2, 1, 4], [100, 150, 64, 1, 0, 40]
    sc = MxScene(rows, lens, 8, 2, 64, 16, seed=1, extra_entries=1)
    sc.table[0, 2] = -1
    sc.table[1, 0] = sc.n_pages
    sc.table[1, 5] = 0x7FFFFFFF
    sc.table[5, :] = -5
    sc.lens[2] = 16 * sc.table.shape[1] + 500
    ref = _check(sc, _attend(sc))
    assert not ref[sc.starts[5]:].any() and not ref[sc.starts[3]].any()


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("rows,heads,kvh", [([40, 1], 8, 2), ([50, 70, 3], 160, 160)])
def test_blocks_that_are_no_numbers(gpu, rows, heads, kvh, hd):
    """A later row's NaN key takes no part in the rows before it; a NaN block of a value spoils its 32 components
    in the rows that attend to it and no others (in both kernels)."""
    lens = [75, 20] if len(rows) == 2 else [75, 90, 30]
    sc = MxScene(rows, lens, heads, kvh, hd, 16, seed=5)
    first = 75 - rows[0]                                # position of the first row
    at = first + 20
    page, slot = sc.table[0, at // 16], at % 16
    sc.v32[page, :, slot, :32] = np.nan
    later = first + 30
    sc.k32[sc.table[0, later // 16], :, later % 16] = np.nan
    sc.settle()
    out = _attend(sc).reshape(sc.total, heads, hd)
    sc.v32[page, :, slot, :32] = 0.0
    sc.settle()
    ref, bound = (x.reshape(sc.total, heads, hd) for x in sc.attention())
    assert (np.abs(out[:20] - ref[:20]) <= bound[:20]).all()
    assert np.isnan(out[20:30][..., :32]).all() and np.isnan(out[30:rows[0]]).all()
    assert (np.abs(out[20:30] - ref[20:30])[..., 32:] <= bound[20:30][..., 32:]).all()
    assert (np.abs(out[rows[0]:] - ref[rows[0]:]) <= bound[rows[0]:]).all()


@pytest.mark.parametrize("power", [-60, -20, 20, 60])
@pytest.mark.parametrize("heads,kvh,rows", [(8, 2, 20), (160, 160, 40)])
def test_sizes_of_keys_and_values(gpu, power, heads, kvh, rows):
    """Blocks far from 1, with queries that bring the scores back."""
    sc = MxScene([1, rows], [200, 70], heads, kvh, 64, 16, seed=16)
    sc.k32 *= np.float32(2.0 ** power)
    sc.v32 *= np.float32(2.0 ** (power - 3))
    sc.q *= np.float32(2.0 ** -power)
    sc.settle()
    _check(sc, _attend(sc))


@pytest.mark.parametrize("prefix", [0, 50])
def test_strides_alignment_and_rows_behind(gpu, prefix):
    sc = MxScene([1, 20, 0, 3], [prefix + 50, prefix + 20, prefix + 5, prefix + 300], 4, 2, 64, 16, prefix=prefix, seed=9, behind=3)
    call = Call(gpu, sc, q_ld=4 * 64 + 5, out_ld=4 * 64 + 3, offset=1)
    call()
    out, between = call.result()
    n = int(sc.starts[-1])
    ref, bound = sc.attention()
    assert (np.abs(out[:n] - ref[:n]) <= bound[:n]).all()
    assert (out[n:] == 7.0).all() and (between == 7.0).all() and call.out.numpy()[0] == 7.0


@pytest.mark.parametrize("prefix", [0, 70])
def test_graph_replays_read_new_lengths(gpu, prefix):
    """A captured call, replayed with other lengths and queries, an eager call between the replays."""
    lens = [[prefix + 30, prefix + 500, prefix + 1], [prefix + 33, prefix + 511, prefix + 64], [prefix + 60, prefix + 9, prefix + 900]]
    sc = MxScene([1, 1, 1], [prefix + 920] * 3, 8, 2, 64, 16, prefix=prefix, seed=11)
    call, eager = Call(gpu, sc, single=True), Call(gpu, sc, single=True)
    graph = Graph(call)
    for n in lens + lens:
        sc.lens = n
        sc.q = sc.rng.standard_normal(sc.q.shape).astype(np.float32)
        for c in (call, eager):
            c.kv_len.upload(np.array(n, np.uint32))
            c.put_q(sc.q)
        graph.replay()
        eager()
        a, b = call.result()[0], eager.result()[0]
        _check(sc, a)
        assert np.array_equal(a, b)


def test_pool_beyond_32_bits(gpu):
    """Pages whose bytes lie past 2^31 and elements past 2^32."""
    kvh, hd, page = 8, 128, 256
    size = kvh * hd * page * 17 // 32
    n_pages = (1 << 32) // (kvh * hd * page) + 40
    sc = MxScene([1, 1, 20], [700, 256, 300], 16, kvh, hd, page, seed=13, spare=0)
    call = Call(gpu, sc)
    small = n_pages - sc.n_pages                  # the scene's pages go to the end of a large pool
    big = [gpu.DeviceBuffer(n_pages * size) for _ in range(2)]
    for b, src in zip(big, (call.k, call.v)):
        gpu.check(gpu.lib().yl_memcpy_d2d(b.ptr + small * size, src.ptr, src.nbytes))
    call.cache.keys, call.cache.values, call.cache.n_pages = big[0].ptr, big[1].ptr, n_pages
    call.table.upload(np.where(sc.table >= 0, sc.table + small, sc.table).astype(np.int32))
    call()
    _check(sc, call.result()[0])
    k, v = (sc.rng.standard_normal((sc.total, kvh * hd), np.float32) for _ in range(2))
    dk, dv, out = buffer(k), buffer(v), filled((2, sc.total, kvh * hd), 0.0)
    gpu.check(gpu.lib().yl_paged_append(C.byref(call.cache), C.byref(call.batch), sc.heads, None, 0, None, 0, dk.ptr, kvh * hd,
                                        dv.ptr, kvh * hd, gpu.ROPE_PAIRS["none"], None, None, 0, None))
    gpu.check(gpu.lib().yl_paged_gather(C.byref(call.cache), C.byref(call.batch), out.ptr, kvh * hd, out.ptr + 4 * k.size, kvh * hd, None))
    gpu.check(gpu.lib().yl_synchronize())
    for got, x in zip(out.numpy(), (k, v)):
        assert np.array_equal(got, X.rounded(x.reshape(sc.total, kvh, hd)).reshape(got.shape))


SCENES = {
    "decode_64": lambda: MxScene([1] * 6, [33, 64, 127, 200, 257, 600], 32, 8, 64, 16, seed=1),
    "decode_128": lambda: MxScene([1] * 6, [33, 64, 127, 200, 257, 600], 8, 1, 128, 16, spread=1.0, seed=1),
    "long_64": lambda: MxScene([1, 1, 1, 2], [3001, 40, 1777, 2050], 4, 1, 64, 64, spread=1.0, seed=2),
    "prompt_32": lambda: MxScene([70, 3], [90, 300], 8, 2, 32, 16, seed=3),
    "prefix_64": lambda: MxScene([1, 5, 1, 2, 40, 1, 3], [334, 342, 383, 333, 393, 330, 334], 8, 2, 64, 16, prefix=333, seed=4),
    "tile_64": lambda: MxScene([40, 0, 33, 70], [40, 7, 530, 75], 160, 160, 64, 16, spread=1.0, seed=5),
    "tile_128": lambda: MxScene([40, 0, 33, 70], [77, 44, 167, 112], 160, 160, 128, 16, prefix=37, seed=5),
    "tile_prefix_64": lambda: MxScene([1] * 35 + [9], [1011 + 7 * i for i in range(36)], 192, 32, 64, 32, prefix=1010, seed=6),
}


@pytest.mark.parametrize("scene", list(SCENES))
def test_no_less_exact_than_f32_loops(gpu, scene):
    """The RMS error over rows and heads is that of an f32 evaluation of the values that the pages stand for."""
    sc = SCENES[scene]()
    plain = sc.plain()
    at = P.sample(plain, 150)
    ref = P.exact(plain, at)
    out = _attend(sc).reshape(sc.total, sc.heads, sc.hd)
    err = P.rms(np.array([out[a] for a in at]) - ref)
    assert err <= P.allowed(plain, at, ref), f"{err / P.allowed(plain, at, ref):.3g} of what is allowed"


@pytest.mark.parametrize("heads,kvh,prefix", [(8, 2, 0), (8, 2, 40), (160, 160, 0)])
def test_serving_steps(gpu, heads, kvh, prefix):
    """Prompts and decoded rows are appended and attended to in one stream: over the pages as the append left them."""
    hd, page, seqs = 64, 16, 3
    sc = MxScene([0] * seqs, [prefix + 80] * seqs, heads, kvh, hd, page, prefix=prefix, seed=30)
    own = [p for row in sc.table for p in row]
    sc.k32[own] = np.nan
    sc.v32[own] = np.nan                      # nothing of their own yet
    cos, sin = _tables(hd, 200, seed=1)
    lens, width = [prefix] * seqs, (heads + 2 * kvh) * hd
    call = None
    for rows in [[20, 1, 33], [1, 1, 1], [1, 4, 1], [1, 1, 1]]:
        lens = [n + r for n, r in zip(lens, rows)]
        sc.rows, sc.lens = rows, lens
        sc.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
        sc.total = sum(rows)
        x = sc.rng.standard_normal((sc.total, width), np.float32)
        sc.q = np.ascontiguousarray(x[:, :heads * hd])
        call = Call(gpu, sc)                  # (uploads the pools as they are now)
        dx, dc, ds, stream = buffer(x), buffer(cos), buffer(sin), Stream()
        gpu.check(gpu.lib().yl_synchronize())
        at, st = dx.ptr, stream.handle
        gpu.check(gpu.lib().yl_paged_append(C.byref(call.cache), C.byref(call.batch), heads, call.q.ptr, heads * hd, at, width,
                                            at + 4 * heads * hd, width, at + 4 * (heads + kvh) * hd, width, 1, dc.ptr, ds.ptr, 200, st))
        call(st)
        out = call.result()[0]
        pos = np.concatenate([np.arange(n - r, n) for r, n in zip(rows, lens)])
        k = _rotated32(x[:, heads * hd:(heads + kvh) * hd], cos, sin, pos, "half", kvh, hd)
        sc.k32, sc.v32 = X.unpacked(call.k.numpy()), X.unpacked(call.v.numpy())
        row = 0
        for s, (r, n) in enumerate(zip(rows, lens)):
            for page_id, slot in sc.places(s, n)[n - r:]:
                assert np.array_equal(sc.k32[page_id, :, slot], X.rounded(k[row]))
                row += 1
        sc.q = call.q.numpy().reshape(sc.total, -1)
        _check(sc, out)


# ---------------------------- one row per sequence, up to four heads per kv head


@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 32), (8, 2, 64), (6, 2, 64), (2, 2, 128), (8, 2, 128)])
@pytest.mark.parametrize("prefix", [0, 37])
@pytest.mark.parametrize("kind", ["few_long", "many_long", "many_short"])
def test_single_rows(gpu, heads, kvh, hd, prefix, kind):
    """Units of four wavefronts and of one, split and whole (128 and 1600 sequences times kv heads, 640 positions), ends
    inside every quad of positions, and entries, lengths and sequences of nothing."""
    rng = np.random.default_rng(heads + hd)
    lens = {"few_long": [1500, 1, 701, 64, 65, 66, 67, 0, 130], "many_long": [1100, 900] + list(range(68)),
            "many_short": [int(x) for x in rng.integers(0, 70, 810)]}[kind]
    lens = [prefix + n for n in lens]
    assert len(lens) * kvh >= {"few_long": 1, "many_long": 128, "many_short": 1600}[kind]
    sc = MxScene([1] * len(lens), lens, heads, kvh, hd, 16, spread=1.0, prefix=prefix, seed=hd, extra_entries=1)
    sc.table[0, 2] = -1
    sc.table[2, 0] = sc.n_pages
    if kind == "few_long":
        sc.lens[3] = prefix + 16 * sc.table.shape[1] + 500      # past its table (this one fills its pages)
    _check(sc, _attend(sc, single=True, max_len=0 if kind == "few_long" else max(lens)))


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("seqs", [3, 70])
@pytest.mark.parametrize("slope", [0.3, -0.3, 2.0])
def test_values_that_grow(gpu, hd, seqs, slope):
    """Values of position p are 2^(slope p / 8) times the first ones (up to 2^120): the exponent that they are held against
    follows; the bound is that of the largest value."""
    sc = MxScene([1] * seqs, [700] + [90] * (seqs - 1), 4, 2, hd, 16, seed=5)
    for s in range(min(seqs, 3)):
        for p, (page, slot) in enumerate(sc.places(s, sc.lens[s])):
            sc.v32[page, :, slot] *= np.float32(2.0 ** np.clip(slope * p / 8, -60, 100))
    sc.settle()
    _check(sc, _attend(sc, single=True))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("seqs", [3, 70])
@pytest.mark.parametrize("power", [12, 40])
def test_keys_of_unlike_blocks(gpu, hd, seqs, power):
    """A block of a key that is 2^12 or 2^40 times the others, in a few positions and with queries that bring it back."""
    sc = MxScene([1] * seqs, [700] + [90] * (seqs - 1), 4, 2, hd, 16, seed=6)
    sc.k32[:, :, ::3, 32:] *= np.float32(2.0 ** power)
    q = sc.q.reshape(seqs, 4, hd)
    q[..., 32:] *= np.float32(2.0 ** -power)
    sc.settle()
    _check(sc, _attend(sc, single=True))


@pytest.mark.parametrize("heads,kvh,hd", [(8, 2, 64), (8, 2, 128), (4, 4, 32)])
@pytest.mark.parametrize("seqs", [3, 70])
@pytest.mark.parametrize("size", [2.0, 5.0, 12.0])
def test_scores_far_apart(gpu, heads, kvh, hd, seqs, size):
    """As over f16 pages: what the weights are taken against rises and falls; the RMS error stays that of an f32 evaluation."""
    sc = MxScene([1] * seqs, [1500, 700] + [80] * (seqs - 2), heads, kvh, hd, 16, seed=int(size))
    sc.q *= np.float32(size)
    for at in (5, 130, 131, 400):
        page, slot = sc.places(0, 600)[at]
        sc.k32[page, :, slot] *= 2.5
    sc.settle()
    plain = sc.plain()
    at = P.sample(plain, 150)
    ref = P.exact(plain, at)
    out = _attend(sc, single=True).reshape(sc.total, sc.heads, sc.hd)
    err = P.rms(np.array([out[a] for a in at]) - ref)
    assert err <= P.allowed(plain, at, ref), f"{err / P.allowed(plain, at, ref):.3g} of what is allowed"


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("seqs", [3, 70])
def test_no_numbers_in_single_rows(gpu, hd, seqs):
    """A NaN block of a value spoils its 32 components of that sequence, a NaN key its row; no other sequence feels it."""
    sc = MxScene([1] * seqs, [700] + [90] * (seqs - 1), 4, 2, hd, 16, seed=7)
    page, slot = sc.places(0, 700)[333]
    sc.v32[page, :, slot, :32] = np.nan
    page1, slot1 = sc.places(1, 90)[17]
    sc.k32[page1, :, slot1, -5] = np.inf
    sc.settle()
    out = _attend(sc, single=True).reshape(seqs, 4, hd)
    sc.v32[page, :, slot, :32] = 0.0
    ref, bound = (x.reshape(seqs, 4, hd) for x in sc.plain().attention())
    assert np.isnan(out[0, :, :32]).all() and np.isnan(out[1]).all()
    assert (np.abs(out[0] - ref[0])[:, 32:] <= bound[0][:, 32:]).all()
    assert (np.abs(out[2:] - ref[2:]) <= bound[2:]).all()


def test_no_queries(gpu):
    """Queries of zero weigh all positions alike; queries that are no numbers spoil their own row and head alone."""
    sc = MxScene([1] * 4, [700, 90, 5, 64], 8, 2, 64, 16, seed=8)
    sc.q[0] = 0.0
    sc.q[1, 64 + 3] = np.nan
    sc.q[3, 7 * 64] = np.inf
    out = _attend(sc, single=True).reshape(4, 8, 64)
    sc.q[1, 64 + 3] = sc.q[3, 7 * 64] = 0.0
    ref, bound = (x.reshape(4, 8, 64) for x in sc.attention())
    fine = np.ones((4, 8), bool)
    fine[1, 1] = fine[3, 7] = False
    assert np.isnan(out[1, 1]).all()
    assert (np.abs(out - ref)[fine] <= bound[fine]).all()


def test_single_rows_same_bits(gpu):
    """No sum's order depends on which workgroup ends first; alone or among others, in place or not."""
    sc = MxScene([1] * 70, [3000, 900] + [60] * 68, 8, 2, 64, 16, seed=12)
    call = Call(gpu, sc, single=True)
    outs = []
    for _ in range(4):
        call.out.upload(np.zeros(call.out.shape, np.float32))
        call()
        outs.append(call.result()[0].copy())
    assert all(np.array_equal(outs[0], o) for o in outs[1:])
    call(in_place=True)
    assert np.array_equal(call.result(call.q)[0], outs[0])
    _check(sc, outs[0])
