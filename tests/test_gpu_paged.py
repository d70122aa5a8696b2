"""yl_paged_append and yl_paged_attention against 64-bit numpy (bounds derived
in paged_np.Scene.attention): types, head layouts, page sizes, lengths from
nothing to several chunks, ragged rows, shared prefixes, missing pages,
garbage wherever nothing is attended to, strides, streams and graphs."""
import ctypes as C

import numpy as np
import pytest

from hip_rt import Graph, Stream, buffer, bytes_of, filled
from paged_np import Scene, logprobs, rotated, to_cache, widened

pytestmark = pytest.mark.gpu


def _check(sc, out):
    ref, bound = sc.attention()
    err = np.abs(out - ref)
    assert np.isfinite(out).all()
    assert (err <= bound).all(), f"off by {np.max(err / np.maximum(bound, 1e-30)):.3g} of the bound"
    return ref


def _attend(sc, single=False, max_len=0):
    from yallma3_mini_inference_amd import ops
    k, v = sc.pools()
    return ops.paged_attention(k, v, sc.batch(ops, single, max_len), sc.q, sc.heads, sc.scale)


LAYOUTS = [(4, 2, 32), (9, 3, 64), (8, 1, 128), (2, 2, 128), (32, 8, 64), (17, 1, 32), (40, 2, 64)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
def test_decode_rows(gpu, dtype, heads, kvh, hd):
    """One row per sequence, lengths around page and tile ends."""
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 200, 257]
    sc = Scene([1] * len(lens), lens, heads, kvh, hd, 16, dtype, seed=heads + hd)
    _check(sc, _attend(sc, single=True))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_ragged_rows(gpu, dtype, page):
    """Prompts, turns and single rows together, with sequences that have no
    rows, and rows before and behind all sequences left as they were."""
    rows, lens = [1, 70, 0, 5, 33, 1, 0, 130, 16], [300, 70, 12, 90, 34, 1, 0, 199, 16]
    sc = Scene(rows, lens, 8, 2, 64, page, dtype, seed=page)
    _check(sc, _attend(sc))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
def test_prompt_rows(gpu, dtype, heads, kvh, hd):
    sc = Scene([90, 41], [90, 170], heads, kvh, hd, 32, dtype, seed=heads)
    _check(sc, _attend(sc))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("prefix", [1, 16, 37, 333])
@pytest.mark.parametrize("heads,kvh,hd", [(4, 2, 32), (8, 2, 64), (8, 1, 128)])
def test_shared_prefix(gpu, dtype, prefix, heads, kvh, hd):
    """Single rows, several rows, rows inside the prefix itself, a sequence
    that holds nothing of its own."""
    rows = [1, 5, 1, 2, 40, 1, 3]
    lens = [prefix + 1, prefix + 9, prefix + 50, prefix, prefix + 60, max(1, prefix - 3), prefix + 1]
    sc = Scene(rows, lens, heads, kvh, hd, 16, dtype, prefix=prefix, seed=prefix)
    _check(sc, _attend(sc))


# (enough rows and kv heads for the tile kernel: 160 workgroups of 128 stacked rows)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,hd", [(160, 160, 32), (160, 160, 64), (160, 160, 128), (160, 80, 64)])
@pytest.mark.parametrize("prefix", [0, 37])
def test_many_prompt_rows(gpu, dtype, heads, kvh, hd, prefix):
    """Prompts beside single rows, sequences without rows and rows inside the prefix."""
    rows = [1, 40, 0, 33, 2, 70] if kvh == 160 else [1, 70, 0, 17, 2, 60]
    lens = [prefix + n for n in (90, 40, 7, 130, 20, 75)]
    lens[1] -= prefix // 2
    sc = Scene(rows, lens, heads, kvh, hd, 16, dtype, prefix=prefix, seed=hd)
    _check(sc, _attend(sc))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_many_prompt_rows_over_gaps_and_no_numbers(gpu, dtype, hd):
    """The tile kernel's masks: missing pages, lengths past the table, later
    positions that hold no numbers, rows behind the sequences, odd strides."""
    sc = Scene([50, 70, 3], [50, 300, 64], 160, 160, hd, 16, dtype, seed=hd, extra_entries=1, behind=2)
    sc.table[1, 3] = -1
    sc.table[1, 7] = sc.n_pages
    sc.lens[2] = 16 * sc.table.shape[1] + 500
    page = sc.table[0, 2]
    sc.v32[page, :, 5, 3] = np.inf          # position 37 of the first sequence
    sc.k32[sc.table[0, 2], :, 9] = np.nan   # position 41
    call = Call(gpu, sc, q_ld=160 * hd + 5, out_ld=160 * hd + 3, offset=1)
    call()
    out, between = call.result()
    n = int(sc.starts[-1])
    assert (out[n:] == 7.0).all() and (between == 7.0).all()
    rows = out[:50].reshape(50, 160, hd)
    assert np.isfinite(rows[:37]).all() and not np.isfinite(rows[37:, :, 3]).any()
    assert np.isfinite(rows[37:41][..., :3]).all() and not np.isfinite(rows[41:]).any()
    sc.v32[page, :, 5, 3] = 0.0
    ref, bound = sc.attention()
    fine = np.isfinite(out[:n]) & np.isfinite(ref[:n])
    assert (np.abs(out[:n] - ref[:n])[fine] <= bound[:n][fine]).all()
    assert fine[:37].all() and fine[50:].all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_long_prefix_under_a_batch(gpu, dtype, hd):
    """A prefix long enough, under rows enough, for the tile kernel (2^23 stacked rows times positions)."""
    prefix, seqs = 1010, 36
    sc = Scene([1] * (seqs - 1) + [9], [prefix + 1 + 7 * i for i in range(seqs)], 192, 32, hd, 32, dtype, prefix=prefix, seed=hd)
    assert 44 * 6 * 32 * prefix >= 8 << 20
    _check(sc, _attend(sc))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_prefix_equals_own_pages(gpu, dtype):
    """The same positions as a prefix and as pages of each sequence's table
    (of one pool: pages may be named by several sequences)."""
    from yallma3_mini_inference_amd import ops
    sc = Scene([1, 1, 4], [64 + 5, 64 + 40, 64 + 17], 8, 2, 64, 16, dtype, prefix=64, seed=3)
    k, v = sc.pools()
    a = ops.paged_attention(k, v, sc.batch(ops), sc.q, sc.heads, sc.scale)
    table = np.concatenate([np.tile(sc.prefix_pages, (3, 1)), sc.table], 1)
    b = ops.paged_attention(k, v, ops.PagedBatch(table, sc.lens, sc.starts), sc.q, sc.heads, sc.scale)
    ref, bound = sc.attention()
    assert (np.abs(a - ref) <= bound).all() and (np.abs(b - ref) <= bound).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("max_len", [0, 100, 5000])
def test_long_contexts_in_chunks(gpu, dtype, hd, max_len):
    """Lengths over several chunks; max_len below, and far above, the real lengths."""
    sc = Scene([1, 1, 1, 2], [3001, 40, 1777, 2050], 4, 1, hd, 64, dtype, seed=hd)
    _check(sc, _attend(sc, max_len=max_len))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_positions_nobody_holds(gpu, dtype):
    """Entries that name no page in the middle of a table, kv_len past the
    table, lengths of zero, rows at negative positions: nothing there."""
    rows, lens = [1, 30, 3, 2, 1, 4], [100, 150, 64, 1, 0, 40]    # (the third fills its pages)
    sc = Scene(rows, lens, 8, 2, 64, 16, dtype, seed=1, extra_entries=1)
    sc.table[0, 2] = -1
    sc.table[1, 0] = sc.n_pages          # not below n_pages
    sc.table[1, 5] = 0x7FFFFFFF
    sc.table[5, :] = -5                  # nothing held at all
    sc.lens[2] = 16 * sc.table.shape[1] + 500   # far past the table (whose last entry names no page)
    ref = _check(sc, _attend(sc))
    assert not ref[sc.starts[5]:].any() and not ref[sc.starts[3]].any()     # zeros, as checked


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_non_finite_values_of_later_positions(gpu, dtype, bad):
    """A later row's key or value that is no number takes no part in the rows before it."""
    sc = Scene([40, 1], [75, 20], 8, 2, 64, 16, dtype, seed=5)
    page, slot = sc.table[0, 60 // 16], 60 % 16
    sc.k32[page, :, slot] = bad
    sc.v32[page, :, slot, ::3] = bad
    out = _attend(sc)
    ref, bound = sc.attention()
    before = 60 - 35                     # rows of positions 35 .. 59
    err = np.abs(out[:before] - ref[:before])
    assert (err <= bound[:before]).all()
    assert not np.isfinite(out[before:40].reshape(15, 8, 64)[..., ::3]).any()
    assert (np.abs(out[40] - ref[40]) <= bound[40]).all()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_non_finite_value_alone(gpu, dtype, bad):
    """Only one value component of a later position: the other components stay numbers in every row."""
    sc = Scene([64], [64], 4, 1, 32, 16, dtype, seed=6)
    sc.v32[sc.table[0, 2], :, 3, 7] = bad       # position 35
    out = _attend(sc).reshape(64, 4, 32)
    fine = np.isfinite(out)
    assert fine[:35].all() and not fine[35:, :, 7].any()
    assert fine[35:][..., [i for i in range(32) if i != 7]].all()
    sc.v32[sc.table[0, 2], :, 3, 7] = 0.0
    ref, bound = sc.attention()
    ref, bound = ref.reshape(64, 4, 32), bound.reshape(64, 4, 32)
    assert (np.abs(out - ref)[fine] <= bound[fine]).all()


@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("dtype,heads,kvh", [("f32", 8, 2), ("f16", 8, 2), ("bf16", 8, 2), ("f16", 160, 160), ("bf16", 160, 160)])
@pytest.mark.parametrize("prefix", [0, 30])
def test_non_finite_queries(gpu, dtype, heads, kvh, bad, prefix):
    """Queries that are no numbers spoil their own row and head alone (in both kernels)."""
    sc = Scene([1, 70, 60, 3], [prefix + n for n in (700, 90, 60, 5)], heads, kvh, 32, 16, dtype, prefix=prefix, seed=17)
    spoilt = [(0, 1), (5, 0), (5, heads - 1), (100, 3), (133, 2)]
    for row, head in spoilt:
        sc.q[row, head * 32 + 3] = bad
    out = _attend(sc).reshape(sc.total, heads, 32)
    for row, head in spoilt:
        sc.q[row, head * 32 + 3] = 0.0
    ref, bound = (x.reshape(sc.total, heads, 32) for x in sc.attention())
    fine = np.ones((sc.total, heads), bool)
    for row, head in spoilt:
        fine[row, head] = False
    assert not np.isnan(bad) or np.isnan(out[~fine]).all()
    assert (np.abs(out - ref)[fine] <= bound[fine]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [1e-4, 30.0])
def test_small_and_large_scores(gpu, dtype, size):
    """Queries far from 1: the parts that a query is held in keep its precision."""
    sc = Scene([1, 20], [500, 90], 4, 2, 64, 16, dtype, seed=8)
    sc.q *= np.float32(size)
    sc.q[3] *= np.float32(1e-6)
    _check(sc, _attend(sc))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
def test_scales(gpu, dtype, scale):
    """A negative scale turns the order of the scores around, 0 makes all weights equal."""
    sc = Scene([1, 20, 60], [500, 90, 60], 4, 2, 64, 16, dtype, seed=15)
    sc.scale = scale
    _check(sc, _attend(sc))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kvh,rows", [(2, 20), (160, 40)])
def test_subnormal_keys_and_values(gpu, dtype, kvh, rows):
    """f16 keys and values below its least normal number (and bf16 ones as small) count in full, in both kernels."""
    sc = Scene([1, rows], [200, 70], kvh, kvh, 32, 16, dtype, seed=16)
    sc.k32 *= np.float32(1e-5)
    sc.v32 *= np.float32(1e-6)
    sc.q *= np.float32(3e5)
    ref = _check(sc, _attend(sc))
    assert 0 < np.abs(ref).max() < 1e-5


class Call:
    """A call on device arrays, as a program that keeps its own memory makes it."""

    def __init__(self, yl, sc, q_ld=None, out_ld=None, single=False, max_len=0, offset=0):
        self.yl, self.sc = yl, sc
        k, v = sc.pools()
        self.k, self.v = buffer(k), buffer(v)
        width = sc.heads * sc.hd
        q_ld, out_ld = q_ld or width, out_ld or width
        self.q_ld, self.out_ld, self.offset, self.width = q_ld, out_ld, offset, width
        self.q, self.out = filled(sc.total * q_ld + offset, 0.0), filled(sc.total * out_ld + offset, 7.0)
        self.put_q(sc.q)
        self.table, self.kv_len, self.starts = buffer(sc.table), buffer(np.array(sc.lens, np.uint32)), buffer(sc.starts)
        self.pre = buffer(sc.prefix_pages) if sc.prefix else None
        self.cache = yl.PagedCacheDesc(self.k.ptr, self.v.ptr, yl.DTYPES[sc.dtype], sc.n_pages, sc.page, sc.kvh, sc.hd)
        self.batch = yl.PagedBatchDesc(len(sc.lens), sc.total, sc.table.shape[1], max_len, self.table.ptr, self.kv_len.ptr,
                                       None if single else self.starts.ptr, sc.prefix, self.pre.ptr if sc.prefix else None)
        self.need = yl.lib().yl_paged_attention_workspace(C.byref(self.cache), C.byref(self.batch), sc.heads)
        self.space = bytes_of(self.need, 255)       # NaN where it is read unwritten

    def put_q(self, q):
        h = np.zeros(self.sc.total * self.q_ld + self.offset, np.float32)
        h[self.offset:].reshape(self.sc.total, self.q_ld)[:, :self.width] = q
        self.q.upload(h)

    def __call__(self, stream=None, in_place=False):
        at = 4 * self.offset
        self.yl.check(self.yl.lib().yl_paged_attention((self.q if in_place else self.out).ptr + at, self.out_ld, self.q.ptr + at,
                                                       self.q_ld, C.byref(self.cache), C.byref(self.batch), self.sc.heads,
                                                       self.sc.scale, self.space.ptr, self.need, stream))

    def result(self, which=None):
        """The rows, and what lies between them."""
        self.yl.check(self.yl.lib().yl_synchronize())
        rows = (which or self.out).numpy()[self.offset:].reshape(self.sc.total, self.out_ld)
        return rows[:, :self.width], rows[:, self.width:]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("prefix", [0, 50])
def test_strides_alignment_and_rows_behind(gpu, dtype, prefix):
    """Rows at odd strides from an odd address; what lies between the rows and
    the rows behind the last sequence stay as they were."""
    sc = Scene([1, 20, 0, 3], [prefix + 50, prefix + 20, prefix + 5, prefix + 300], 4, 2, 64, 16, dtype, prefix=prefix, seed=9, behind=3)
    call = Call(gpu, sc, q_ld=4 * 64 + 5, out_ld=4 * 64 + 3, offset=1)
    call()
    out, between = call.result()
    n = int(sc.starts[-1])
    ref, bound = sc.attention()
    assert (np.abs(out[:n] - ref[:n]) <= bound[:n]).all()
    assert (out[n:] == 7.0).all() and (between == 7.0).all() and call.out.numpy()[0] == 7.0


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("prefix", [0, 50])
def test_in_place(gpu, dtype, prefix):
    sc = Scene([1, 40, 3], [prefix + 1500, prefix + 60, prefix + 30], 8, 2, 64, 16, dtype, prefix=prefix, seed=10)
    call = Call(gpu, sc)
    call(in_place=True)
    _check(sc, call.result(call.q)[0])


def test_streams_side_by_side(gpu):
    """Two calls at once on streams of their own, each with its workspace."""
    scs = [Scene([1] * 6, [900, 40, 1300, 7, 600, 90], 8, 2, 64, 16, "f16", seed=20),
           Scene([60, 1], [200, 800], 8, 2, 64, 16, "bf16", prefix=0, seed=21)]
    calls, streams = [Call(gpu, s) for s in scs], [Stream() for _ in scs]
    gpu.check(gpu.lib().yl_synchronize())
    for _ in range(5):
        for c, st in zip(calls, streams):
            c(st.handle)
    for c, s in zip(calls, scs):
        _check(s, c.result()[0])


@pytest.mark.parametrize("prefix", [0, 70])
def test_graph_replays_read_new_lengths(gpu, prefix):
    """A captured call, replayed with other lengths and queries, an eager call between the replays."""
    lens = [[prefix + 30, prefix + 500, prefix + 1], [prefix + 33, prefix + 511, prefix + 64], [prefix + 60, prefix + 9, prefix + 600]]
    sc = Scene([1, 1, 1], [prefix + 620] * 3, 8, 2, 64, 16, "f16", prefix=prefix, seed=11)
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


def test_same_call_same_bits(gpu):
    """No sum's order depends on which workgroup ends first."""
    sc = Scene([1, 1, 9, 50], [3000, 150, 700, 90], 8, 2, 64, 16, "f16", prefix=0, seed=12)
    call = Call(gpu, sc)
    outs = []
    for _ in range(4):
        call.out.upload(np.zeros(call.out.shape, np.float32))
        call()
        outs.append(call.result()[0].copy())
    assert all(np.array_equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_pool_beyond_32_bits(gpu, dtype):
    """Pages whose elements lie past 2^31 (and, in f32, bytes past 2^33)."""
    kvh, hd, page = 8, 128, 256
    n_pages = (1 << 31) // (kvh * hd * page) + 40
    sc = Scene([1, 1, 20], [700, 256, 300], 16, kvh, hd, page, dtype, seed=13, spare=0)
    call = Call(gpu, sc)
    small = n_pages - sc.n_pages                  # the scene's pages go to the end of a large pool
    size = kvh * hd * page * (4 if dtype == "f32" else 2)
    big = [gpu.DeviceBuffer(n_pages * size) for _ in range(2)]
    for b, src in zip(big, (call.k, call.v)):
        gpu.check(gpu.lib().yl_memcpy_d2d(b.ptr + small * size, src.ptr, src.nbytes))
    call.cache.keys, call.cache.values, call.cache.n_pages = big[0].ptr, big[1].ptr, n_pages
    call.table.upload(np.where(sc.table >= 0, sc.table + small, sc.table).astype(np.int32))
    call()
    _check(sc, call.result()[0])
    k, v = (sc.rng.standard_normal((sc.total, kvh * hd), np.float32) for _ in range(2))
    dk, dv = buffer(k), buffer(v)
    gpu.check(gpu.lib().yl_paged_append(C.byref(call.cache), C.byref(call.batch), sc.heads, None, 0, None, 0, dk.ptr, kvh * hd,
                                        dv.ptr, kvh * hd, gpu.ROPE_PAIRS["none"], None, None, 0, None))
    for b, src in zip(big, (call.k, call.v)):
        gpu.check(gpu.lib().yl_memcpy_d2d(src.ptr, b.ptr + small * size, src.nbytes))
    _, pk, pv, _, touched = _appended(sc, sc.q, k, v, None, None, "none", 0)
    for got, ref in ((call.k, pk), (call.v, pv)):
        assert np.array_equal(got.numpy()[touched], ref[touched].astype(got.dtype))


def test_many_sequences(gpu):
    """More sequences than any tile of threads, some without rows."""
    rng = np.random.default_rng(14)
    rows = [int(x) for x in rng.integers(0, 3, 700)]
    lens = [int(r + x) for r, x in zip(rows, rng.integers(0, 30, 700))]
    sc = Scene(rows, lens, 2, 1, 32, 16, "f16", seed=14)
    _check(sc, _attend(sc))


@pytest.mark.parametrize("seqs", [200, 256, 257, 512, 513, 1500])
@pytest.mark.parametrize("single,prefix", [(True, 0), (False, 0), (False, 37), (True, 37)])
def test_long_sequences_among_many(gpu, seqs, single, prefix):
    """Two long sequences among many short ones, on both sides of every number
    of sequences from which on the work is divided in another way."""
    rng = np.random.default_rng(seqs)
    rows = [1] * seqs if single else [int(x) for x in rng.integers(0, 4, seqs)]
    lens = [prefix + int(r + x) for r, x in zip(rows, rng.integers(0, 40, seqs))]
    for at, n in ((seqs // 3, 2500), (seqs - 1, 1900)):
        rows[at], lens[at] = max(rows[at], 1), prefix + n
    sc = Scene(rows, lens, 2, 1, 32, 16, "f16", prefix=prefix, seed=seqs)
    _check(sc, _attend(sc, single))


@pytest.mark.parametrize("seqs", [300, 1040])
@pytest.mark.parametrize("prefix", [0, 20])
def test_prompts_among_many_sequences(gpu, seqs, prefix):
    """The same, with prompts among them that the tile kernel takes (160 workgroups of 128 stacked rows)."""
    rows = [1] * seqs
    for at in range(5, 300, 15):
        rows[at] = 33 + at // 3
    lens = [prefix + r + i % 9 for i, r in enumerate(rows)]
    lens[7] = prefix + 800
    sc = Scene(rows, lens, 16, 16, 32, 16, "bf16", prefix=prefix, seed=seqs)
    assert -(-sum(rows) // 128) * 16 >= 160
    _check(sc, _attend(sc))


# ------------------------------------------------------------------ append


def _tables(hd, rows, seed=0):
    a = np.random.default_rng(seed).uniform(0, 2 * np.pi, (rows, hd // 2))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _appended(sc, q, k, v, cos, sin, pairs, rope_rows):
    """The pools after the call (f64; NaN as before), q, and which rows are passed over."""
    pk, pv = (widened(x) for x in sc.pools())
    pos = np.zeros(sc.total, int)
    out = [None] * sc.total
    for s, n in enumerate(sc.lens):
        for r in range(sc.starts[s], sc.starts[s + 1]):
            pos[r] = n - (int(sc.starts[s + 1]) - r)
            out[r] = s if pos[r] >= 0 and (pairs == "none" or pos[r] < rope_rows) else None
    at = np.clip(pos, 0, len(cos) - 1 if cos is not None else None)
    rq, rk = rotated(q, cos, sin, at, pairs, sc.heads, sc.hd), rotated(k, cos, sin, at, pairs, sc.kvh, sc.hd)
    touched = np.zeros(pk.shape[:3], bool)
    for r, s in enumerate(out):
        if s is None or pos[r] < sc.prefix:
            continue
        i = pos[r] - sc.prefix
        if i // sc.page < sc.table.shape[1] and 0 <= sc.table[s, i // sc.page] < sc.n_pages:
            page, slot = sc.table[s, i // sc.page], i % sc.page
            pk[page, :, slot], pv[page, :, slot] = rk[r], v[r].reshape(sc.kvh, sc.hd)
            touched[page, :, slot] = True
    return rq.reshape(sc.total, -1), pk, pv, np.array([s is not None for s in out]), touched


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairs", ["none", "adjacent", "half"])
@pytest.mark.parametrize("heads,kvh,hd,page", [(4, 2, 32, 16), (9, 3, 64, 32), (8, 1, 128, 256), (2, 2, 64, 64)])
def test_append(gpu, dtype, pairs, heads, kvh, hd, page):
    from yallma3_mini_inference_amd import ops
    prefix = 20
    rows, lens = [1, 40, 0, 3, 1, 5, 2, 1], [90, 40, 7, 300, 1, 22, 21, 400]
    sc = Scene(rows, lens, heads, kvh, hd, page, dtype, prefix=prefix, seed=hd)
    sc.table[3, (299 - prefix) // page] = sc.n_pages     # the last page of the fourth sequence is missing
    rope_rows = 350                                      # the last row lies beyond the tables
    cos, sin = _tables(hd, rope_rows) if pairs != "none" else (None, None)
    k, v = (sc.rng.standard_normal((sc.total, kvh * hd), np.float32) for _ in range(2))
    pk, pv = sc.pools()
    q2, k2, v2 = ops.paged_append(pk, pv, sc.batch(ops), sc.q, k, v, heads, pairs, cos, sin)
    rq, rk, rv, live, touched = _appended(sc, sc.q, k, v, cos, sin, pairs, rope_rows)
    # two rounded products and their sum: 2 U |a| + U |result|, |a c| + |b s| <= |a| + |b|
    big = 2.0 * np.abs(sc.q).max()
    if pairs == "none":
        assert np.array_equal(q2[live], sc.q[live])
    else:
        assert np.abs(q2[live] - rq[live]).max() <= 3 * 2.0 ** -24 * big
    assert np.array_equal(q2[~live], sc.q[~live])        # in place, passed over
    assert touched.any() and not touched.all()
    for got, ref, before, x in ((k2, rk, pk, k), (v2, rv, pv, v)):
        assert np.array_equal(got[~touched].view(np.uint8), before[~touched].view(np.uint8))
        err = np.abs(widened(got)[touched] - ref[touched])
        assert (err <= STEP[dtype] * np.abs(ref[touched]) * (1 + 2.0 ** -10) + 2.0 ** -24 * (1 if dtype == "f16" else 0)
                + 3 * 2.0 ** -24 * 2 * np.abs(x).max()).all()
    rounded = to_cache(v.reshape(sc.total, kvh, hd), dtype)          # values are rounded once, to nearest
    s, r = 1, int(sc.starts[1])
    i = lens[1] - 40 - prefix                                        # rows inside the prefix write nothing
    for j in range(40):
        if i + j >= 0:
            assert np.array_equal(v2[sc.table[s, (i + j) // page], :, (i + j) % page], rounded[r + j])


def test_append_rotates_as_rope_gguf(gpu):
    """The bits of yl_rope_gguf from yl_rope_table's tables."""
    from yallma3_mini_inference_amd import ops
    from yallma3_mini_inference_amd._lib import RopeParams
    hd, heads, kvh, start, rows = 64, 8, 2, 37, 21
    p = RopeParams(hd, heads, kvh, 500000.0, 1.0, 0.0, 1.0, 8192)
    sc = Scene([rows], [start + rows], heads, kvh, hd, 16, "f32", seed=2)
    k, v = (sc.rng.standard_normal((rows, kvh * hd), np.float32) for _ in range(2))
    cos, sin = ops.rope_table(p, "adjacent", 64)
    q2, k2, _ = ops.paged_append(*sc.pools(), sc.batch(ops), sc.q, k, v, heads, "adjacent", cos, sin)
    rq, rk = ops.rope_gguf(p, sc.q, k, start, rows)
    assert np.array_equal(q2.view(np.uint32), rq.view(np.uint32))
    got = np.stack([k2[pg, :, sl] for pg, sl in sc.places(0, start + rows)[start:]])
    assert np.array_equal(got.reshape(rows, -1).view(np.uint32), rk.view(np.uint32))


def test_append_keys_and_values_only(gpu):
    from yallma3_mini_inference_amd import ops
    sc = Scene([2], [20], 4, 2, 32, 16, "f16", seed=4)
    k, v = (sc.rng.standard_normal((2, 64), np.float32) for _ in range(2))
    q2, k2, v2 = ops.paged_append(*sc.pools(), sc.batch(ops), None, k, v, 4)
    assert q2 is None
    for r, (pg, sl) in enumerate(sc.places(0, 20)[18:]):
        assert np.array_equal(k2[pg, :, sl].ravel(), k[r].astype(np.float16)) and np.array_equal(v2[pg, :, sl].ravel(), v[r].astype(np.float16))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_append_rounds_extremes(gpu, dtype):
    """Ties, values beyond f16, subnormals, infinities and NaN."""
    from yallma3_mini_inference_amd import ops
    sc = Scene([1], [1], 1, 1, 32, 16, dtype, seed=4)
    v = np.zeros((1, 32), np.float32)
    v[0, :14] = [1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 65519.0, 65520.0, -1e38, 2.0 ** -25,
                 3 * 2.0 ** -25, 1e-40, -0.0, np.inf, -np.inf, np.nan]
    _, k2, v2 = ops.paged_append(*sc.pools(), sc.batch(ops), None, -v, v, 1)
    pg = sc.table[0, 0]
    with np.errstate(over="ignore"):
        for got, x in ((v2, v[0]), (k2, -v[0])):
            got = widened(got[pg, 0, 0])
            ref = widened(to_cache(np.where(np.isnan(x), 0, x), dtype))
            assert np.isnan(got[13])
            assert np.array_equal(got[:13], ref[:13]) and np.array_equal(np.signbit(got[:13]), np.signbit(ref[:13]))


@pytest.mark.parametrize("pairs", ["adjacent", "half"])
def test_append_fused_rows_at_odd_strides(gpu, pairs):
    """q, k and v as parts of fused rows whose length and address are odd; q to another array."""
    sc = Scene([1, 17], [40, 30], 6, 2, 64, 16, "f16", seed=5)
    ld, heads, kvh, hd = (6 + 4) * 64 + 3, 6, 2, 64
    x = sc.rng.standard_normal((sc.total, ld), np.float32)
    cos, sin = _tables(hd, 64)
    call = Call(gpu, sc)
    dx, dc, ds = buffer(np.concatenate([[0], x.ravel()]).astype(np.float32)), buffer(cos), buffer(sin)
    q_out = filled((sc.total, heads * hd + 1), 7.0)
    at = dx.ptr + 4
    gpu.check(gpu.lib().yl_paged_append(C.byref(call.cache), C.byref(call.batch), heads, q_out.ptr, heads * hd + 1, at, ld,
                                        at + 4 * heads * hd, ld, at + 4 * (heads + kvh) * hd, ld, gpu.ROPE_PAIRS[pairs],
                                        dc.ptr, ds.ptr, 64, None))
    k, v = x[:, heads * hd:(heads + kvh) * hd], x[:, (heads + kvh) * hd:(heads + 2 * kvh) * hd]
    rq, rk, rv, live, touched = _appended(sc, x[:, :heads * hd], k, v, cos, sin, pairs, 64)
    got = q_out.numpy()
    assert live.all() and (got[:, -1] == 7.0).all()
    assert np.abs(got[:, :-1] - rq).max() <= 6 * 2.0 ** -24 * np.abs(x).max()
    assert np.array_equal(call.v.numpy()[touched], rv[touched].astype(np.float16))


# ------------------------------------------------------- as they are used


def test_serving_steps(gpu):
    """A batch with a shared prefix: prompts and then decoded rows are appended
    and attended to in one stream, the results scored as logits."""
    from yallma3_mini_inference_amd import ops
    heads, kvh, hd, page, prefix, seqs = 8, 2, 64, 16, 40, 3
    sc = Scene([0] * seqs, [prefix + 80] * seqs, heads, kvh, hd, page, "f16", prefix=prefix, seed=30)
    own = [p for row in sc.table for p in row]
    sc.k32[own] = np.nan
    sc.v32[own] = np.nan                      # nothing of their own yet
    cos, sin = _tables(hd, 200, seed=1)
    lens = [prefix] * seqs
    width = (heads + 2 * kvh) * hd
    for step, rows in enumerate([[20, 1, 33], [1, 1, 1], [1, 4, 1], [1, 1, 1]]):
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
                                            at + 4 * heads * hd, width, at + 4 * (heads + kvh) * hd, width, 0, dc.ptr, ds.ptr, 200, st))
        call(st)
        out = call.result()[0]
        k, v = x[:, heads * hd:(heads + kvh) * hd], x[:, (heads + kvh) * hd:]
        rq, pk, pv, live, touched = _appended(sc, sc.q, k, v, cos, sin, "adjacent", 200)
        # the pools and queries as the call left them carry on
        sc.k32 = call.k.numpy().astype(np.float32)
        sc.v32 = call.v.numpy().astype(np.float32)
        assert (np.abs(sc.k32[touched] - pk[touched]) <= 2.0 ** -11 * np.abs(pk[touched]) * 1.01 + 2.0 ** -20).all()
        sc.q = call.q.numpy().reshape(sc.total, -1)
        ref = _check(sc, out)
        tokens = np.arange(sc.total) % 7
        lp, ent, ids, tlp = ops.token_logprobs(out, tokens, top=3)
        rlp, rent, rids, rtlp = logprobs(out.astype(np.float64), tokens, 3)
        assert np.array_equal(ids, rids)
        for a, b in ((lp, rlp), (ent, rent), (tlp, rtlp)):
            assert np.abs(a - b).max() <= 1e-5


@pytest.mark.parametrize("dtype,heads,kvh,prefix", [("f16", 8, 2, 0), ("bf16", 8, 2, 40), ("f32", 4, 4, 20), ("f16", 160, 160, 0)])
def test_a_captured_step(gpu, dtype, heads, kvh, prefix):
    """Append, attention and scoring captured once and replayed with other
    rows per sequence and lengths, eager calls of the same between the replays."""
    hd = 32
    sc = Scene([0] * 4, [prefix + n for n in (900, 60, 300, 90)], heads, kvh, hd, 16, dtype, prefix=prefix, seed=31, behind=70)
    width = (heads + 2 * kvh) * hd
    cos, sin = _tables(hd, prefix + 900, seed=2)
    dc, ds = buffer(cos), buffer(sin)
    tokens = np.arange(sc.total) % 11

    class Step:
        def __init__(self):
            self.call, self.x, self.tokens = Call(gpu, sc), filled((sc.total, width), 0.0), buffer(tokens.astype(np.uint32))
            self.lp, self.ent = filled(sc.total, 0.0), filled(sc.total, 0.0)
            self.ids, self.tlp = filled((sc.total, 5), 0, np.uint32), filled((sc.total, 5), 0.0)
            self.need = gpu.lib().yl_token_logprobs_workspace(sc.total, heads * hd, 5)
            self.space = bytes_of(self.need, 255)

        def set(self, x):
            self.x.upload(x)
            self.call.put_q(x[:, :heads * hd])
            self.call.kv_len.upload(np.array(sc.lens, np.uint32))
            self.call.starts.upload(sc.starts)
            self.call.out.upload(np.full(self.call.out.shape, 7.0, np.float32))

        def __call__(self, stream=None):
            c, at = self.call, self.x.ptr
            gpu.check(gpu.lib().yl_paged_append(C.byref(c.cache), C.byref(c.batch), heads, c.q.ptr, heads * hd, at, width,
                                                at + 4 * heads * hd, width, at + 4 * (heads + kvh) * hd, width,
                                                gpu.ROPE_PAIRS["half"], dc.ptr, ds.ptr, prefix + 900, stream))
            c(stream)
            gpu.check(gpu.lib().yl_token_logprobs(c.out.ptr, 0, sc.total, heads * hd, heads * hd, self.tokens.ptr, self.lp.ptr,
                                                  self.ent.ptr, 5, self.ids.ptr, self.tlp.ptr, self.space.ptr, self.need, stream))

        def results(self):
            gpu.check(gpu.lib().yl_synchronize())
            return [b.numpy().copy() for b in (self.call.out, self.call.q, self.call.k, self.call.v, self.lp, self.ent, self.ids, self.tlp)]

    captured, eager = Step(), Step()
    graph = Graph(captured)
    for rows, own in ([1, 20, 33, 6], [900, 60, 300, 90]), ([1, 1, 1, 1], [850, 30, 299, 1]), ([3, 0, 60, 7], [700, 10, 60, 90]), \
                     ([70, 0, 0, 0], [70, 0, 5, 1]), ([0, 35, 0, 35], [1, 60, 1, 80]):
        sc.rows, sc.lens = rows, [prefix + n for n in own]
        sc.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32)
        x = sc.rng.standard_normal((sc.total, width), np.float32)
        for step in (captured, eager):
            step.set(x)
        graph.replay()
        eager()
        a, b = captured.results(), eager.results()
        for p, q in zip(a, b):
            assert np.array_equal(p.view(np.uint8), q.view(np.uint8))
        out, q = a[0].reshape(sc.total, -1), a[1].reshape(sc.total, -1)
        n = sum(rows)
        sc.q = q
        sc.k32, sc.v32 = widened(a[2]).astype(np.float32), widened(a[3]).astype(np.float32)
        ref, bound = sc.attention()
        assert (np.abs(out[:n] - ref[:n]) <= bound[:n]).all() and (out[n:] == 7.0).all()
        pos = np.concatenate([np.arange(m - r, m) for r, m in zip(rows, sc.lens)])
        assert np.abs(q[:n] - rotated(x[:n, :heads * hd], cos, sin, pos, "half", heads, hd).reshape(n, -1)).max() <= 6 * 2.0 ** -24 * np.abs(x).max()
        assert np.array_equal(q[n:], x[n:, :heads * hd])
        rlp, rent, rids, rtlp = logprobs(out.astype(np.float64), tokens, 5)
        assert np.array_equal(a[6], rids)
        for got, want in zip((a[4], a[5], a[7]), (rlp, rent, rtlp)):
            assert np.abs(got - want).max() <= 1e-5
