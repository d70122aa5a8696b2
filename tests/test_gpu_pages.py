"""yl_paged_reserve, _fork, _release, _compact and _copy against the same
operations entry by entry: tables, lengths, references and every byte of the
pools, exactly."""
import ctypes as C

import numpy as np
import pytest

from hip_rt import Graph, Stream, buffer, bytes_of, filled
from mx_np import MxScene
from pages_np import Pages
from paged_np import Scene

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16", "mxfp4"]


def _pool(rng, dtype, n_pages, kvh, page, hd):
    if dtype == "mxfp4":
        return rng.integers(0, 256, (n_pages, kvh, page, 17 * hd // 32)).astype(np.uint8)
    if dtype == "f32":
        return rng.standard_normal((n_pages, kvh, page, hd)).astype(np.float32)
    return rng.integers(0, 0x7800, (n_pages, kvh, page, hd)).astype(np.uint16).view(np.float16 if dtype == "f16" else np.uint16)


def _made(rng, lens, rows, entries, n_pages, page, layers=(), prefix=0):
    """Sequences of these lengths (rows of the table beyond them are free), a few pages named twice."""
    order = rng.permutation(n_pages)
    shared = -(-prefix // page)
    table, refs, at = np.full((rows, entries), -1), np.zeros(n_pages, int), shared
    refs[order[:shared]] = 1
    for s, n in enumerate(lens):
        need = min(entries, -(-max(0, n - prefix) // page))
        table[s, :need] = order[at:at + need]
        at += need
    assert at <= n_pages
    if len(lens) > 1 and lens[0] - prefix >= page and lens[1] - prefix >= page:
        table[1, 0] = table[0, 0]
    for e in table[table >= 0]:
        refs[e] += 1
    kv_len = np.zeros(rows, int)
    kv_len[:len(lens)] = lens
    return Pages(table, kv_len, refs, page, layers, prefix, order[:shared])


def _tables(ops, m):
    return ops.PagedTables(m.table.copy(), m.kv_len.copy(), m.refs.copy(), m.page, m.prefix, m.prefix_pages.copy() if m.prefix else None)


def _same(t, m, layers=None):
    assert np.array_equal(t.page_table, m.table)
    assert np.array_equal(t.kv_len, m.kv_len)
    assert np.array_equal(t.refs, m.refs)
    if m.prefix:
        assert np.array_equal(t.prefix_pages, m.prefix_pages)
    for got, want in zip(layers or [], m.layers):
        for a, b in zip(got, want):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kvh,page,hd", [(2, 16, 32), (3, 32, 64), (1, 256, 128), (8, 16, 64)])
@pytest.mark.parametrize("prefix", [0, 21])
def test_fork(gpu, dtype, kvh, page, hd, prefix):
    """Lengths of nothing, inside the prefix, one slot, one less than a page, whole pages, past the table; several branches of one parent."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(page + hd)
    lens = [prefix + n for n in (2 * page + 3, page, page - 1, 1, 0, 3 * page + page // 2)] + [prefix // 2, prefix + 9 * page]
    n = len(lens)
    layers = [tuple(_pool(rng, dtype, 40, kvh, page, hd) for _ in range(2)) for _ in range(3)]
    m = _made(rng, lens, n + 14, 4, 40, page, layers, prefix)
    m.refs[m.table[5, 1]] -= 1
    m.table[5, 1] = 99                        # an entry that names no page
    parents = list(range(n)) + [0, 0, 3, 5, 900, 2]
    children = list(range(n, n + 12)) + [n, 2]               # 900: no sequence; (2, 2): the same one twice
    t = _tables(ops, m)
    m.check()
    lacking, got = ops.paged_fork(t, m.layers, parents, children)
    assert lacking == m.fork(parents, children) == 0
    _same(t, m, got)
    m.check()


def test_fork_of_more_pages_than_there_are(gpu):
    """The first children are served; the others' rows are empty and their parents' references as they were."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(3)
    layers = [tuple(_pool(rng, "f16", 12, 2, 16, 32) for _ in range(2))]
    m = _made(rng, [37, 50, 16], 20, 4, 12, 16, layers)
    free = len(m.free())
    parents, children = [0, 1, 2] * 5, list(range(3, 18))
    t = _tables(ops, m)
    lacking, got = ops.paged_fork(t, m.layers, parents, children)
    assert lacking == m.fork(parents, children) == 10 - free > 0
    _same(t, m, got)
    m.check()


@pytest.mark.parametrize("n_pages", [1, 63, 1024, 1025, 5000, 1100000])
@pytest.mark.parametrize("full", [False, True])
def test_reserve(gpu, n_pages, full):
    """Pools around the shares of a workgroup; the free pages last, or scattered; more wanted than there is."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(n_pages)
    refs = (np.arange(n_pages) < n_pages - min(n_pages, 40)).astype(int) if full else rng.integers(-1, 2, n_pages)
    table = np.full((70, 9), -1)
    table[3, 1] = n_pages
    table[4, 0] = 0x7FFFFFFF
    m = Pages(table, np.zeros(70), refs, 32)
    if n_pages > 1000:                        # entries that are there stay
        held = rng.choice(n_pages, 100, replace=False)
        m.table.reshape(-1)[rng.choice(630, 100, replace=False)] = held
        m.refs[held] = 1
    for want in (rng.integers(0, 200, 70), rng.integers(100, 400, 70), np.full(70, 0xFFFFFFFF)):
        t = _tables(ops, m)
        assert ops.paged_reserve(t, want) == m.reserve(want)
        _same(t, m)


@pytest.mark.parametrize("entries", [0, 1, 63, 64, 65, 300])
def test_reserve_of_wide_tables(gpu, entries):
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(entries)
    table = np.where(rng.random((5, entries)) < 0.5, -1, rng.permutation(5 * entries).reshape(5, entries))
    refs = np.zeros(3000, int)
    refs[table[table >= 0]] = 1
    m = Pages(table, np.zeros(5), refs, 16, prefix=5, prefix_pages=[2999])
    m.refs[2999] = 1
    want = np.array([0, 3, 16 * entries + 5, 16 * entries + 6, 8 * entries + 1])
    t = _tables(ops, m)
    assert ops.paged_reserve(t, want) == m.reserve(want) == (want[3] > 16 * entries + 5)
    _same(t, m)


def test_release(gpu):
    """Sequences that are there twice, empty ones, ids that are none; pages that others still name stay in use."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(5)
    m = _made(rng, [40, 33, 700, 0, 5], 7, 50, 60, 16)
    m.table[2, 7] = -7
    seqs = [1, 2, 1, 6, 7, 0xFFFFFFFF, 3]
    t = _tables(ops, m)
    ops.paged_release(t, seqs)
    m.release([1, 2, 6, 3])
    _same(t, m)
    assert (m.refs >= 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n_pages,prefix", [(60, 0), (60, 37), (39, 0), (1300, 21), (3000, 0)])
def test_compact(gpu, dtype, n_pages, prefix):
    """Pools that are nearly empty, half full and full; a page that two sequences name; then again, when nothing moves."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(n_pages)
    layers = [tuple(_pool(rng, dtype, n_pages, 2, 16, 32) for _ in range(2)) for _ in range(2)]
    m = _made(rng, [prefix + n for n in (100, 230, 16, 1, 0, 240)], 8, 16, n_pages, 16, layers, prefix)
    m.table[3, 5] = n_pages + 4
    m.check()
    for _ in range(2):
        t = _tables(ops, m)
        used, got = ops.paged_compact(t, m.layers)
        assert used == m.compact()
        _same(t, m, got)
        m.check()
        assert (m.refs[:used] > 0).all() and not (m.refs[used:] > 0).any()
        m.release([0, 2])


@pytest.mark.parametrize("refs", [[0], [1], [0, 0, 0], [1, 2, 1], [0, 0, 5], [3, 0, 0], [-1, 2, -1, 1]])
def test_compact_of_few_pages(gpu, refs):
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(0)
    layers = [tuple(_pool(rng, "f16", len(refs), 1, 16, 32) for _ in range(2))]
    m = Pages([[len(refs) - 1, 0, -1]], [5], refs, 16, layers)      # (entries may name free pages: they stay)
    t = _tables(ops, m)
    used, got = ops.paged_compact(t, m.layers)
    assert used == m.compact()
    _same(t, m, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers", [1, 5, 70])
def test_copy(gpu, dtype, layers):
    """Between pools of other numbers of pages, and within one; pairs that name no page."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(layers)
    a = [tuple(_pool(rng, dtype, 9, 2, 16, 32) for _ in range(2)) for _ in range(layers)]
    b = [tuple(_pool(rng, dtype, 30, 2, 16, 32) for _ in range(2)) for _ in range(layers)]
    dst, src = [3, 0, -1, 9, 8, 2], [29, 4, 5, 6, 30, 4]
    got = ops.paged_copy(a, b, dst, src)
    for (x, y), (p, q) in zip(zip(a, b), zip(got, got)):
        for old, new, other in zip(x, p, y):
            want = old.copy()
            want[[3, 0, 2]] = other[[29, 4, 4]]
            assert np.array_equal(new.view(np.uint8), want.view(np.uint8))
    got = ops.paged_copy(a, None, [1, 2], [5, 5])
    for x, p in zip(a, got):
        for old, new in zip(x, p):
            want = old.copy()
            want[[1, 2]] = old[5]
            assert np.array_equal(new.view(np.uint8), want.view(np.uint8))


def test_pools_beyond_32_bits(gpu):
    """Pages whose bytes lie past 2^32."""
    kvh, page, hd = 8, 256, 128
    size = kvh * page * hd * 4
    n_pages = (1 << 32) // size + 6
    rng = np.random.default_rng(1)
    big = [gpu.DeviceBuffer(n_pages * size) for _ in range(2)]
    src = _pool(rng, "f32", 1, kvh, page, hd)
    at = n_pages - 2
    for b in big:
        gpu.check(gpu.lib().yl_memcpy_h2d(b.ptr + at * size, src.ctypes.data, size))
    cache = gpu.PagedCacheDesc(big[0].ptr, big[1].ptr, 0, n_pages, page, kvh, hd)
    refs = np.zeros(n_pages, np.int32)
    refs[at] = 1
    refs[:at] = (np.arange(at) < 3)                  # the first free page is 3
    table, kv_len = buffer(np.array([[at, -1], [-1, -1]], np.int32)), buffer(np.array([100, 0], np.uint32))
    drefs, par, chi, used = buffer(refs), buffer(np.array([0], np.uint32)), buffer(np.array([1], np.uint32)), filled(1, 0, np.uint32)
    t = gpu.PagedTablesDesc(2, 2, n_pages, page, table.ptr, kv_len.ptr, drefs.ptr, 0, None)
    L = gpu.lib()
    need = L.yl_paged_tables_workspace(C.byref(t), 1)
    space = bytes_of(need, 255)
    gpu.check(L.yl_paged_fork(C.byref(t), C.byref(cache), 1, par.ptr, chi.ptr, 1, None, space.ptr, need, None))
    gpu.check(L.yl_paged_compact(C.byref(t), C.byref(cache), 1, used.ptr, space.ptr, need, None))
    gpu.check(L.yl_synchronize())
    assert int(used.numpy()[0]) == 5 and np.array_equal(table.numpy(), [[4, -1], [3, -1]])
    got = np.empty_like(src)
    for b in big:
        gpu.check(L.yl_memcpy_d2h(got.ctypes.data, b.ptr + 4 * size, size))
        assert np.array_equal(got, src)
        gpu.check(L.yl_memcpy_d2h(got.ctypes.data, b.ptr + 3 * size, size))
        assert np.array_equal(got[:, :, :100], src[:, :, :100])


class Device:
    """Tables and pools on the device, as a program keeps them."""

    def __init__(self, yl, m, dtype, hd, forks):
        self.yl, self.m = yl, m
        self.table, self.kv_len, self.refs = buffer(m.table), buffer(m.kv_len.astype(np.uint32)), buffer(m.refs)
        self.pools = [tuple(buffer(x) for x in l) for l in m.layers]
        kvh = m.layers[0][0].shape[1]
        self.caches = (yl.PagedCacheDesc * len(self.pools))(*[
            yl.PagedCacheDesc(k.ptr, v.ptr, yl.DTYPES[dtype], len(m.refs), m.page, kvh, hd) for k, v in self.pools])
        self.t = yl.PagedTablesDesc(*m.table.shape, len(m.refs), m.page, self.table.ptr, self.kv_len.ptr, self.refs.ptr, 0, None)
        self.need = yl.lib().yl_paged_tables_workspace(C.byref(self.t), forks)
        self.space, self.lacking = bytes_of(self.need, 255), filled(3, 77, np.uint32)
        self.parents, self.children, self.want = (filled(forks, 0, np.uint32) for _ in range(2)), None, None
        self.parents, self.children = (filled(forks, 0, np.uint32) for _ in range(2))
        self.want = filled(m.table.shape[0], 0, np.uint32)
        self.forks = forks

    def step(self, stream=None):
        """Last step's branches end, new ones are made and get room, the pool is compacted."""
        L, n, lack = self.yl.lib(), self.forks, self.lacking.ptr
        self.yl.check(L.yl_paged_release(C.byref(self.t), self.children.ptr, n, stream))
        self.yl.check(L.yl_paged_fork(C.byref(self.t), self.caches, len(self.caches), self.parents.ptr, self.children.ptr, n, lack, self.space.ptr, self.need, stream))
        self.yl.check(L.yl_paged_reserve(C.byref(self.t), self.want.ptr, lack + 4, self.space.ptr, self.need, stream))
        self.yl.check(L.yl_paged_compact(C.byref(self.t), self.caches, len(self.caches), lack + 8, self.space.ptr, self.need, stream))

    def compare(self, lacking):
        self.yl.check(self.yl.lib().yl_synchronize())
        m = self.m
        assert list(self.lacking.numpy()) == lacking
        assert np.array_equal(self.table.numpy(), m.table) and np.array_equal(self.kv_len.numpy(), m.kv_len) and np.array_equal(self.refs.numpy(), m.refs)
        for got, want in zip(self.pools, m.layers):
            for a, b in zip(got, want):
                assert np.array_equal(a.numpy().view(np.uint8), b.view(np.uint8))


def _model_step(m, parents, children, want):
    m.release(children)
    return [m.fork(parents, children), m.reserve(want), m.compact()]


@pytest.mark.parametrize("dtype,hd", [("f16", 32), ("mxfp4", 64)])
def test_captured_steps(gpu, dtype, hd):
    """A step of all operations captured once and replayed with other branches and lengths, an eager step of another pool between the replays."""
    rng = np.random.default_rng(9)
    make = lambda: _made(np.random.default_rng(8), [70, 33, 16, 5], 16, 8, 60, 16,  # noqa: E731
                         [tuple(_pool(np.random.default_rng(7 + i), dtype, 60, 2, 16, hd) for i in range(2)) for _ in range(2)])
    captured, eager = Device(gpu, make(), dtype, hd, 6), Device(gpu, make(), dtype, hd, 6)
    graph = Graph(captured.step)
    for k in range(6):
        parents, children = rng.integers(0, 4, 6), 4 + rng.permutation(12)[:6]
        if k == 3:
            parents[2] = 99
        want = np.where(np.arange(16) < 4, 0, rng.integers(60, 128, 16))
        for d in (captured, eager):
            d.parents.upload(parents.astype(np.uint32))
            d.children.upload(children.astype(np.uint32))
            d.want.upload(want.astype(np.uint32))
        graph.replay()
        eager.step()
        for d in (captured, eager):
            # (rows that this step does not fork keep what earlier steps reserved)
            d.compare(_model_step(d.m, parents, children, want))
        m = eager.m
        if k % 2:
            rest = [s for s in range(4, 16)]
            for d in (captured, eager):
                d.m.release(rest)
                d.table.upload(d.m.table)
                d.kv_len.upload(d.m.kv_len.astype(np.uint32))
                d.refs.upload(d.m.refs)


def test_streams_side_by_side(gpu):
    """Two pools on streams of their own, each with its workspace."""
    devices = [Device(gpu, _made(np.random.default_rng(i), [300, 33, 90], 9, 40, 300, 16,
                                 [tuple(_pool(np.random.default_rng(i), "f16", 300, 4, 16, 64) for _ in range(2))]), "f16", 64, 4) for i in range(2)]
    streams = [Stream() for _ in devices]
    parents, children, want = [0, 1, 2, 0], [3, 4, 5, 6], np.array([0] * 3 + [400] * 6)
    for d in devices:
        d.parents.upload(np.array(parents, np.uint32))
        d.children.upload(np.array(children, np.uint32))
        d.want.upload(want.astype(np.uint32))
    gpu.check(gpu.lib().yl_synchronize())
    for _ in range(3):
        for d, st in zip(devices, streams):
            d.step(st.handle)
    for d in devices:
        for _ in range(3):
            lacking = _model_step(d.m, parents, children, want)
        d.compare(lacking)


@pytest.mark.parametrize("dtype", ["f16", "mxfp4"])
def test_branches_attend_as_their_parents(gpu, dtype):
    """A fork of every conversation, each branch with one more position of its own, then everything moved: the attention sees
    each branch's own history."""
    from yallma3_mini_inference_amd import ops
    heads, kvh, hd, page = 4, 2, 64, 16
    lens = [37, 16, 50, 1]
    n, b = len(lens), 3
    args = ([1] * n, lens, heads, kvh, hd, page)
    base = MxScene(*args, seed=3, spare=60) if dtype == "mxfp4" else Scene(*args, dtype, seed=3, spare=60)
    table = np.full((n * (1 + b), 5), -1, np.int32)
    table[:n, :base.table.shape[1]] = base.table
    refs = np.zeros(base.n_pages, np.int32)
    refs[table[table >= 0]] = 1
    t = ops.PagedTables(table, np.array(lens + [0] * n * b), refs, page)
    parents, children = np.repeat(np.arange(n), b), np.arange(n, n * (1 + b))
    lacking, layers = ops.paged_fork(t, [tuple(base.pools())], parents, children)
    assert lacking == 0
    want = t.kv_len.copy()
    want[n:] += 1
    assert ops.paged_reserve(t, want) == 0
    rng = np.random.default_rng(4)
    rows = n * b
    q, k, v = (rng.standard_normal((rows, m * hd), np.float32) for m in (heads, kvh, kvh))
    batch = ops.PagedBatch(t.page_table[n:], want[n:])
    q2, *pools = ops.paged_append(*layers[0], batch, q, k, v, heads)
    out = ops.paged_attention(*pools, batch, q2, heads, base.scale)
    # every branch alone, its history gathered from its parent's own pages
    ref_batch = ops.PagedBatch(base.table, np.array(lens), np.cumsum([0] + lens))
    hk, hv = ops.paged_gather(*base.pools(), ref_batch, sum(lens))
    starts = np.cumsum([0] + lens)
    for i in range(rows):
        p = parents[i]
        kk, vv = ops.paged_gather(*pools, ops.PagedBatch(t.page_table[n + i:n + i + 1], want[n + i:n + i + 1], np.array([0, want[n + i]])), int(want[n + i]))
        assert np.array_equal(kk[:-1], hk[starts[p]:starts[p + 1]]) and np.array_equal(vv[:-1], hv[starts[p]:starts[p + 1]])
        for h in range(heads):
            g = h // (heads // kvh)
            sc = kk[:, g * hd:(g + 1) * hd].astype(np.float64) @ q[i, h * hd:(h + 1) * hd].astype(np.float64) * base.scale
            w = np.exp(sc - sc.max())
            ref = w @ vv[:, g * hd:(g + 1) * hd] / w.sum()
            # (scores of some units over up to 51 positions: the bound of f32 sums is some 300 U of the largest value)
            assert np.abs(out[i, h * hd:(h + 1) * hd] - ref).max() <= 300 * 2.0 ** -24 * np.abs(vv).max()
    ops.paged_release(t, np.arange(n))
    used, moved = ops.paged_compact(t, [tuple(pools)])
    assert used == len(set(t.page_table[t.page_table >= 0])) < base.n_pages and t.page_table.max() == used - 1
    again = ops.paged_attention(*moved[0], ops.PagedBatch(t.page_table[n:], want[n:]), q2, heads, base.scale)
    assert np.array_equal(again, out)


@pytest.mark.parametrize("n_pages", [1, 1023, 1024, 1025, 4096, 4097, 16384, 16385, 40000])
def test_forks_and_moves_in_pools_of_any_size(gpu, n_pages):
    """Both sides of the sizes from which on pools are looked through in another way; the free pages scattered."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(n_pages)
    used = rng.permutation(n_pages)[:n_pages // 2]
    table = np.full((12, max(1, len(used) // 6)), -1)
    lens = np.zeros(12, int)
    refs = np.zeros(n_pages, int)
    for s, pages in enumerate(np.array_split(used, 6)):
        pages = pages[:table.shape[1]]
        table[s, :len(pages)] = pages
        refs[pages] = 1
        lens[s] = max(0, 16 * len(pages) - s * 3)
    layers = [(rng.integers(0, 1 << 15, (n_pages, 1, 16, 32)).astype(np.uint16).view(np.float16), rng.integers(0, 1 << 15, (n_pages, 1, 16, 32)).astype(np.uint16).view(np.float16))]
    m = Pages(table, lens, refs, 16, layers)
    parents, children = [0, 1, 2, 3, 4, 5], [6, 7, 8, 9, 10, 11]
    t = _tables(ops, m)
    lacking, got = ops.paged_fork(t, m.layers, parents, children)
    assert lacking == m.fork(parents, children)
    _same(t, m, got)
    ops.paged_release(t, [1, 4, 9])
    m.release([1, 4, 9])
    used, got = ops.paged_compact(t, got)
    assert used == m.compact()
    _same(t, m, got)


@pytest.mark.parametrize("n", [1, 1024, 1025, 5000])
def test_many_forks(gpu, n):
    """More children than threads look at one each; not pages enough for all."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(n)
    n_pages = 3 * n // 2 + 3
    layers = [tuple(_pool(rng, "f16", n_pages, 1, 16, 32) for _ in range(2))]
    m = _made(rng, [16 * (1 + i % 3) + i % 16 for i in range(max(1, n // 5))], n // 5 + 1 + n, 4, n_pages, 16, layers)
    parents = rng.integers(0, max(1, n // 5), n)
    children = max(1, n // 5) + rng.permutation(n)
    t = _tables(ops, m)
    lacking, got = ops.paged_fork(t, m.layers, parents, children)
    assert lacking == m.fork(parents, children)
    _same(t, m, got)
