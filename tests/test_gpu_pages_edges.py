"""Corners of the operators on pages and logits: batches that are not divided, as
many kv heads as there may be, tables wider than their pool or empty, captured
calls that share a workspace, streams side by side, offsets past 32 bits."""
import ctypes as C

import numpy as np
import pytest

from hip_rt import Graph, Stream, buffer, filled
from mx_np import MxScene
from pages_np import Pages
from paged_np import widened
from test_gpu_logit_rules import Rows
from test_gpu_paged import Call, _check
from test_gpu_pages import Device, _made, _model_step, _pool, _same, _tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kvh,hd", [(2, 1, 32), (4, 1, 64), (3, 1, 128), (8, 2, 64), (8, 1, 64)])
def test_more_sequences_than_are_divided(gpu, heads, kvh, hd):
    """Beyond 512 sequences one of 900 positions is walked as a whole, whatever the others have."""
    rng = np.random.default_rng(hd)
    lens = [900] + [int(x) for x in rng.integers(0, 40, 530)]
    sc = MxScene([1] * len(lens), lens, heads, kvh, hd, 16, spread=1.0, seed=hd)
    call = Call(gpu, sc, single=True)
    call()
    _check(sc, call.result()[0])


@pytest.mark.parametrize("kvh,single", [(1024, True), (256, True), (1024, False)])
def test_as_many_heads_as_there_may_be(gpu, kvh, single):
    sc = MxScene([1, 1, 1] if single else [2, 1, 5], [70, 1, 16], 1024, kvh, 32, 16, seed=kvh)
    call = Call(gpu, sc, single=single)
    call()
    _check(sc, call.result()[0])


@pytest.mark.parametrize("hd,power", [(64, 40), (64, -40), (128, 100), (128, -100)])
@pytest.mark.parametrize("seqs", [3, 70])
def test_large_keys_where_queries_are_zero(gpu, hd, power, seqs):
    """Queries of 2^40 or 2^100, or so much smaller, in one half of a head, keys of 2^120 in the other and of zero in the first: all scores are
    zero, whatever the scales multiply to."""
    sc = MxScene([1] * seqs, [700] + [90] * (seqs - 1), 4, 2, hd, 16, seed=9)
    q = sc.q.reshape(seqs, 4, hd)
    q[..., :hd // 2] *= np.float32(2.0 ** power)
    q[..., hd // 2:] = 0.0
    sc.k32[..., :hd // 2] *= 0.0
    sc.k32[..., hd // 2:] *= np.float32(2.0 ** 120)
    sc.k32[~np.isfinite(sc.k32)] = np.nan                # (slots that nothing holds)
    sc.settle()
    call = Call(gpu, sc, single=True)
    call()
    _check(sc, call.result()[0])


@pytest.mark.parametrize("prefix", [0, 40])
def test_captured_calls_share_a_workspace(gpu, prefix):
    """Single rows and prompts in graphs of their own over the workspace of the larger one, replayed in turn."""
    ones = MxScene([1] * 5, [prefix + n for n in (2000, 900, 3, 64, 700)], 8, 2, 64, 16, prefix=prefix, seed=1)
    rows = MxScene([60, 1, 7], [prefix + n for n in (800, 1500, 30)], 8, 2, 64, 16, prefix=prefix, seed=2)
    calls = [Call(gpu, ones, single=True), Call(gpu, rows)]
    large = max(calls, key=lambda c: c.need)
    for c in calls:
        c.space, c.need = large.space, large.need
    graphs = [Graph(c) for c in calls]
    for _ in range(3):
        for g, c, sc in zip(graphs, calls, (ones, rows)):
            sc.q = sc.rng.standard_normal(sc.q.shape).astype(np.float32)
            c.put_q(sc.q)
            g.replay()
            _check(sc, c.result()[0])


def test_attention_on_streams_side_by_side(gpu):
    scenes = [MxScene([1] * 40, [300 + 40 * i for i in range(40)], 8, 2, 128, 16, seed=1), MxScene([200, 30], [900, 2000], 8, 2, 64, 16, seed=2)]
    calls, streams = [Call(gpu, scenes[0], single=True), Call(gpu, scenes[1])], [Stream() for _ in scenes]
    gpu.check(gpu.lib().yl_synchronize())
    for _ in range(5):
        for c, st in zip(calls, streams):
            c(st.handle)
    for c, sc in zip(calls, scenes):
        _check(sc, c.result()[0])


@pytest.mark.parametrize("refs", [[0, 3, 0, 2, 1], [1] * 5, [0] * 5])
def test_compact_of_tables_wider_than_their_pool(gpu, refs):
    """Far more entries than pages to move: every one is rewritten, those of free pages and of none stay."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(3)
    table = rng.integers(-2, 8, (50, 3001))
    layers = [tuple(_pool(rng, "mxfp4", 5, 1, 16, 32) for _ in range(2))]
    m = Pages(table, np.zeros(50), refs, 16, layers, prefix=17, prefix_pages=[4, 1])
    t = _tables(ops, m)
    used, got = ops.paged_compact(t, m.layers)
    assert used == m.compact()
    _same(t, m, got)


def test_pools_whose_workgroups_look_through_more_pages(gpu):
    """Beyond 2^20 pages a workgroup has more than one stretch of them; used pages in all parts of the pool."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(5)
    n_pages = 1100000
    pool = rng.integers(0, 256, (n_pages, 1, 16, 17)).astype(np.uint8)
    used = rng.choice(n_pages, 400, replace=False)
    table, refs = np.full((20, 40), -1), np.zeros(n_pages, int)
    table[:10] = used.reshape(10, 40)
    refs[used] = 1
    lens = np.where(np.arange(20) < 10, 640 - 7 * np.arange(20), 0)
    m = Pages(table, lens, refs, 16, [(pool, pool[::-1])])
    parents, children = np.arange(10), 10 + rng.permutation(10)
    t = _tables(ops, m)
    lacking, got = ops.paged_fork(t, m.layers, parents, children)
    assert lacking == m.fork(parents, children) == 0
    _same(t, m, got)
    ops.paged_release(t, [3, 8, 14])
    m.release([3, 8, 14])
    count, got = ops.paged_compact(t, got)
    assert count == m.compact()
    _same(t, m, got)


@pytest.mark.parametrize("rows,entries", [(0, 4), (3, 0), (0, 0)])
def test_tables_of_nothing(gpu, rows, entries):
    """No sequences, or no entries: ids name nothing, lengths are within the prefix or lack."""
    from yallma3_mini_inference_amd import ops
    rng = np.random.default_rng(4)
    layers = [tuple(_pool(rng, "f16", 3, 1, 16, 32) for _ in range(2))]
    m = Pages(np.full((rows, entries), -1), np.zeros(rows), [0, 0, 1], 16, layers, prefix=9, prefix_pages=[2])
    t = _tables(ops, m)
    want = np.array([0, 9, 10][:rows])
    assert ops.paged_reserve(t, want) == m.reserve(want)
    _same(t, m)
    lacking, got = ops.paged_fork(t, m.layers, [0, 1], [2, 7])
    assert lacking == m.fork([0, 1], [2, 7]) == 0
    _same(t, m, got)
    lacking, got = ops.paged_fork(t, m.layers, [], [])
    assert lacking == 0
    ops.paged_release(t, [0, 5])
    m.release([0, 5])
    ops.paged_release(t, [])
    _same(t, m, got)
    used, got = ops.paged_compact(t, m.layers)
    assert used == m.compact() == 1
    _same(t, m, got)


def test_captured_steps_share_a_workspace(gpu):
    """Two pools, a large and a small one, whose captured steps use one workspace in turn."""
    sizes = [(60, 16), (3000, 90)]
    devices = [Device(gpu, _made(np.random.default_rng(i), [70, 33, 16, 5], rows, 8, n, 16,
                                 [tuple(_pool(np.random.default_rng(i + k), "f16", n, 2, 16, 32) for k in range(2))]), "f16", 32, 6)
               for i, (n, rows) in enumerate(sizes)]
    devices[0].space, devices[0].need = devices[1].space, devices[1].need
    graphs = [Graph(d.step) for d in devices]
    rng = np.random.default_rng(1)
    for k in range(2):
        for d, g in zip(devices, graphs):
            rows = len(d.m.kv_len)
            parents, children = rng.integers(0, 4, 6), 4 + 6 * k + np.arange(6)
            want = np.where(np.arange(rows) < 4, 0, np.where(np.arange(rows) < 10 + 6 * k, 100, 0))
            d.parents.upload(parents.astype(np.uint32))
            d.children.upload(children.astype(np.uint32))
            d.want.upload(want.astype(np.uint32))
            g.replay()
            d.compare(_model_step(d.m, parents, children, want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_logits_beyond_32_bits(gpu, dtype):
    """Rows so far apart that their elements lie past 2^31, in place."""
    w = Rows(3, 5003, dtype, seed=11)
    ld, size = (1 << 31) + 5 if dtype == "bf16" else (1 << 30) + 3, w.x.itemsize
    big, host = gpu.DeviceBuffer((2 * ld + w.vocab) * size), buffer(w.x)
    for r in range(3):
        gpu.check(gpu.lib().yl_memcpy_d2d(big.ptr + r * ld * size, host.ptr + r * w.vocab * size, w.vocab * size))
    starts = lambda lists: np.cumsum([0] + [len(x) for x in lists]).astype(np.uint32)  # noqa: E731
    ids = [b[0] for b in w.biases]
    h = [buffer(a) for a in (np.concatenate(w.tokens), starts(w.tokens), w.n_prompt, w.repetition, w.presence, w.frequency, np.concatenate(ids),
                             np.concatenate([b[1] for b in w.biases]), starts(ids), w.mask, w.mask_of)]
    rules = gpu.LogitRules(h[0].ptr, h[1].ptr, h[2].ptr, sum(map(len, w.tokens)), *[x.ptr for x in h[3:9]], sum(map(len, ids)), h[9].ptr, w.mask.shape[1],
                           len(w.mask), h[10].ptr)
    gpu.check(gpu.lib().yl_adjust_logits(big.ptr, ld, big.ptr, ld, gpu.DTYPES[dtype], 3, w.vocab, C.byref(rules), None))
    out = filled(w.x.shape, 0, w.x.dtype)
    for r in range(3):
        gpu.check(gpu.lib().yl_memcpy_d2d(out.ptr + r * w.vocab * size, big.ptr + r * ld * size, w.vocab * size))
    gpu.check(gpu.lib().yl_synchronize())
    w.check(out.numpy(), **w.rules())
    assert not np.array_equal(widened(out.numpy()), widened(w.x))
