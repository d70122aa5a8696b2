"""Per-op entry points of the forward path on host arrays (device compute).

Each wraps one C-ABI op so tests can compare it with the reference function
it mirrors:
  rmsnorm_quantize  util::rmsnorm (util.rs:389-426) + quantize
  rope_gguf         util::rope_gguf (util.rs:653-718)
  attention         forward.rs fused_attention (forward.rs:299-400)
  swiglu_quantize   forward.rs:220-237 + quantize
  math_selftest     device exp / sqrt / division / f16 widening probes
  serial_sum_selftest  the one-wavefront exact serial f32 sum (softmax denominator)

Ops for programs that serve many conversations from one pool of cache pages
(no counterparts in the reference; yl_paged_cache and yl_paged_batch in
include/yallma3.h say what they hold):
  rope_table        the (cos, sin) tables that paged_append rotates by
  paged_append      rows' keys and values into pages, rotated on the way
  paged_gather      keys and values back out of their pages
  paged_attention   causal attention over pages, a shared prefix read once
  paged_reserve, paged_fork, paged_release, paged_compact, paged_copy
                    the pages themselves: handed out, shared by branches of a
                    conversation, given back, moved together, copied
  adjust_logits     penalties for repeated tokens, biases, grammar masks
  token_logprobs    log probabilities of tokens, entropy, top alternatives
"""
from __future__ import annotations

import ctypes as C
import dataclasses

import numpy as np

from ._lib import DTYPES, ROPE_PAIRS, LogitRules, PagedBatchDesc, PagedCacheDesc, PagedTablesDesc, RopeParams, check, lib
from .device import DeviceBuffer


def rmsnorm_quantize(x: np.ndarray, weight: np.ndarray, eps: float, qfmt: int = -1):
    """Rows of x [batch][size] -> (normalized f32, q int8 or None, scales or None)."""
    x = np.ascontiguousarray(x, np.float32)
    batch, size = (1, x.size) if x.ndim == 1 else x.shape
    dx, dw = DeviceBuffer.from_numpy(x), DeviceBuffer.from_numpy(np.ascontiguousarray(weight, np.float32))
    dn = DeviceBuffer.zeros(x.size, np.float32)
    dq = DeviceBuffer.zeros(max(1, x.size), np.int8)
    ds = DeviceBuffer.zeros(max(1, x.size // 32), np.float32)
    check(lib().yl_rmsnorm_quantize(dx.ptr, dw.ptr, size, eps, batch, dn.ptr, qfmt, dq.ptr if qfmt >= 0 else None,
                                    ds.ptr if qfmt >= 0 else None, None))
    check(lib().yl_synchronize())
    xn = dn.numpy().reshape(x.shape)
    if qfmt < 0:
        return xn, None, None
    return xn, dq.numpy()[: x.size], ds.numpy()[: x.size // 32]


def rope_gguf(params: RopeParams, q: np.ndarray, k: np.ndarray, start_pos: int, batch: int = 1):
    dq = DeviceBuffer.from_numpy(np.ascontiguousarray(q, np.float32))
    dk = DeviceBuffer.from_numpy(np.ascontiguousarray(k, np.float32))
    check(lib().yl_rope_gguf(C.byref(params), dq.ptr, dk.ptr, batch, start_pos, None))
    return dq.numpy().reshape(np.shape(q)), dk.numpy().reshape(np.shape(k))


def attention(q: np.ndarray, key_cache: np.ndarray, value_cache: np.ndarray, batch: int, start_pos: int,
              n_heads: int, n_kv_heads: int, head_size: int, attn_scale: float) -> np.ndarray:
    dq = DeviceBuffer.from_numpy(np.ascontiguousarray(q, np.float32))
    dk = DeviceBuffer.from_numpy(np.ascontiguousarray(key_cache, np.float32))
    dv = DeviceBuffer.from_numpy(np.ascontiguousarray(value_cache, np.float32))
    out = DeviceBuffer.zeros(batch * n_heads * head_size, np.float32)
    check(lib().yl_attention(out.ptr, dq.ptr, dk.ptr, dv.ptr, batch, start_pos, n_heads, n_kv_heads, head_size,
                             attn_scale, None))
    return out.numpy()


def attention_split(q: np.ndarray, key_cache: np.ndarray, value_cache: np.ndarray, start_pos: int,
                    n_heads: int, n_kv_heads: int, head_size: int, attn_scale: float) -> np.ndarray:
    """The split decode attention (one query row at start_pos): equal to
    fused_attention (forward.rs:299-400) up to rounding."""
    dq = DeviceBuffer.from_numpy(np.ascontiguousarray(q, np.float32))
    dk = DeviceBuffer.from_numpy(np.ascontiguousarray(key_cache, np.float32))
    dv = DeviceBuffer.from_numpy(np.ascontiguousarray(value_cache, np.float32))
    out = DeviceBuffer.zeros(n_heads * head_size, np.float32)
    check(lib().yl_attention_split(out.ptr, dq.ptr, dk.ptr, dv.ptr, start_pos, n_heads, n_kv_heads, head_size,
                                   attn_scale, None))
    return out.numpy()


def swiglu_quantize(gate: np.ndarray, up: np.ndarray, qfmt: int = -1):
    g = np.ascontiguousarray(gate, np.float32)
    batch, hidden = (1, g.size) if g.ndim == 1 else g.shape
    dg, du = DeviceBuffer.from_numpy(g), DeviceBuffer.from_numpy(np.ascontiguousarray(up, np.float32))
    dh = DeviceBuffer.zeros(g.size, np.float32)
    dq = DeviceBuffer.zeros(max(1, g.size), np.int8)
    ds = DeviceBuffer.zeros(max(1, g.size // 32), np.float32)
    check(lib().yl_swiglu_quantize(dg.ptr, du.ptr, hidden, batch, dh.ptr, qfmt, dq.ptr if qfmt >= 0 else None,
                                   ds.ptr if qfmt >= 0 else None, None))
    check(lib().yl_synchronize())
    h = dh.numpy().reshape(g.shape)
    if qfmt < 0:
        return h, None, None
    return h, dq.numpy()[: g.size], ds.numpy()[: g.size // 32]


def math_selftest(x: np.ndarray):
    x = np.ascontiguousarray(x, np.float32)
    dx = DeviceBuffer.from_numpy(x)
    outs = [DeviceBuffer.zeros(x.size, np.float32) for _ in range(4)]
    check(lib().yl_math_selftest(dx.ptr, x.size, *[o.ptr for o in outs]))
    return tuple(o.numpy() for o in outs)


def serial_sum_selftest(segments, piece: int = 0):
    """Device serial f32 sums ((0 + v0) + v1) + ... of each nonnegative segment
    (piece > 0: summed in consecutive pieces of that many values, each piece
    continuing from the previous one's sum; piece -1: by the decode
    attention's segmented sum over four wavefronts; piece -2: by the
    long-context softmax's wide segmented sum over eight wavefronts)."""
    segs = [np.ascontiguousarray(s, np.float32).ravel() for s in segments]
    offs = np.zeros(len(segs) + 1, np.uint32)
    offs[1:] = np.cumsum([s.size for s in segs])
    v = np.concatenate(segs) if segs else np.zeros(1, np.float32)
    dv, do = DeviceBuffer.from_numpy(v if v.size else np.zeros(1, np.float32)), DeviceBuffer.from_numpy(offs)
    out = DeviceBuffer.zeros(max(1, len(segs)), np.float32)
    check(lib().yl_serial_sum_selftest(dv.ptr, do.ptr, len(segs), int(piece) & 0xFFFFFFFF, out.ptr))
    return out.numpy()[: len(segs)]


# numpy has no bfloat16: such values travel as their bits
_DTYPE_OF = {np.dtype(np.float32): "f32", np.dtype(np.float16): "f16", np.dtype(np.uint16): "bf16"}


@dataclasses.dataclass
class PagedBatch:
    """yl_paged_batch on host arrays: page_table [seqs][entries], kv_len
    [seqs], row_start [seqs + 1] or None (one row per sequence)."""
    page_table: np.ndarray
    kv_len: np.ndarray
    row_start: np.ndarray | None = None
    prefix_len: int = 0
    prefix_pages: np.ndarray | None = None
    max_len: int = 0

    def upload(self, n_rows: int):
        """(descriptor, the device arrays it points to)"""
        table = np.ascontiguousarray(self.page_table, np.int32)
        kv_len = np.ascontiguousarray(self.kv_len, np.uint32)
        if table.ndim != 2 or table.shape[0] != kv_len.size:
            raise ValueError("page_table holds a row of entries per sequence")
        if self.row_start is not None and np.size(self.row_start) != kv_len.size + 1:
            raise ValueError("row_start holds one entry more than there are sequences")
        held = [DeviceBuffer.from_numpy(table), DeviceBuffer.from_numpy(kv_len), None, None]
        if self.row_start is not None:
            held[2] = DeviceBuffer.from_numpy(np.ascontiguousarray(self.row_start, np.uint32))
        if self.prefix_pages is not None:
            held[3] = DeviceBuffer.from_numpy(np.ascontiguousarray(self.prefix_pages, np.int32))
        ptr = [b.ptr if b is not None else None for b in held]
        return PagedBatchDesc(kv_len.size, n_rows, table.shape[1], int(self.max_len), ptr[0], ptr[1], ptr[2],
                              int(self.prefix_len), ptr[3]), held

    def check_prefix(self, page_size: int) -> None:
        if self.prefix_len and (self.prefix_pages is None or np.size(self.prefix_pages) * page_size < self.prefix_len):
            raise ValueError("prefix_pages does not reach prefix_len")


def _pool(keys, values):
    """Device copies and the descriptor of pages [n_pages][kv_heads][page_size][head_size]
    (float32, float16, or bf16 bits as uint16); uint8: MXFP4 bytes, 17 / 32 of
    head_size in the last dimension (codes and scales stand as yl_paged_cache says)."""
    keys, values = np.ascontiguousarray(keys), np.ascontiguousarray(values)
    if keys.ndim != 4 or keys.shape != values.shape or keys.dtype != values.dtype or keys.dtype not in (*_DTYPE_OF, np.uint8):
        raise ValueError("keys and values: [pages][kv_heads][page_size][head_size] of float32, float16, uint16 (bf16 bits) or uint8 (MXFP4)")
    n_pages, kvh, page, hd = keys.shape
    if keys.dtype == np.uint8:
        if hd % 17:
            raise ValueError("MXFP4 pages take 17 bytes for 32 elements")
        hd = hd // 17 * 32
    dk, dv = DeviceBuffer.from_numpy(keys), DeviceBuffer.from_numpy(values)
    return dk, dv, PagedCacheDesc(dk.ptr, dv.ptr, DTYPES[_DTYPE_OF.get(keys.dtype, "mxfp4")], n_pages, page, kvh, hd)


def _rows(x):
    """Activations [rows][width]: (device copy, pointer, floats from row to row)."""
    x = np.asarray(x, np.float32)
    if x.ndim != 2:
        raise ValueError("activations: [rows][width]")
    d = DeviceBuffer.from_numpy(x)
    return d, d.ptr, x.shape[1]


def rope_table(params: RopeParams, pairs: str, rows: int):
    """(cos, sin) [rows][head_size / 2] of positions 0 .. rows - 1 (host)."""
    cos, sin = (np.empty((rows, params.head_size // 2), np.float32) for _ in range(2))
    check(lib().yl_rope_table(C.byref(params), ROPE_PAIRS[pairs], rows, cos.ctypes.data, sin.ctypes.data))
    return cos, sin


def paged_append(keys, values, batch: PagedBatch, q, k, v, n_heads: int, pairs: str = "none", cos=None, sin=None):
    """yl_paged_append -> (q rotated or None, keys, values)."""
    dk, dv, cache = _pool(keys, values)
    batch.check_prefix(cache.page_size)
    k, v = np.asarray(k, np.float32), np.asarray(v, np.float32)
    kv = cache.n_kv_heads * cache.head_size
    if k.ndim != 2 or k.shape != v.shape or k.shape[1] != kv or (q is not None and np.shape(q) != (len(k), n_heads * cache.head_size)):
        raise ValueError("q, k, v: [rows][heads * head_size]")
    if cos is not None and (np.shape(cos) != np.shape(sin) or np.shape(cos)[1:] != (cache.head_size // 2,)):
        raise ValueError("cos, sin: [positions][head_size / 2]")
    desc, held = batch.upload(len(k))
    (bk, pk, lk), (bv, pv, lv) = _rows(k), _rows(v)
    bq, pq, lq = _rows(q) if q is not None else (None, None, 0)
    bc, bs = (DeviceBuffer.from_numpy(np.ascontiguousarray(t, np.float32)) if t is not None else None for t in (cos, sin))
    check(lib().yl_paged_append(C.byref(cache), C.byref(desc), n_heads, pq, lq, pq, lq, pk, lk, pv, lv, ROPE_PAIRS[pairs],
                                bc.ptr if bc else None, bs.ptr if bs else None, len(cos) if cos is not None else 0, None))
    check(lib().yl_synchronize())
    return bq.numpy() if bq else None, dk.numpy(), dv.numpy()


def paged_gather(keys, values, batch: PagedBatch, rows: int, fill: float = 0.0):
    """yl_paged_gather of `rows` rows -> (keys, values) [rows][kv_heads *
    head_size]; rows whose position nothing holds come back as `fill`."""
    dk, dv, cache = _pool(keys, values)
    batch.check_prefix(cache.page_size)
    desc, held = batch.upload(rows)
    kv = cache.n_kv_heads * cache.head_size
    out = [DeviceBuffer.from_numpy(np.full((rows, kv), fill, np.float32)) for _ in range(2)]
    check(lib().yl_paged_gather(C.byref(cache), C.byref(desc), out[0].ptr, kv, out[1].ptr, kv, None))
    check(lib().yl_synchronize())
    return out[0].numpy(), out[1].numpy()


def paged_attention(keys, values, batch: PagedBatch, q, n_heads: int, attn_scale: float) -> np.ndarray:
    """yl_paged_attention of q [rows][n_heads * head_size] (rows of no sequence come back as zeros)."""
    dk, dv, cache = _pool(keys, values)
    batch.check_prefix(cache.page_size)
    dq, pq, lq = _rows(q)
    if lq != n_heads * cache.head_size:
        raise ValueError("q: [rows][n_heads * head_size]")
    desc, held = batch.upload(len(q))
    out = DeviceBuffer.zeros((len(q), lq), np.float32)
    need = lib().yl_paged_attention_workspace(C.byref(cache), C.byref(desc), n_heads)
    space = DeviceBuffer(need)
    check(lib().yl_paged_attention(out.ptr, lq, pq, lq, C.byref(cache), C.byref(desc), n_heads, attn_scale, space.ptr,
                                   need, None))
    check(lib().yl_synchronize())
    return out.numpy()


@dataclasses.dataclass
class PagedTables:
    """yl_paged_tables on host arrays: page_table [seqs][entries], kv_len
    [seqs], refs [pages].  The operations below update them in place."""
    page_table: np.ndarray
    kv_len: np.ndarray
    refs: np.ndarray
    page_size: int
    prefix_len: int = 0
    prefix_pages: np.ndarray | None = None

    def __post_init__(self):
        self.page_table = np.ascontiguousarray(self.page_table, np.int32)
        self.kv_len = np.ascontiguousarray(self.kv_len, np.uint32)
        self.refs = np.ascontiguousarray(self.refs, np.int32)
        if self.page_table.ndim != 2 or self.page_table.shape[0] != self.kv_len.size:
            raise ValueError("page_table holds a row of entries per sequence")
        if self.prefix_pages is not None:
            self.prefix_pages = np.ascontiguousarray(self.prefix_pages, np.int32)
        if self.prefix_len and (self.prefix_pages is None or self.prefix_pages.size * self.page_size < self.prefix_len):
            raise ValueError("prefix_pages does not reach prefix_len")

    def _run(self, forks: int, call):
        """call(descriptor, workspace pointer, its bytes) on device copies, which are read back."""
        arrays = [self.page_table, self.kv_len, self.refs] + ([self.prefix_pages] if self.prefix_len else [])
        held = [DeviceBuffer.from_numpy(a) for a in arrays]
        desc = PagedTablesDesc(*self.page_table.shape, self.refs.size, self.page_size, held[0].ptr, held[1].ptr, held[2].ptr,
                               self.prefix_len, held[3].ptr if self.prefix_len else None)
        need = lib().yl_paged_tables_workspace(C.byref(desc), forks)
        space = DeviceBuffer(need)
        check(call(C.byref(desc), space.ptr, need))
        check(lib().yl_synchronize())
        for a, b in zip(arrays, held):
            a[...] = b.numpy()


def _layer_pools(layers):
    """Device copies and descriptors of [(keys, values), ...]."""
    pools = [_pool(k, v) for k, v in layers]
    return pools, (PagedCacheDesc * max(1, len(pools)))(*[p[2] for p in pools])


def _pools_back(pools):
    return [(p[0].numpy(), p[1].numpy()) for p in pools]


def _ids(x, dtype=np.uint32):
    x = np.ascontiguousarray(x, dtype)
    if x.ndim != 1:
        raise ValueError("ids: one dimension")
    return x, DeviceBuffer.from_numpy(x)


def paged_reserve(tables: PagedTables, want_len) -> int:
    """yl_paged_reserve -> entries that got no page."""
    want, dw = _ids(want_len)
    if want.size != tables.kv_len.size:
        raise ValueError("want_len: one per sequence")
    lacking = DeviceBuffer.zeros(1, np.uint32)
    tables._run(0, lambda t, w, n: lib().yl_paged_reserve(t, dw.ptr, lacking.ptr, w, n, None))
    return int(lacking.numpy()[0])


def paged_fork(tables: PagedTables, layers, parents, children):
    """yl_paged_fork of layers [(keys, values), ...] -> (children that got no page, layers)."""
    (p, dp), (c, dc) = _ids(parents), _ids(children)
    if p.size != c.size:
        raise ValueError("a child for every parent")
    pools, descs = _layer_pools(layers)
    lacking = DeviceBuffer.zeros(1, np.uint32)
    tables._run(p.size, lambda t, w, n: lib().yl_paged_fork(t, descs, len(pools), dp.ptr, dc.ptr, p.size, lacking.ptr, w, n, None))
    return int(lacking.numpy()[0]), _pools_back(pools)


def paged_release(tables: PagedTables, seqs) -> None:
    """yl_paged_release."""
    s, ds = _ids(seqs)
    tables._run(0, lambda t, w, n: lib().yl_paged_release(t, ds.ptr, s.size, None))


def paged_compact(tables: PagedTables, layers):
    """yl_paged_compact of layers [(keys, values), ...] -> (pages in use, layers)."""
    pools, descs = _layer_pools(layers)
    used = DeviceBuffer.zeros(1, np.uint32)
    tables._run(0, lambda t, w, n: lib().yl_paged_compact(t, descs, len(pools), used.ptr, w, n, None))
    return int(used.numpy()[0]), _pools_back(pools)


def paged_copy(dst_layers, src_layers, dst_pages, src_pages):
    """yl_paged_copy from one set of layers [(keys, values), ...] to another (None: the same pools) -> the written ones."""
    (d, dd), (s, ds) = _ids(dst_pages, np.int32), _ids(src_pages, np.int32)
    if d.size != s.size or (src_layers is not None and len(src_layers) != len(dst_layers)):
        raise ValueError("as many sources as destinations")
    to, to_desc = _layer_pools(dst_layers)
    src, src_desc = _layer_pools(src_layers) if src_layers is not None else (to, to_desc)
    check(lib().yl_paged_copy(to_desc, src_desc, len(to), dd.ptr, ds.ptr, d.size, None))
    check(lib().yl_synchronize())
    return _pools_back(to)


def _row_lists(lists, dtype):
    """(entries of all rows, starts) of a list of arrays per row."""
    rows = [np.ascontiguousarray(x, dtype).ravel() for x in lists]
    return np.concatenate(rows + [np.empty(0, dtype)]), np.concatenate([[0], np.cumsum([r.size for r in rows])]).astype(np.uint32)


def adjust_logits(logits, tokens=None, n_prompt=None, repetition=None, presence=None, frequency=None, biases=None, mask=None,
                  mask_of=None) -> np.ndarray:
    """yl_adjust_logits of logits [rows][vocab] (float32, float16, or bf16 bits
    as uint16).  tokens: an array of ids per row; biases: (ids, values) per row;
    mask: uint32 words [grammars][ceil(vocab / 32)]; the others one per row."""
    x = np.ascontiguousarray(logits)
    if x.ndim != 2 or x.dtype not in _DTYPE_OF:
        raise ValueError("logits: [rows][vocab] of float32, float16 or uint16 (bf16 bits)")
    rows, vocab = x.shape
    per_row = dict(n_prompt=n_prompt, repetition=repetition, presence=presence, frequency=frequency, mask_of=mask_of, tokens=tokens, biases=biases)
    for name, v in per_row.items():
        if v is not None and len(v) != rows:
            raise ValueError(name + ": one per row")
    ids, starts = _row_lists(tokens, np.uint32) if tokens is not None else (None, None)
    bias_ids, bias_start = _row_lists([b[0] for b in biases], np.uint32) if biases is not None else (None, None)
    bias, ends = _row_lists([b[1] for b in biases], np.float32) if biases is not None else (None, None)
    if biases is not None and not np.array_equal(bias_start, ends):
        raise ValueError("biases: a value for every id")
    if mask is not None and np.ndim(mask) != 2:
        raise ValueError("mask: [grammars][words]")
    held = []

    def put(a, dtype):
        if a is None:
            return None
        held.append(DeviceBuffer.from_numpy(np.ascontiguousarray(a, dtype)))
        return held[-1].ptr

    r = LogitRules(put(ids, np.uint32), put(starts, np.uint32), put(n_prompt, np.uint32), ids.size if ids is not None else 0,
                   put(repetition, np.float32), put(presence, np.float32), put(frequency, np.float32), put(bias_ids, np.uint32),
                   put(bias, np.float32), put(bias_start, np.uint32), bias.size if bias is not None else 0, put(mask, np.uint32),
                   np.shape(mask)[1] if mask is not None else 0, np.shape(mask)[0] if mask is not None else 0, put(mask_of, np.int32))
    dx = DeviceBuffer.from_numpy(x)
    check(lib().yl_adjust_logits(dx.ptr, vocab, dx.ptr, vocab, DTYPES[_DTYPE_OF[x.dtype]], rows, vocab, C.byref(r), None))
    check(lib().yl_synchronize())
    return dx.numpy()


def token_logprobs(logits, tokens=None, top: int = 0):
    """yl_token_logprobs of logits [rows][vocab] (float32, float16, or bf16
    bits as uint16) -> (log probabilities of tokens or None, entropies,
    ids [rows][top], their log probabilities)."""
    x = np.ascontiguousarray(logits)
    if x.ndim != 2 or x.dtype not in _DTYPE_OF:
        raise ValueError("logits: [rows][vocab] of float32, float16 or uint16 (bf16 bits)")
    rows, vocab = x.shape
    if tokens is not None and np.shape(tokens) != (rows,):
        raise ValueError("one token per row")
    dx = DeviceBuffer.from_numpy(x)
    dt = DeviceBuffer.from_numpy(np.ascontiguousarray(tokens, np.uint32)) if tokens is not None else None
    lp, ent = DeviceBuffer.zeros(rows, np.float32), DeviceBuffer.zeros(rows, np.float32)
    ids, tlp = DeviceBuffer.zeros((rows, top), np.uint32), DeviceBuffer.zeros((rows, top), np.float32)
    need = lib().yl_token_logprobs_workspace(rows, vocab, top)
    space = DeviceBuffer(need)
    check(lib().yl_token_logprobs(dx.ptr, DTYPES[_DTYPE_OF[x.dtype]], rows, vocab, vocab, dt.ptr if dt else None,
                                  lp.ptr if dt else None, ent.ptr, top, ids.ptr if top else None,
                                  tlp.ptr if top else None, space.ptr, need, None))
    check(lib().yl_synchronize())
    return lp.numpy() if dt else None, ent.numpy(), ids.numpy(), tlp.numpy()
