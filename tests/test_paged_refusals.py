"""What the paged cache's and the scoring entry points refuse, before any work
is enqueued, and the paged kernels' index arithmetic on the host (no GPU)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARG, FORMAT, RANGE = -1, -2, -8
P = 1 << 20     # an aligned address that no refused call reads


def _cache(yl, **kw):
    f = dict(keys=P, values=P, dtype=1, n_pages=4, page_size=16, n_kv_heads=2, head_size=64)
    f.update(kw)
    return yl.PagedCacheDesc(*f.values())


def _batch(yl, **kw):
    f = dict(n_seqs=2, n_rows=2, max_pages=2, max_len=0, page_table=P, kv_len=P, row_start=None, prefix_len=0, prefix_pages=None)
    f.update(kw)
    return yl.PagedBatchDesc(*f.values())


def _append(yl, cache, batch, heads=4, **kw):
    f = dict(q_out=P, q_out_ld=4 * 64, q=P, q_ld=4 * 64, k=P, k_ld=128, v=P, v_ld=128, pairs=0, cos=P, sin=P, rows=10)
    f.update(kw)
    return yl.lib().yl_paged_append(C.byref(cache) if cache else None, C.byref(batch) if batch else None, heads, *f.values(), None)


def _attention(yl, cache, batch, heads=4, **kw):
    f = dict(out=P, out_ld=4 * 64, q=P, q_ld=4 * 64)
    f.update(kw)
    need = yl.lib().yl_paged_attention_workspace(C.byref(cache) if cache else None, C.byref(batch) if batch else None, heads)
    return yl.lib().yl_paged_attention(*f.values(), C.byref(cache) if cache else None, C.byref(batch) if batch else None,
                                       heads, 0.125, P, need, None)


BAD_CACHE = [dict(dtype=3), dict(dtype=-1), dict(n_pages=0), dict(n_pages=1 << 27), dict(page_size=8), dict(page_size=48),
             dict(page_size=0), dict(page_size=512), dict(n_kv_heads=0), dict(n_kv_heads=3), dict(head_size=0),
             dict(head_size=96), dict(head_size=256), dict(keys=None), dict(values=None), dict(keys=P + 8), dict(values=P + 4)]
BAD_BATCH = [dict(n_rows=3), dict(n_rows=1 << 30, row_start=P), dict(n_seqs=1 << 24, row_start=P), dict(kv_len=None),
             dict(page_table=None), dict(max_pages=1 << 27), dict(prefix_len=3), dict(prefix_len=0xFFFFFFFF, prefix_pages=P)]


@pytest.mark.parametrize("call", [_append, _attention])
@pytest.mark.parametrize("bad", BAD_CACHE)
def test_bad_caches(yl, call, bad):
    assert call(yl, _cache(yl, **bad), _batch(yl)) == (FORMAT if "dtype" in bad else ARG)
    assert b"paged" in yl.lib().yl_last_error()


@pytest.mark.parametrize("call", [_append, _attention])
@pytest.mark.parametrize("bad", BAD_BATCH)
def test_bad_batches(yl, call, bad):
    assert call(yl, _cache(yl), _batch(yl, **bad)) in (ARG, RANGE)


@pytest.mark.parametrize("call", [_append, _attention])
def test_missing_descriptions_and_heads(yl, call):
    assert call(yl, None, _batch(yl)) == ARG
    assert call(yl, _cache(yl), None) == ARG
    for heads in (0, 3, 2048):
        assert call(yl, _cache(yl), _batch(yl), heads) == ARG


@pytest.mark.parametrize("bad", [dict(pairs=2), dict(pairs=-2), dict(cos=None), dict(sin=None), dict(k=None), dict(v=None),
                                 dict(q=None), dict(q_out=None), dict(q_ld=255), dict(q_out_ld=255), dict(k_ld=127),
                                 dict(v_ld=0), dict(q_ld=300)])
def test_append_refuses(yl, bad):
    assert _append(yl, _cache(yl), _batch(yl), **bad) == ARG


@pytest.mark.parametrize("bad", [dict(out=None), dict(q=None), dict(q_ld=255), dict(out_ld=12), dict(out_ld=300)])
def test_attention_refuses(yl, bad):
    assert _attention(yl, _cache(yl), _batch(yl), **bad) == ARG


def test_attention_refuses_a_small_workspace(yl):
    c, b, L = _cache(yl, n_pages=1 << 16), _batch(yl, n_seqs=1, n_rows=1, max_pages=1 << 12), yl.lib()
    need = L.yl_paged_attention_workspace(C.byref(c), C.byref(b), 4)
    if need:
        assert L.yl_paged_attention(P, 256, P, 256, C.byref(c), C.byref(b), 4, 0.125, P, need - 1, None) == RANGE
        for at in (None, P + 4):
            assert L.yl_paged_attention(P, 256, P, 256, C.byref(c), C.byref(b), 4, 0.125, at, need, None) == ARG
    # a description that the call refuses needs none
    assert L.yl_paged_attention_workspace(C.byref(_cache(yl, page_size=8)), C.byref(b), 4) == 0
    assert L.yl_paged_attention_workspace(None, C.byref(b), 4) == 0


def test_nothing_to_do_is_no_error(yl):
    for b in (_batch(yl, n_seqs=0, n_rows=0), _batch(yl, n_seqs=2, n_rows=0, row_start=P), _batch(yl, n_seqs=0, n_rows=2, row_start=P)):
        assert _append(yl, _cache(yl), b) == 0
        assert _attention(yl, _cache(yl), b) == 0


def _logprobs(yl, **kw):
    f = dict(logits=P, dtype=0, rows=2, vocab=100, ld=100, tokens=P, logprob=P, entropy=P, top=5, ids=P, tlp=P, space=P)
    f.update(kw)
    need = yl.lib().yl_token_logprobs_workspace(f["rows"], f["vocab"], f["top"])
    return yl.lib().yl_token_logprobs(*f.values(), need, None)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=3), FORMAT), (dict(dtype=-1), FORMAT), (dict(vocab=0), ARG), (dict(ld=99), ARG), (dict(vocab=1 << 31, ld=1 << 31), ARG),
    (dict(top=33), ARG), (dict(vocab=4, top=5), ARG), (dict(rows=1 << 31), RANGE), (dict(logits=None), ARG),
    (dict(logits=P + 2), ARG), (dict(logits=P + 1, dtype=1), ARG), (dict(tokens=None), ARG), (dict(logprob=None), ARG),
    (dict(ids=None), ARG), (dict(tlp=None), ARG), (dict(tokens=None, logprob=None, entropy=None, top=0), ARG)])
def test_logprobs_refuses(yl, bad, status):
    assert _logprobs(yl, **bad) == status
    assert b"token_logprobs" in yl.lib().yl_last_error()


def test_logprobs_refuses_a_small_workspace(yl):
    L = yl.lib()
    need = L.yl_token_logprobs_workspace(1, 128256, 20)
    if need:
        args = (P, 0, 1, 128256, 128256, P, P, P, 20, P, P)
        assert L.yl_token_logprobs(*args, P, need - 1, None) == RANGE
        assert L.yl_token_logprobs(*args, None, need, None) == ARG


def test_logprobs_of_no_rows(yl):
    assert _logprobs(yl, rows=0) == 0


def test_host_wrappers_refuse(yl):
    """Array shapes that the descriptions cannot express are refused before any allocation."""
    from yallma3_mini_inference_amd import ops
    k = np.zeros((2, 1, 16, 32), np.float16)
    b = ops.PagedBatch(np.zeros((1, 1), np.int32), np.ones(1, np.uint32))
    q = np.zeros((1, 32), np.float32)
    with pytest.raises(ValueError):
        ops.token_logprobs(np.zeros(5, np.float32))
    with pytest.raises(ValueError):
        ops.token_logprobs(np.zeros((1, 5), np.float64))
    with pytest.raises(ValueError):
        ops._pool(k, k.astype(np.float32))
    with pytest.raises(ValueError):
        ops.PagedBatch(b.page_table, b.kv_len, np.zeros(1, np.uint32)).upload(1)
    with pytest.raises(ValueError):
        ops.PagedBatch(b.page_table, b.kv_len, None, 17, np.zeros(1, np.int32)).check_prefix(16)
    assert q.shape == (1, 32)


@pytest.mark.parametrize("pairs,half_pairs", [("adjacent", False), ("half", True)])
def test_rope_table(yl, pairs, half_pairs):
    """Angles in f64 from the formula; an f32 angle of position p carries an
    error of p times the frequency's (the f32 power and, adjacent, up to 15
    chained products: 20 U) and its own rounding."""
    from yallma3_mini_inference_amd import ops
    from yallma3_mini_inference_amd._lib import RopeParams
    hd, rows = 32, 70
    p = RopeParams(hd, 4, 2, 10000.0, 1.0, 0.0, 1.0, 1 << 30)
    cos, sin = ops.rope_table(p, pairs, rows)
    angle = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(0, hd, 2) / hd)[None]
    bound = 24 * 2.0 ** -24 * angle + 2.0 ** -23
    assert (np.abs(cos - np.cos(angle)) <= bound).all() and (np.abs(sin - np.sin(angle)) <= bound).all()


def test_rope_table_refuses(yl):
    from yallma3_mini_inference_amd._lib import RopeParams
    L, t = yl.lib(), np.zeros(64, np.float32).ctypes.data
    good = RopeParams(32, 4, 2, 10000.0, 1.0, 0.0, 1.0, 4096)
    assert L.yl_rope_table(None, 0, 1, t, t) == ARG
    for pairs in (-1, 2):
        assert L.yl_rope_table(C.byref(good), pairs, 1, t, t) == ARG
    assert L.yl_rope_table(C.byref(good), 0, 1, None, t) == ARG
    for hd in (0, 31, 2048):
        assert L.yl_rope_table(C.byref(RopeParams(hd, 4, 2, 10000.0, 1.0, 0.0, 1.0, 4096)), 0, 1, t, t) == ARG
    assert L.yl_rope_table(C.byref(good), 0, 0, None, None) == 0


HARNESS = r"""
#include <stdio.h>
#include <random>
#include <vector>
#include "yl_paged.h"
using namespace yl;
// Tables, lengths and row starts of random content, valid and not: every
// address has to lie in the pool, every table access in the table.
int main() {
    std::mt19937 r(7);
    long placed = 0, nothing = 0;
    for (int it = 0; it < 3000; it++) {
        PagedArgs a{};
        a.n_pages = 1 + r() % 9; a.page_shift = 4 + r() % 5; a.n_kv = 1 + r() % 3; a.hd = 32 << (r() % 3);
        a.n_seqs = r() % 6; a.n_rows = r() % 40; a.max_pages = r() % 5; a.prefix_len = r() % 3 ? 0 : r() % 100;
        std::vector<int32_t> table(a.n_seqs * a.max_pages), pre((a.prefix_len + (1 << a.page_shift) - 1) >> a.page_shift);
        std::vector<uint32_t> len(a.n_seqs), st(a.n_seqs + 1);
        const uint32_t odd[] = {0u, 0xFFFFFFFFu, 0x80000000u, 0x7FFFFFFFu, 1000000u};
        for (auto& t : table) t = r() % 4 ? (int)(r() % a.n_pages) : (int)odd[r() % 5];
        for (auto& t : pre) t = r() % 4 ? (int)(r() % a.n_pages) : (int)odd[r() % 5];
        for (auto& l : len) l = r() % 4 ? r() % 300 : odd[r() % 5];
        uint32_t at = 0;
        for (auto& s : st) { s = r() % 8 ? at : odd[r() % 5]; at += r() % 9; }
        a.table = table.data(); a.prefix_pages = pre.data(); a.kv_len = len.data(); a.row_start = st.data();
        const size_t pool = ((size_t)a.n_pages * a.n_kv << a.page_shift) * a.hd;
        for (int row = 0; row < a.n_rows; row++) {
            const int s = paged_seq_of_row(a, row);
            if (s < -1 || s >= a.n_seqs) { printf("sequence %d\n", s); return 1; }
            if (s < 0) continue;
            int f, e;
            paged_rows(a, s, &f, &e);
            if (f < 0 || e > a.n_rows || f > e) { printf("rows %d %d\n", f, e); return 1; }
            if (row < f || row >= e) continue;
            const int64_t pos = paged_row_pos(len[s], e, row);
            const int lim = paged_limit(a, pos);
            if (lim < 0 || lim > paged_capacity(a)) { printf("limit %d\n", lim); return 1; }
            for (int64_t p : {(int64_t)-1, (int64_t)0, pos, (int64_t)lim - 1, (int64_t)lim, paged_capacity(a) - 1, paged_capacity(a), (int64_t)1 << 33}) {
                int page, slot;
                // (table accesses run under the host's bounds checks below)
                if (!paged_place(a, s, p, &page, &slot)) { nothing++; continue; }
                placed++;
                if (page < 0 || page >= a.n_pages || slot < 0 || slot >> a.page_shift) { printf("place %d %d\n", page, slot); return 1; }
                if (paged_offset(a, page, a.n_kv - 1, slot) + a.hd > pool) { printf("offset\n"); return 1; }
            }
        }
    }
    printf("%ld placed, %ld nothing\n", placed, nothing);
    return placed > 1000 && nothing > 1000 ? 0 : 1;
}
"""


def test_index_arithmetic_stays_in_bounds(tmp_path):
    """Random tables, lengths and row starts, some of them nonsense, through
    the kernels' own index functions under the host's address checks."""
    src, exe = tmp_path / "h.cpp", tmp_path / "h"
    src.write_text(HARNESS)
    cmd = ["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-I",
           os.path.join(ROOT, "yallma3_mini_inference_amd", "csrc"), str(src), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
