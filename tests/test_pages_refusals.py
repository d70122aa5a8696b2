"""What the page operations and the rules on logits refuse before any work is
enqueued, their workspaces, and the page arithmetic on the host (no GPU)."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from test_paged_refusals import ARG, BAD_CACHE, FORMAT, RANGE, ROOT, P, _cache


def _tables(yl, **kw):
    f = dict(n_seqs=4, max_pages=3, n_pages=4, page_size=16, page_table=P, kv_len=P, refs=P, prefix_len=0, prefix_pages=None)
    f.update(kw)
    return yl.PagedTablesDesc(*f.values())


def _ref(t):
    return C.byref(t) if t is not None else None


def _layers(yl, n=2, **kw):
    return (yl.PagedCacheDesc * n)(*[_cache(yl, **kw) for _ in range(n)])


def _fork(yl, t, layers=None, n_layers=2, parents=P, children=P, n=3, space=P, less=0):
    layers = _layers(yl) if layers is None else layers
    return yl.lib().yl_paged_fork(_ref(t), layers or None, n_layers, parents, children, n, None, space, _need(yl, t, n) - less, None)


def _compact(yl, t, layers=None, n_layers=2, used=P, space=P, less=0):
    layers = _layers(yl) if layers is None else layers
    return yl.lib().yl_paged_compact(_ref(t), layers or None, n_layers, used, space, _need(yl, t, 0) - less, None)


def _reserve(yl, t, want=P, space=P, less=0):
    return yl.lib().yl_paged_reserve(_ref(t), want, None, space, _need(yl, t, 0) - less, None)


def _release(yl, t, seqs=P, n=3):
    return yl.lib().yl_paged_release(_ref(t), seqs, n, None)


def _need(yl, t, n):
    return max(1, yl.lib().yl_paged_tables_workspace(_ref(t), n))


BAD_TABLES = [dict(page_size=0), dict(page_size=24), dict(page_size=512), dict(n_pages=0), dict(n_pages=1 << 27), dict(n_seqs=(1 << 22) + 1),
              dict(n_seqs=1 << 20, max_pages=1 << 12), dict(max_pages=1 << 26), dict(page_table=None), dict(kv_len=None), dict(refs=None), dict(prefix_len=3),
              dict(prefix_len=0xFFFFFFFF, prefix_pages=P)]


@pytest.mark.parametrize("call", [_fork, _compact, _reserve, _release])
@pytest.mark.parametrize("bad", BAD_TABLES)
def test_bad_tables(yl, call, bad):
    assert call(yl, _tables(yl, **bad)) in (ARG, RANGE)
    assert b"paged tables" in yl.lib().yl_last_error()
    assert yl.lib().yl_paged_tables_workspace(_ref(_tables(yl, **bad)), 0) == 0


@pytest.mark.parametrize("call", [_fork, _compact, _reserve, _release])
def test_no_tables(yl, call):
    assert call(yl, None) == ARG


@pytest.mark.parametrize("call", [_fork, _compact])
@pytest.mark.parametrize("bad", BAD_CACHE)
def test_bad_layers(yl, call, bad):
    if bad == dict(n_kv_heads=3):
        return                            # (a bad ratio to n_heads, of which the pages know none)
    assert call(yl, _tables(yl), _layers(yl, **bad)) == (FORMAT if "dtype" in bad else ARG)


@pytest.mark.parametrize("call", [_fork, _compact])
@pytest.mark.parametrize("unlike", [dict(dtype=0), dict(n_kv_heads=4), dict(head_size=32), dict(n_pages=5), dict(page_size=32)])
def test_layers_unlike_each_other_or_the_tables(yl, call, unlike):
    mixed = (yl.PagedCacheDesc * 2)(_cache(yl), _cache(yl, **unlike))
    assert call(yl, _tables(yl), mixed) == ARG
    if "n_pages" in unlike or "page_size" in unlike:
        assert call(yl, _tables(yl), _layers(yl, **unlike)) == ARG


@pytest.mark.parametrize("call", [_fork, _compact])
def test_numbers_of_layers(yl, call):
    assert call(yl, _tables(yl), _layers(yl, 130), 129) == ARG
    assert call(yl, _tables(yl), _layers(yl), 0) == ARG
    assert call(yl, _tables(yl), False) == ARG


def test_missing_arguments(yl):
    t = _tables(yl)
    assert _fork(yl, t, parents=None) == ARG and _fork(yl, t, children=None) == ARG and _fork(yl, t, n=(1 << 22) + 1) == RANGE
    assert _release(yl, t, seqs=None) == ARG and _release(yl, t, n=(1 << 22) + 1) == RANGE
    assert _reserve(yl, t, want=None) == ARG and _compact(yl, t, used=None) == ARG
    for call in (_fork, _compact, _reserve):
        assert call(yl, t, space=None) == ARG and call(yl, t, space=P + 8) == ARG and call(yl, t, less=1) == RANGE
    assert _release(yl, t, n=0) == 0
    assert yl.lib().yl_paged_tables_workspace(_ref(t), (1 << 22) + 1) == 0


def test_workspaces_serve_smaller_tables(yl):
    need = lambda n=0, **kw: yl.lib().yl_paged_tables_workspace(_ref(_tables(yl, **kw)), n)  # noqa: E731
    most = need(500, n_seqs=300, max_pages=70, n_pages=9000)
    for kw in (dict(n_seqs=299), dict(max_pages=1), dict(n_pages=1024), dict(n_pages=1), dict(n_seqs=0, max_pages=0)):
        assert 0 < need(500, **{**dict(n_seqs=300, max_pages=70, n_pages=9000), **kw}) <= most
    assert need(0, n_seqs=300, max_pages=70, n_pages=9000) <= need(400, n_seqs=300, max_pages=70, n_pages=9000) <= most
    needs = [need(7, n_pages=n) for n in range(1, 5000, 13)]
    assert needs == sorted(needs)


def test_copy_refuses(yl):
    L = yl.lib()
    copy = lambda d, s, n=2, dp=P, sp=P, pairs=1: L.yl_paged_copy(d, s, n, dp, sp, pairs, None)  # noqa: E731
    a = _layers(yl)
    assert copy(None, a) == ARG and copy(a, None) == ARG and copy(a, a, 0) == ARG and copy(_layers(yl, 130), _layers(yl, 130), 129) == ARG
    assert copy(a, a, dp=None) == ARG and copy(a, a, sp=None) == ARG and copy(a, a, pairs=1 << 31) == RANGE
    for unlike in (dict(dtype=0), dict(dtype=4), dict(n_kv_heads=4), dict(head_size=32), dict(page_size=32)):
        assert copy(a, _layers(yl, **unlike)) == ARG
    assert copy(a, _layers(yl, dtype=7)) == FORMAT
    assert copy(a, a, dp=None, sp=None, pairs=0) == 0


def _adjust(yl, rules=(), **kw):
    f = dict(out=P, out_ld=100, x=P, ld=100, dtype=0, rows=2, vocab=100)
    f.update(kw)
    r = dict(tokens=P, token_start=P, n_prompt=None, n_tokens=5, repetition=P, presence=None, frequency=None, bias_ids=P, bias=P, bias_start=P, n_biases=2,
             mask=P, mask_ld=4, mask_rows=2, mask_of=None)
    r.update(rules or {})
    desc = yl.LogitRules(*r.values())
    return yl.lib().yl_adjust_logits(*f.values(), C.byref(desc) if rules is not None else None, None)


@pytest.mark.parametrize("bad,status", [
    (dict(dtype=3), FORMAT), (dict(dtype=-1), FORMAT), (dict(dtype=4), FORMAT), (dict(vocab=0), ARG), (dict(ld=99), ARG), (dict(out_ld=99), ARG),
    (dict(vocab=1 << 31, ld=1 << 31, out_ld=1 << 31), ARG), (dict(rows=1 << 31), RANGE), (dict(x=None), ARG), (dict(out=None), ARG), (dict(x=P + 2), ARG),
    (dict(out=P + 1, dtype=1), ARG), (dict(out_ld=101), ARG), (dict(rules=None), ARG), (dict(rules=dict(tokens=None)), ARG),
    (dict(rules=dict(token_start=None)), ARG), (dict(rules=dict(n_tokens=1 << 31)), RANGE), (dict(rules=dict(n_biases=1 << 31)), RANGE),
    (dict(rules=dict(bias=None)), ARG), (dict(rules=dict(bias_ids=None)), ARG), (dict(rules=dict(bias_start=None)), ARG), (dict(rules=dict(mask_ld=3)), ARG),
    (dict(rules=dict(mask_rows=1)), ARG)])
def test_adjust_logits_refuses(yl, bad, status):
    assert _adjust(yl, **bad) == status
    assert b"adjust_logits" in yl.lib().yl_last_error()


def test_adjust_logits_of_no_rows(yl):
    assert _adjust(yl, rows=0) == 0


def test_wrappers_refuse(yl):
    """Shapes that the descriptions cannot express, before any allocation."""
    from yallma3_mini_inference_amd import ops
    x = np.zeros((2, 40), np.float32)
    for kw in (dict(tokens=[[1]]), dict(n_prompt=[1, 2, 3]), dict(biases=[([1], [1.0])]), dict(mask_of=[0]), dict(biases=[([1], []), ([], [])]), dict(mask=np.zeros(2, np.uint32))):
        with pytest.raises(ValueError):
            ops.adjust_logits(x, **kw)
    with pytest.raises(ValueError):
        ops.adjust_logits(np.zeros(4, np.float32))
    with pytest.raises(ValueError):
        ops.adjust_logits(np.zeros((1, 4)))
    with pytest.raises(ValueError):
        ops.PagedTables(np.zeros((2, 3)), np.zeros(3), np.zeros(5), 16)
    with pytest.raises(ValueError):
        ops.PagedTables(np.zeros((2, 3)), np.zeros(2), np.zeros(5), 16, 17, np.zeros(1))


HARNESS = r"""
#include <stdio.h>
#include <random>
#include <vector>
#include "yl_paged.h"
using namespace yl;
int main() {
    // shares of the pages: every page in one, at most 1024 of them
    for (long n : {1l, 2l, 1023l, 1024l, 1025l, 1048575l, 1048576l, 1048577l, 5000000l, (1l << 27) - 1}) {
        const long per = pages_per_group((int)n), groups = page_groups((int)n);
        if (groups < 1 || groups > 1024 || per % kPagesPerStep || per * groups < n || per * (groups - 1) >= n) { printf("%ld pages\n", n); return 1; }
    }
    // entries and slots stay in the table, whatever the lengths
    std::mt19937 r(3);
    for (int it = 0; it < 200000; it++) {
        TableArgs t{};
        t.page_shift = 4 + r() % 5; t.max_pages = r() % 6; t.prefix_len = r() % 2 ? 0 : r() % 400;
        const uint32_t odd[] = {0u, 1u, 0xFFFFFFFFu, 0x80000000u, 0x7FFFFFFFu}, len = r() % 3 ? r() % 2000 : odd[r() % 5];
        int full, slots;
        bool past;
        table_filled(t, len, &full, &slots);
        const int n = table_entries(t, len, &past);
        const long own = len > (uint32_t)t.prefix_len ? (long)len - t.prefix_len : 0, page = 1 << t.page_shift;
        if (full < 0 || full > t.max_pages || slots < 0 || slots >= page || (slots && full >= t.max_pages)) return 2;
        if (!past && own != full * page + slots) return 3;
        if (n < 0 || n > t.max_pages || past != (own > t.max_pages * page) || (!past && n != (own + page - 1) / page)) return 4;
    }
    return 0;
}
"""


def test_page_arithmetic(tmp_path):
    src, exe = tmp_path / "h.cpp", tmp_path / "h"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-I", os.path.join(ROOT, "yallma3_mini_inference_amd", "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
