"""What the entry points refuse of MXFP4 pages and of gathering, and the pages' byte arithmetic on the host (no GPU)."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

from test_paged_workspaces import LAYOUTS
from test_paged_refusals import ARG, BAD_BATCH, BAD_CACHE, FORMAT, RANGE, ROOT, P, _append, _attention, _batch, _cache

MX = 4


def _gather(yl, cache, batch, **kw):
    f = dict(k=P, k_ld=128, v=P, v_ld=128)
    f.update(kw)
    return yl.lib().yl_paged_gather(C.byref(cache) if cache else None, C.byref(batch) if batch else None, *f.values(), None)


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_gather_refuses_bad_caches(yl, bad):
    if bad == dict(n_kv_heads=3):
        return                    # (a bad ratio to n_heads, of which gathering knows none)
    assert _gather(yl, _cache(yl, **bad), _batch(yl)) == (FORMAT if "dtype" in bad else ARG)
    assert b"paged" in yl.lib().yl_last_error()


@pytest.mark.parametrize("bad", BAD_BATCH)
def test_gather_refuses_bad_batches(yl, bad):
    assert _gather(yl, _cache(yl), _batch(yl, **bad)) in (ARG, RANGE)


@pytest.mark.parametrize("bad", [dict(k=None, v=None), dict(k_ld=127), dict(v_ld=0)])
def test_gather_refuses(yl, bad):
    assert _gather(yl, _cache(yl), _batch(yl), **bad) == ARG


def test_gather_of_nothing(yl):
    assert _gather(yl, None, _batch(yl)) == ARG and _gather(yl, _cache(yl), None) == ARG
    for b in (_batch(yl, n_seqs=0, n_rows=0), _batch(yl, n_seqs=2, n_rows=0, row_start=P), _batch(yl, n_seqs=0, n_rows=2, row_start=P)):
        assert _gather(yl, _cache(yl), b) == 0


@pytest.mark.parametrize("call", [_append, _attention])
@pytest.mark.parametrize("bad", [b for b in BAD_CACHE if "dtype" not in b])
def test_mx_pages_are_checked_as_others(yl, call, bad):
    assert call(yl, _cache(yl, dtype=MX, **bad), _batch(yl)) == ARG


def test_logits_are_not_mx(yl):
    L = yl.lib()
    assert L.yl_token_logprobs(P, MX, 1, 100, 100, P, P, P, 0, None, None, P, 1 << 20, None) == FORMAT


def test_wrapper_refuses(yl):
    from yallma3_mini_inference_amd import ops
    for shape in ((2, 1, 16, 32), (2, 16, 34)):
        with pytest.raises(ValueError):
            ops._pool(np.zeros(shape, np.uint8), np.zeros(shape, np.uint8))


@pytest.mark.parametrize("layout", LAYOUTS)
def test_a_workspace_serves_smaller_batches(yl, layout):
    """As test_paged_workspaces.py has it for the other types: no more sequences, rows, entries, positions and prefix."""
    heads, kvh, hd = layout

    def need_of(seqs, rows, pages, max_len, starts, prefix):
        cache = yl.PagedCacheDesc(P, P, MX, 1 << 20, 16, kvh, hd)
        batch = yl.PagedBatchDesc(seqs, rows, pages, max_len, P, P, P if starts else None, prefix, P if prefix else None)
        return yl.lib().yl_paged_attention_workspace(C.byref(cache), C.byref(batch), heads)

    r = random.Random(f"mx{layout}")
    ln = lambda hi: int(round(hi ** r.random()))  # noqa: E731
    for _ in range(60):
        seqs, rows, pages, prefix = ln(3000), ln(12000), ln(3000), r.choice([0, 0, ln(9000)])
        max_len = r.choice([0, ln(60000)])
        most = need_of(seqs, rows, pages, max_len, True, prefix)
        for _ in range(150):
            edge = lambda hi, *at: min(hi, r.choice([hi, ln(hi), *at]))  # noqa: E731
            n, q = edge(seqs, 1, 16, 17, 32, 200, 511, 512, 513), edge(rows, 1, 16, 128, 512, 600, 2400)
            p, e = edge(prefix) if prefix and r.random() < 0.8 else 0, edge(pages, 40, 41, 128, 129)
            ml = edge(max_len, 640, 641, 2048, 2049) if max_len else r.choice([0, ln(60000)])
            starts = r.random() < 0.4
            if not starts:
                n = q = min(n, q)
            need = need_of(n, q, e, ml, starts, p)
            assert need <= most, (seqs, rows, pages, max_len, prefix, "|", n, q, e, ml, p, starts, need, most)


HARNESS = r"""
#include <stdio.h>
#include <string.h>
#include <vector>
#include "yl_paged.h"
using namespace yl;
// Codes and scales of all slots fill a pool once, without gaps.
int main() {
    for (int hd : {32, 64, 128})
        for (int shift = 4; shift <= 8; shift++) {
            PagedArgs a{};
            a.n_pages = 3; a.n_kv = 2; a.hd = hd; a.page_shift = shift;
            const size_t bytes = a.n_pages * a.n_kv * paged_mx_block(a);
            if (bytes % 16 || bytes * 32 != (size_t)17 * hd * a.n_pages * a.n_kv << shift) return 1;
            std::vector<char> seen(bytes);
            for (int p = 0; p < a.n_pages; p++)
                for (int h = 0; h < a.n_kv; h++)
                    for (int s = 0; s < 1 << shift; s++) {
                        for (int i = 0; i < hd / 2; i++) seen.at(paged_mx_codes(a, p, h, s) + i)++;
                        for (int i = 0; i < hd / 32; i++) seen.at(paged_mx_scales(a, p, h, s) + i)++;
                    }
            for (char c : seen)
                if (c != 1) return 2;
        }
    PagedArgs a{};
    a.n_kv = 8; a.hd = 128; a.page_shift = 8;
    return paged_mx_codes(a, (1 << 23) - 1, 7, 255) > ((size_t)1 << 40) ? 0 : 3;
}
"""


def test_byte_arithmetic(tmp_path):
    src, exe = tmp_path / "h.cpp", tmp_path / "h"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "yallma3_mini_inference_amd", "csrc"), str(src), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    assert subprocess.run([str(exe)]).returncode == 0
