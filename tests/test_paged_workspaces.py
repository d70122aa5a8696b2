"""A workspace that the size functions give for a batch serves every smaller one (no GPU)."""
import ctypes as C
import random

import pytest

P = 1 << 20     # an address that no size function reads
DTYPES = {"f32": 0, "f16": 1, "bf16": 2}
LAYOUTS = [(32, 8, 64), (32, 8, 128), (9, 3, 64), (8, 1, 128), (4, 2, 32), (64, 1, 64), (160, 160, 32)]


def _attention(yl, layout, dtype, seqs, rows, pages, max_len, starts, prefix, page=16):
    heads, kvh, hd = layout
    cache = yl.PagedCacheDesc(P, P, DTYPES[dtype], 1 << 20, page, kvh, hd)
    batch = yl.PagedBatchDesc(seqs, rows, pages, max_len, P, P, P if starts else None, prefix, P if prefix else None)
    return yl.lib().yl_paged_attention_workspace(C.byref(cache), C.byref(batch), heads)


def test_fewer_decoded_sequences(yl):
    """Also past the numbers where a batch is divided in another way."""
    for dtype in DTYPES:
        needs = [_attention(yl, (32, 8, 128), dtype, n, n, 500, 8000, False, 0) for n in range(1, 700)]
        assert needs == sorted(needs) and needs[0] > 0


def test_fewer_rows_of_logits(yl):
    L = yl.lib()
    for vocab in (512, 16384, 16385, 49152, 128256, 5_000_000):
        for top in (0, 1, 20, 32):
            needs = [L.yl_token_logprobs_workspace(n, vocab, top) for n in range(1, 400)]
            assert needs == sorted(needs)
    for rows in (1, 31, 32, 300):
        needs = [L.yl_token_logprobs_workspace(rows, v, 20) for v in range(1, 300000, 777)]
        assert needs == sorted(needs)
        assert L.yl_token_logprobs_workspace(rows, 128256, 5) <= L.yl_token_logprobs_workspace(rows, 128256, 20)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("layout", LAYOUTS)
def test_any_smaller_batch(yl, dtype, layout):
    """No more sequences, rows, entries, positions and prefix; row_start or none."""
    r = random.Random(f"{dtype}{layout}")
    ln = lambda hi: int(round(hi ** r.random()))
    for _ in range(60):
        seqs, rows, pages, prefix = ln(3000), ln(12000), ln(3000), r.choice([0, 0, ln(9000)])
        max_len = r.choice([0, ln(60000)])
        most = _attention(yl, layout, dtype, seqs, rows, pages, max_len, True, prefix)
        for _ in range(150):
            edge = lambda hi, *at: min(hi, r.choice([hi, ln(hi), *at]))
            n, q = edge(seqs, 1, 255, 256, 512, 513), edge(rows, 1, 600, 2400, 2500)
            p, e = edge(prefix) if prefix and r.random() < 0.8 else 0, edge(pages, 40, 41, 128, 129)
            ml = edge(max_len, 640, 641, 2048, 2049) if max_len else r.choice([0, ln(60000)])
            starts = r.random() < 0.6
            if not starts:
                n = q = min(n, q)
            need = _attention(yl, layout, dtype, n, q, e, ml, starts, p)
            assert need <= most, (seqs, rows, pages, max_len, prefix, "|", n, q, e, ml, p, starts, need, most)
