"""More serving steps as measurable cases: a paged cache held in 4 bits, the
pages of branching conversations, and rules on logits.

Five kinds of calls, each with its plain form in torch operations:

* `append`: rows of a fused QKV projection, rotated, keys and values rounded to
  MXFP4 pages (4-bit E2M1 codes, one power-of-two scale per 32 elements), and
  the values that the rows' slots now stand for;
* `attention`: causal attention of a ragged batch over such pages;
* `fork`: the last step's branches are released, every conversation gets new
  ones that share its full pages and own a copy of its last, partly filled
  page in all layers, and each branch gets room for its next positions;
* `compact`: the pages in use move to the front of the pool, in all layers;
* `logits`: penalties for repeated tokens, biases and grammar masks.

Activations are f32, as everywhere in the forward path.  Lengths belong to the
case (`lengths` is the start of their random stream), values to the seed.
"""
import ctypes
import math
import random

import torch

own = False   # False: the plain forms; True: the library's entry points

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MX_BITS = 4 + 8 / 32       # of an element: its code and its share of the block's scale


def listed():
    return [
        # one decode step of a full batch
        dict(name="append_batch", op="append", heads=32, kv_heads=8, hd=128, page=64, pairs="half",
             seqs=64, rows_lo=1, rows_hi=1, singles=1.0, past_lo=50, past_hi=6000, prefix=0, lengths=2),
        # the prompts of several new conversations in one call
        dict(name="append_prompts", op="append", heads=32, kv_heads=8, hd=64, page=16, pairs="adjacent",
             seqs=7, rows_lo=300, rows_hi=2500, singles=0.0, past_lo=1, past_hi=500, prefix=0, lengths=3),
        # one decoded token at a context of some 600 positions
        dict(name="decode_one", op="attention", heads=32, kv_heads=8, hd=64, page=16,
             seqs=1, rows_lo=1, rows_hi=1, singles=1.0, past_lo=600, past_hi=600, prefix=0, lengths=4),
        # a decode step of a full batch whose conversations differ in length
        dict(name="decode_batch", op="attention", heads=32, kv_heads=8, hd=128, page=64,
             seqs=64, rows_lo=1, rows_hi=1, singles=1.0, past_lo=100, past_hi=8000, prefix=0, lengths=5),
        # two documents at the end of a context of 131072
        dict(name="decode_long", op="attention", heads=32, kv_heads=8, hd=64, page=256,
             seqs=2, rows_lo=1, rows_hi=1, singles=1.0, past_lo=125000, past_hi=131071, prefix=0, lengths=6),
        # prompts and further turns of a few conversations
        dict(name="prompts", op="attention", heads=32, kv_heads=8, hd=64, page=16,
             seqs=4, rows_lo=600, rows_hi=3000, singles=0.0, past_lo=1, past_hi=1500, prefix=0, lengths=5),
        # four candidates of one answer
        dict(name="fork_one", op="fork", dtype="f16", layers=16, kv_heads=8, hd=64, page=16,
             parents=1, branches=4, ahead=1, past_lo=600, past_hi=600, lengths=7),
        # a beam search step of a full batch
        dict(name="fork_batch", op="fork", dtype="bf16", layers=16, kv_heads=8, hd=64, page=32,
             parents=64, branches=4, ahead=5, past_lo=20, past_hi=700, lengths=8),
        # a small model's pool after a few conversations have ended
        dict(name="compact_small", op="compact", dtype="f32", layers=2, kv_heads=3, hd=64, page=16,
             seqs=13, past_lo=1, past_hi=300, prefix=37, spare=0.6, lengths=9),
        # a pool of which most conversations have ended
        dict(name="compact_batch", op="compact", dtype="f16", layers=16, kv_heads=8, hd=64, page=16,
             seqs=48, past_lo=50, past_hi=700, prefix=333, spare=0.55, lengths=10),
        # one sampled token under a grammar
        dict(name="logits_step", op="logits", dtype="f32", rows=1, vocab=128256, past_lo=600, past_hi=600, biases=20,
             masks=1, masked=1.0, lengths=11),
        # one step of a full batch, half of its rows under one of a few grammars
        dict(name="logits_batch", op="logits", dtype="f32", rows=256, vocab=128256, past_lo=20, past_hi=4000, biases=40,
             masks=9, masked=0.5, lengths=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


LAYOUTS = [(32, 8, 64), (32, 8, 128), (9, 3, 64), (8, 1, 128), (4, 2, 32), (2, 2, 128), (16, 16, 64)]


def draw(rng):
    """One more case: layouts of the repository's models, lengths by their
    logarithm, so many sequences, pages and rows that the largest listed case
    is not passed."""
    op = rng.choice(["append", "append", "attention", "attention", "attention", "prefix", "fork", "fork", "compact",
                     "logits", "logits"])
    lengths = rng.randrange(1 << 20)
    heads, kv_heads, hd = rng.choice(LAYOUTS)
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "logits":
        vocab = rng.choice([512, 2048, 49152, 128256, rng.randint(40, 130000)])
        past = _log_int(rng, 1, 9000)
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), rows=_log_int(rng, 1, min(900, 30_000_000 // vocab)),
                    vocab=vocab, past_lo=max(1, past // 10), past_hi=past, biases=rng.choice([0, 1, 30, 300]),
                    masks=rng.choice([1, 5, 40]), masked=rng.choice([0.0, 0.3, 1.0]), lengths=lengths)
    if op in ("fork", "compact"):
        dtype, layers = rng.choice(["f32", "f16", "bf16"]), rng.choice([1, 2, 10, 16, 30])
        # pages that 500 MB hold, all layers together
        room = 500_000_000 // (2 * layers * kv_heads * page * hd * BYTES[dtype])
        past = _log_int(rng, 3, 2000)
        if op == "fork":
            branches = rng.choice([1, 2, 3, 4, 8])
            most = max(1, min(64, room // (-(-past // page) + 3 * branches)))
            return dict(op=op, dtype=dtype, layers=layers, kv_heads=kv_heads, hd=hd, page=page, parents=_log_int(rng, 1, most),
                        branches=branches, ahead=rng.choice([1, 1, 5, 40]), past_lo=max(1, past // 8), past_hi=past, lengths=lengths)
        prefix = rng.choice([0, 0, _log_int(rng, 1, 900)])
        most = max(1, min(100, (room // 2 - -(-prefix // page)) // -(-past // page)))
        return dict(op=op, dtype=dtype, layers=layers, kv_heads=kv_heads, hd=hd, page=page, seqs=_log_int(rng, 1, most),
                    past_lo=max(1, past // 8), past_hi=past, prefix=prefix, spare=rng.choice([0.0, 0.1, 0.4, 0.6]), lengths=lengths)
    if op == "append":
        past = _log_int(rng, 1, 5000)
        case = dict(op=op, heads=heads, kv_heads=kv_heads, hd=hd, page=page, pairs=rng.choice(["adjacent", "half"]),
                    seqs=_log_int(rng, 1, 64), rows_lo=1, rows_hi=_log_int(rng, 1, 2000), singles=rng.choice([0.0, 0.5, 1.0]),
                    past_lo=max(1, past // 20), past_hi=past, prefix=0, lengths=lengths)
        while sum(_lengths(case)[0]) * (heads + 2 * kv_heads) * hd > 25_000_000:
            case["seqs"] = max(1, case["seqs"] // 2)
            case["rows_hi"] = max(1, case["rows_hi"] // 2)
        return case
    prefix = _log_int(rng, 10, 6000) if op == "prefix" else 0
    rows = rng.choice([1, 1, _log_int(rng, 2, 900)])
    past = _log_int(rng, 4, 9000 if not prefix else 500)
    case = dict(op="attention", heads=heads, kv_heads=kv_heads, hd=hd, page=page,
                seqs=_log_int(rng, 2 if prefix else 1, 64), rows_lo=1, rows_hi=rows, singles=rng.choice([0.0, 0.7, 1.0]),
                past_lo=max(1, past // 50), past_hi=past, prefix=prefix, lengths=lengths)
    while True:
        n, lens = _lengths(case)
        pairs = case["seqs"] * max(n) * max(lens) * heads          # what the plain form lays out
        if pairs <= 600_000_000 and case["seqs"] * max(lens) * kv_heads * hd <= 500_000_000:
            return case
        case["seqs"], case["rows_hi"] = max(1, case["seqs"] // 2), max(1, case["rows_hi"] * 2 // 3)


def _lengths(case):
    """Per sequence: rows of this call, and its length after the call (the
    shared prefix, what it held before, these rows)."""
    r = random.Random(case["lengths"])
    rows, lens = [], []
    for _ in range(case["seqs"]):
        n = 1 if r.random() < case["singles"] else _log_int(r, case["rows_lo"], case["rows_hi"])
        rows.append(n)
        lens.append(case["prefix"] + _log_int(r, case["past_lo"], case["past_hi"]) + n)
    return rows, lens


def _pasts(case, n):
    r = random.Random(case["lengths"])
    return [_log_int(r, case["past_lo"], case["past_hi"]) for _ in range(n)]


# ---------------------------------------------------------------- MXFP4 pages

# One (page, kv head): page_size rows of hd / 2 bytes of codes (element 2i in
# the low half of byte i), then page_size rows of hd / 32 scale bytes, which
# stand for 2^(byte - 127).

def _block_scales(x):
    """Scale bytes of blocks of 32: the largest element lies below 7 of the unit, so that rounding it to 6 is off by at
    most half a step."""
    amax = x.abs().amax(-1)
    return (((amax.view(torch.int32) + 0x200000) >> 23) - 2).clamp(2, 252)


def _power(e):
    """2^(e - 127) of scale bytes."""
    return (e.int() << 23).view(torch.float32)


def _codes(x):
    """MXFP4 of x [..., hd]: codes 0 .. 15 [..., hd] and scale bytes [..., hd / 32], to nearest, ties to even codes."""
    b = x.unflatten(-1, (-1, 32))
    e = _block_scales(b)
    y = b * _power(254 - e)[..., None]
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
            + (a > 5.0).int())
    return (code + 8 * (y < 0).int()).flatten(-2), e


def _values(codes, scales):
    """What codes [..., hd] and scale bytes [..., hd / 32] stand for, in f32."""
    unit = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV)
    v = unit[(codes & 7).long()] * (1.0 - 2.0 * (codes >> 3).float())
    return (v.unflatten(-1, (-1, 32)) * _power(scales)[..., None]).flatten(-2)


def _parts(pool, page, hd):
    """Views of a pool [n_pages][kv_heads][bytes]: code bytes [..., page, hd / 2], scale bytes [..., page, hd / 32]."""
    cut = page * hd // 2
    return pool[..., :cut].unflatten(-1, (page, hd // 2)), pool[..., cut:].unflatten(-1, (page, hd // 32))


def _opened(code_bytes):
    return torch.stack((code_bytes & 15, code_bytes >> 4), -1).flatten(-2)


def _closed(codes):
    c = codes.unflatten(-1, (-1, 2))
    return (c[..., 0] + 16 * c[..., 1]).to(torch.uint8)


# ---------------------------------------------------------------- inputs

def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000 + salt)
    return g


def _normal(seed, salt, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=_gen(seed, salt), device=DEV, dtype=dtype)


def _order(seed, n):
    return torch.randperm(n, generator=_gen(seed, 5), device=DEV).to(torch.int32)


def _table(need, order, width):
    """Tables of sequences that hold `need` pages each, taken from `order` one after the other."""
    table, at = torch.full((len(need), width), -1, dtype=torch.int32), 0
    ids = order.cpu()
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table.to(DEV)


def _mx_pool(seed, salt, n_pages, kvh, page, hd):
    """Pages of normal keys or values, some dimensions larger than the rest as in real caches."""
    x = _normal(seed, salt, n_pages, kvh, page, hd)
    x *= torch.exp(0.7 * _normal(seed, salt + 20, hd))
    codes, scales = _codes(x)
    return torch.cat((_closed(codes).flatten(-2), scales.to(torch.uint8).flatten(-2)), -1)


def _prepare_cache(case, seed):
    rows, lens = _lengths(case)
    heads, kvh, hd, page, prefix = case["heads"], case["kv_heads"], case["hd"], case["page"], case["prefix"]
    need = [-(-(n - prefix) // page) for n in lens]     # pages that each sequence holds of its own
    shared = -(-prefix // page)
    n_pages, total = sum(need) + shared + 3, sum(rows)  # a few pages are free
    order = _order(seed, n_pages)
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    s = {"case": case, "table": _table(need, order[shared:], max(need)), "prefix_pages": order[:max(1, shared)].contiguous(),
         "kv_len": torch.tensor(lens, dtype=torch.int32, device=DEV),
         "row_start": torch.tensor(starts, dtype=torch.int32, device=DEV), "max_rows": max(rows), "max_len": max(lens),
         "keys": _mx_pool(seed, 1, n_pages, kvh, page, hd), "values": _mx_pool(seed, 2, n_pages, kvh, page, hd)}
    if case["op"] == "append":
        s["qkv"] = _normal(seed, 3, total, (heads + 2 * kvh) * hd)
        s["q_out"] = torch.empty(total, heads * hd, device=DEV)
        s["k_out"], s["v_out"] = (torch.empty(total, kvh * hd, device=DEV) for _ in range(2))
        # the tables of a model at theta 500000, as far as its longest sequence
        angle = torch.arange(max(lens), device=DEV, dtype=torch.float64)[:, None] * torch.pow(
            500000.0, -torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)[None]
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = _normal(seed, 3, total, heads * hd)
        s["out"] = torch.empty(total, heads * hd, device=DEV)
    return s


def _fork_sizes(case):
    lens, page, branches = _pasts(case, case["parents"]), case["page"], case["branches"]
    need = [-(-n // page) for n in lens]
    # a branch's own pages: the copy of the last one, and what its next positions take
    more = [branches * (-(-(n + case["ahead"]) // page) - n // page) for n in lens]
    width = max(-(-(n + case["ahead"]) // page) for n in lens) + 1
    return lens, need, sum(need) + sum(more) + 5, width


def _prepare_fork(case, seed):
    lens, need, n_pages, width = _fork_sizes(case)
    n, b = case["parents"], case["branches"]
    table = torch.full((n * (1 + b), width), -1, dtype=torch.int32, device=DEV)
    table[:n] = _table(need, _order(seed, n_pages), width)
    refs = torch.zeros(n_pages + 1, dtype=torch.int32, device=DEV)
    refs.index_add_(0, torch.where(table < 0, n_pages, table).flatten(), torch.ones(table.numel(), dtype=torch.int32, device=DEV))
    children = torch.arange(n, n * (1 + b), dtype=torch.int32, device=DEV)
    kv_len = torch.zeros(n * (1 + b), dtype=torch.int32, device=DEV)
    kv_len[:n] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = kv_len.clone()
    parents = torch.arange(n, dtype=torch.int32, device=DEV).repeat_interleave(b)
    want[n:] = kv_len[:n].repeat_interleave(b) + case["ahead"]
    return {"case": case, "table": table, "refs": refs[:n_pages].contiguous(), "kv_len": kv_len, "parents": parents,
            "children": children, "want": want, "lacking": torch.zeros(2, dtype=torch.int32, device=DEV),
            "pool": _normal(seed, 1, case["layers"], 2, n_pages, case["kv_heads"], case["page"], case["hd"],
                            dtype=DTYPES[case["dtype"]])}


def _compact_sizes(case):
    lens, page = _pasts(case, case["seqs"]), case["page"]
    need = [-(-n // page) for n in lens]
    shared = -(-case["prefix"] // page)
    return lens, need, shared, int((sum(need) + shared) / (1.0 - case["spare"])) + 1


def _prepare_compact(case, seed):
    lens, need, shared, n_pages = _compact_sizes(case)
    order = _order(seed, n_pages)
    table = _table(need, order[shared:], max(need) + 1)
    refs = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    refs[order[:shared + sum(need)].long()] = 1
    if len(need) > 1:      # the second conversation shares the first one's first page
        page0 = table[0, 0].clone()
        refs[table[1, 0].long()] = 0
        table[1, 0] = page0
        refs[page0.long()] = 2
    return {"case": case, "found": (table, refs, order[:max(1, shared)].clone()),
            "table": table.clone(), "refs": refs.clone(), "prefix_pages": order[:max(1, shared)].clone(),
            "kv_len": torch.tensor([case["prefix"] + n for n in lens], dtype=torch.int32, device=DEV),
            "used": torch.zeros(1, dtype=torch.int32, device=DEV),
            "pool": _normal(seed, 1, case["layers"], 2, n_pages, case["kv_heads"], case["page"], case["hd"],
                            dtype=DTYPES[case["dtype"]])}


def _prepare_logits(case, seed):
    rows, vocab = case["rows"], case["vocab"]
    g = _gen(seed, 9)
    past = _pasts(case, rows)
    starts = [0]
    for n in past:
        starts.append(starts[-1] + n)
    # text repeats itself: a few tokens of the vocabulary are most of it
    tokens = (vocab * torch.rand(starts[-1], generator=g, device=DEV) ** 4).int().clamp(max=vocab - 1)
    uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device=DEV)  # noqa: E731
    n_bias = min(case["biases"], vocab)
    words = -(-vocab // 32)
    # grammars allow from a few tokens to half of them
    share = torch.rand(case["masks"], 1, generator=g, device=DEV) ** 3 * 0.5
    bits = torch.rand(case["masks"], words * 32, generator=g, device=DEV) < share
    mask = (bits.view(case["masks"], words, 32).long() << torch.arange(32, device=DEV)).sum(-1)
    of = torch.randint(0, case["masks"], (rows,), generator=g, device=DEV, dtype=torch.int32)
    first = torch.randint(0, vocab, (rows, 1), generator=g, device=DEV)
    ids = (first + torch.arange(n_bias, device=DEV) * max(1, vocab // max(1, n_bias))) % vocab    # one token is biased once
    return {"case": case, "logits": (2.5 * _normal(seed, 1, rows, vocab)).to(DTYPES[case["dtype"]]),
            "out": torch.empty(rows, vocab, device=DEV, dtype=DTYPES[case["dtype"]]),
            "tokens": tokens, "token_start": torch.tensor(starts, dtype=torch.int32, device=DEV),
            "n_prompt": torch.tensor([n // 2 for n in past], dtype=torch.int32, device=DEV),
            "repetition": uniform(1.0, 1.4), "presence": uniform(0.0, 1.0), "frequency": uniform(0.0, 0.4),
            "bias_ids": ids.to(torch.int32).flatten().contiguous(),
            "bias": 5.0 * torch.randn(rows * n_bias, generator=g, device=DEV),
            "bias_start": torch.arange(rows + 1, dtype=torch.int32, device=DEV) * n_bias,
            "mask": mask.to(torch.int32), "mask_of": torch.where(uniform(0.0, 1.0) < case["masked"], of, -1)}


def prepare(case, seed):
    op = case["op"]
    return (_prepare_fork if op == "fork" else _prepare_compact if op == "compact" else _prepare_logits if op == "logits"
            else _prepare_cache)(case, seed)


# ---------------------------------------------------------------- plain forms

def _rows_of(s, total):
    """Per row: its sequence, its place among the sequence's rows, its position."""
    row = torch.arange(total, device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(s["row_start"], row, right=True) - 1
    first, after = s["row_start"][seq], s["row_start"][seq + 1]
    return seq, row - first, s["kv_len"][seq] - (after - row)


def _plain_append(s):
    c = s["case"]
    heads, kvh, hd, page = c["heads"], c["kv_heads"], c["hd"], c["page"]
    total = s["qkv"].shape[0]
    x = s["qkv"].view(total, heads + 2 * kvh, hd)
    seq, _, pos = _rows_of(s, total)
    pos = pos.long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    qk = x[:, :heads + kvh]
    if c["pairs"] == "adjacent":
        a, b = qk[..., 0::2], qk[..., 1::2]
        rot = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).reshape(total, heads + kvh, hd)
    else:
        a, b = qk[..., :hd // 2], qk[..., hd // 2:]
        rot = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    where, slot = s["table"][seq, pos // page].long(), pos % page
    codes, scales = _codes(torch.stack((rot[:, heads:], x[:, heads + kvh:])))
    code_bytes, scale_bytes = _closed(codes), scales.to(torch.uint8)
    kc, ks = _parts(s["keys"], page, hd)
    vc, vs = _parts(s["values"], page, hd)
    kc[where, :, slot], ks[where, :, slot] = code_bytes[0], scale_bytes[0]
    vc[where, :, slot], vs[where, :, slot] = code_bytes[1], scale_bytes[1]
    held = _values(codes, scales).flatten(-2)
    s["k_out"].copy_(held[0])
    s["v_out"].copy_(held[1])
    s["q_out"].copy_(rot[:, :heads].reshape(total, heads * hd))
    return s["q_out"], s["k_out"], s["v_out"]


def _gathered(s, pool):
    """The pool's pages in the sequences' order, in f32: [seqs][kv_heads][prefix + own positions][hd]."""
    c = s["case"]
    seqs, kvh, hd, page, prefix = c["seqs"], c["kv_heads"], c["hd"], c["page"], c["prefix"]
    codes, scales = _parts(pool, page, hd)
    held = _values(_opened(codes), scales)
    x = held[s["table"].clamp_min(0).long()].transpose(1, 2).reshape(seqs, kvh, -1, hd)
    if prefix:
        p = held[s["prefix_pages"].long()].transpose(0, 1).reshape(kvh, -1, hd)[None, :, :prefix]
        x = torch.cat((p.expand(seqs, -1, -1, -1), x), 2)
    return x


def _plain_attention(s):
    c = s["case"]
    heads, kvh, hd, seqs, most = c["heads"], c["kv_heads"], c["hd"], c["seqs"], s["max_rows"]
    total, group = s["q"].shape[0], heads // kvh
    seq, place, pos = _rows_of(s, total)
    place = place.long()
    q = torch.zeros(seqs, most, heads, hd, device=DEV)
    q[seq, place] = s["q"].view(total, heads, hd)
    limit = torch.full((seqs, most), -1, device=DEV, dtype=torch.int32)
    limit[seq, place] = pos
    q = q.view(seqs, most, kvh, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, group * most, hd)
    score = torch.matmul(q, _gathered(s, s["keys"]).transpose(2, 3).contiguous()) / math.sqrt(hd)
    masked = torch.arange(score.shape[-1], device=DEV, dtype=torch.int32) > limit[..., None]
    score = score.view(seqs, kvh, group, most, -1).masked_fill(masked[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top)).view(seqs, kvh, group * most, -1)
    out = torch.matmul(p, _gathered(s, s["values"])) / p.sum(-1, keepdim=True)
    out = out.view(seqs, kvh, group, most, hd).permute(0, 3, 1, 2, 4).reshape(seqs, most, heads * hd)
    s["out"].copy_(out[seq, place])
    return s["out"]


def _uncount(s, entries):
    """Takes one from the references of every page that `entries` names."""
    refs = torch.cat((s["refs"], s["refs"].new_zeros(1)))
    at = torch.where(entries < 0, len(s["refs"]), entries).flatten()
    refs.index_add_(0, at, torch.full_like(at, -1))
    s["refs"].copy_(refs[:-1])


def _free_pages(s):
    """All pages, the free ones first, each kind by rising id; and how many are free."""
    return torch.sort((s["refs"] > 0).int(), stable=True)[1].int(), (s["refs"] <= 0).sum()


def _plain_fork(s):
    page, table, refs, kv_len, pool = s["case"]["page"], s["table"], s["refs"], s["kv_len"], s["pool"]
    parents, children = s["parents"].long(), s["children"].long()
    # the last step's branches are given back
    _uncount(s, table[children])
    table[children] = -1
    kv_len[children] = 0
    # the new ones share the full pages and take a free page for the copy of the last one
    lens = kv_len[parents]
    full, filled = lens // page, lens % page
    order, free = _free_pages(s)
    rank = (filled > 0).cumsum(0) - 1
    got = order[rank.clamp(0, len(order) - 1)]
    made = (filled == 0) | (rank < free)
    entry = torch.arange(table.shape[1], device=DEV)
    row = torch.where(entry < full[:, None], table[parents], -1)
    row = torch.where((entry == full[:, None]) & (filled > 0)[:, None], got[:, None], row)
    row = torch.where(made[:, None], row, -1)
    last = table[parents].gather(1, full.clamp(max=table.shape[1] - 1)[:, None].long())[:, 0]
    # the copies: the filled slots of their pages
    some = torch.nonzero(made & (filled > 0))[:, 0]
    src, dst = last[some].long(), got[some].long()
    slot = torch.arange(page, device=DEV)[:, None] < filled[some][:, None, None, None]
    pool[:, :, dst] = torch.where(slot, pool[:, :, src], pool[:, :, dst])
    table[children] = row
    kv_len[children] = torch.where(made, lens, 0)
    count = torch.cat((refs, refs.new_zeros(1)))
    at = torch.where(row < 0, len(refs), row).flatten()
    count.index_add_(0, at, torch.ones_like(at))
    refs.copy_(count[:-1])
    s["lacking"][0] = (~made).sum()
    # room for the positions below `want`: missing entries take the free pages, sequence by sequence
    missing = (table < 0) & (entry < ((s["want"] + page - 1) // page)[:, None])
    order, free = _free_pages(s)
    rank = missing.flatten().cumsum(0).view(table.shape) - 1
    given = missing & (rank < free)
    table.copy_(torch.where(given, order[rank.clamp(0, len(order) - 1)], table))
    count = torch.cat((refs, refs.new_zeros(1)))
    at = torch.where(given, table, len(refs)).flatten()
    count.index_add_(0, at, torch.ones_like(at))
    refs.copy_(count[:-1])
    s["lacking"][1] = (missing & ~given).sum()
    return table, refs, kv_len, s["lacking"], pool


def _found(s):
    """The tables as they were found: a pass compacts the same pool again."""
    for name, t in zip(("table", "refs", "prefix_pages"), s["found"]):
        s[name].copy_(t)


def _plain_compact(s):
    _found(s)
    table, refs, pool = s["table"], s["refs"], s["pool"]
    held = refs > 0
    used = held.sum()
    page = torch.arange(len(refs), device=DEV)
    holes, movers = torch.nonzero(~held & (page < used))[:, 0], torch.nonzero(held & (page >= used))[:, 0]
    pool[:, :, holes] = pool[:, :, movers]
    now = page.int()
    now[movers] = holes.int()
    refs[holes] = refs[movers]
    refs[movers] = 0
    for t in (table, s["prefix_pages"]):
        t.copy_(torch.where(t < 0, t, now[t.clamp_min(0).long()]))
    s["used"].copy_(used.int())
    return table, refs, s["prefix_pages"], s["used"], pool


def _plain_logits(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    at = torch.arange(len(s["tokens"]), device=DEV, dtype=torch.int32)
    row = torch.searchsorted(s["token_start"], at, right=True) - 1
    answered = at - s["token_start"][row] >= s["n_prompt"][row]
    place = row * vocab + s["tokens"]
    count = torch.zeros(rows * vocab, device=DEV).index_add_(0, place, answered.float()).view(rows, vocab)
    seen = torch.zeros(rows * vocab, device=DEV).index_fill_(0, place, 1.0).view(rows, vocab) > 0
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if len(s["bias"]):
        at = torch.arange(len(s["bias"]), device=DEV, dtype=torch.int32)
        row = torch.searchsorted(s["bias_start"], at, right=True) - 1
        x.view(-1).index_add_(0, row * vocab + s["bias_ids"], s["bias"])
    bits = (s["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
    allowed = bits.flatten(1)[:, :vocab].bool()[s["mask_of"].clamp_min(0).long()] | (s["mask_of"] < 0)[:, None]
    s["out"].copy_(x.masked_fill(~allowed, -math.inf))
    return s["out"]


# ---------------------------------------------------------------- the library's calls

def _ok(Y, status):
    if status != 0:
        raise RuntimeError("yallma3: %d: %s" % (status, Y.lib().yl_last_error().decode()))


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _space(need):
    return torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)


def _cache(Y, s):
    c = s["case"]
    return Y.PagedCacheDesc(s["keys"].data_ptr(), s["values"].data_ptr(), Y.DTYPES["mxfp4"], s["keys"].shape[0], c["page"],
                            c["kv_heads"], c["hd"])


def _batch(Y, s, total):
    c, table = s["case"], s["table"]
    # one row per sequence in order needs no row_start
    start = None if total == c["seqs"] and s["max_rows"] == 1 else s["row_start"].data_ptr()
    return Y.PagedBatchDesc(c["seqs"], total, table.shape[1], s["max_len"], table.data_ptr(), s["kv_len"].data_ptr(),
                            start, c["prefix"], s["prefix_pages"].data_ptr() if c["prefix"] else None)


def _own_append(s):
    import yallma3_mini_inference_amd as Y
    c, x, q, L = s["case"], s["qkv"], s["q_out"], Y.lib()
    heads, kvh, hd, ld = c["heads"], c["kv_heads"], c["hd"], x.shape[1]
    cache, batch, at = _cache(Y, s), _batch(Y, s, x.shape[0]), x.data_ptr()
    _ok(Y, L.yl_paged_append(ctypes.byref(cache), ctypes.byref(batch), heads, q.data_ptr(), q.shape[1], at, ld,
                             at + 4 * heads * hd, ld, at + 4 * (heads + kvh) * hd, ld, Y.ROPE_PAIRS[c["pairs"]],
                             s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0], _stream()))
    _ok(Y, L.yl_paged_gather(ctypes.byref(cache), ctypes.byref(batch), s["k_out"].data_ptr(), kvh * hd, s["v_out"].data_ptr(),
                             kvh * hd, _stream()))
    return q, s["k_out"], s["v_out"]


def _own_attention(s):
    import yallma3_mini_inference_amd as Y
    c, q, out, L = s["case"], s["q"], s["out"], Y.lib()
    cache, batch = _cache(Y, s), _batch(Y, s, q.shape[0])
    need = L.yl_paged_attention_workspace(ctypes.byref(cache), ctypes.byref(batch), c["heads"])
    space = _space(need)
    _ok(Y, L.yl_paged_attention(out.data_ptr(), out.shape[1], q.data_ptr(), q.shape[1], ctypes.byref(cache),
                                ctypes.byref(batch), c["heads"], 1.0 / math.sqrt(c["hd"]), space.data_ptr(), need, _stream()))
    return out


def _layers(Y, s):
    """One pool per layer, and the tables that name their pages."""
    c, pool = s["case"], s["pool"]
    layers, _, n_pages, kvh, page, hd = pool.shape
    at, step = pool.data_ptr(), pool.stride(1) * pool.element_size()
    caches = (Y.PagedCacheDesc * layers)(*[Y.PagedCacheDesc(at + 2 * i * step, at + (2 * i + 1) * step, Y.DTYPES[c["dtype"]],
                                                            n_pages, page, kvh, hd) for i in range(layers)])
    prefix = c.get("prefix", 0)
    tables = Y.PagedTablesDesc(s["table"].shape[0], s["table"].shape[1], n_pages, page, s["table"].data_ptr(),
                               s["kv_len"].data_ptr(), s["refs"].data_ptr(), prefix,
                               s["prefix_pages"].data_ptr() if prefix else None)
    return caches, tables


def _own_fork(s):
    import yallma3_mini_inference_amd as Y
    L, n, lacking = Y.lib(), len(s["children"]), s["lacking"].data_ptr()
    caches, tables = _layers(Y, s)
    need = L.yl_paged_tables_workspace(ctypes.byref(tables), n)
    space = _space(need)
    _ok(Y, L.yl_paged_release(ctypes.byref(tables), s["children"].data_ptr(), n, _stream()))
    _ok(Y, L.yl_paged_fork(ctypes.byref(tables), caches, len(caches), s["parents"].data_ptr(), s["children"].data_ptr(), n,
                           lacking, space.data_ptr(), need, _stream()))
    _ok(Y, L.yl_paged_reserve(ctypes.byref(tables), s["want"].data_ptr(), lacking + 4, space.data_ptr(), need, _stream()))
    return s["table"], s["refs"], s["kv_len"], s["lacking"], s["pool"]


def _own_compact(s):
    import yallma3_mini_inference_amd as Y
    _found(s)
    L = Y.lib()
    caches, tables = _layers(Y, s)
    need = L.yl_paged_tables_workspace(ctypes.byref(tables), 0)
    space = _space(need)
    _ok(Y, L.yl_paged_compact(ctypes.byref(tables), caches, len(caches), s["used"].data_ptr(), space.data_ptr(), need, _stream()))
    return s["table"], s["refs"], s["prefix_pages"], s["used"], s["pool"]


def _own_logits(s):
    import yallma3_mini_inference_amd as Y
    c, x, out = s["case"], s["logits"], s["out"]
    rules = Y.LogitRules(s["tokens"].data_ptr(), s["token_start"].data_ptr(), s["n_prompt"].data_ptr(), s["tokens"].numel(),
                         s["repetition"].data_ptr(), s["presence"].data_ptr(), s["frequency"].data_ptr(),
                         s["bias_ids"].data_ptr(), s["bias"].data_ptr(), s["bias_start"].data_ptr(), s["bias"].numel(),
                         s["mask"].data_ptr(), s["mask"].shape[1], s["mask"].shape[0], s["mask_of"].data_ptr())
    _ok(Y, Y.lib().yl_adjust_logits(out.data_ptr(), c["vocab"], x.data_ptr(), c["vocab"], Y.DTYPES[c["dtype"]], c["rows"],
                                    c["vocab"], ctypes.byref(rules), _stream()))
    return out


def run(s):
    op = s["case"]["op"]
    if own:
        return (_own_append if op == "append" else _own_attention if op == "attention" else _own_fork if op == "fork"
                else _own_compact if op == "compact" else _own_logits)(s)
    return (_plain_append if op == "append" else _plain_attention if op == "attention" else _plain_fork if op == "fork"
            else _plain_compact if op == "compact" else _plain_logits)(s)


# ---------------------------------------------------------------- what it takes

def work(case):
    op = case["op"]
    if op == "logits":
        n, past = case["rows"] * case["vocab"], sum(_pasts(case, case["rows"]))
        # each logit in and out, the tokens, the biases, the masks
        return {"bytes": 2 * n * BYTES[case["dtype"]] + 4 * past + 8 * case["rows"] * case["biases"]
                + case["masks"] * case["vocab"] // 8, "flops": 2 * n}
    if op == "fork":
        lens, _, n_pages, width = _fork_sizes(case)
        slots = case["branches"] * sum(n % case["page"] for n in lens)
        # the filled slots of every copied page, in and out, in all layers; tables and references in and out
        return {"bytes": 4 * slots * case["layers"] * case["kv_heads"] * case["hd"] * BYTES[case["dtype"]]
                + 8 * (len(lens) * (1 + case["branches"]) * width + n_pages), "flops": 0}
    if op == "compact":
        _, need, shared, n_pages = _compact_sizes(case)
        used = sum(need) + shared
        # of pages in random order, as many lie behind the last one's new place as are free before it
        moved = used * (n_pages - used) // n_pages
        return {"bytes": 4 * moved * case["layers"] * case["kv_heads"] * case["page"] * case["hd"] * BYTES[case["dtype"]]
                + 8 * (case["seqs"] * (max(need) + 1) + n_pages), "flops": 0}
    rows, lens = _lengths(case)
    heads, kvh, hd, prefix = case["heads"], case["kv_heads"], case["hd"], case["prefix"]
    total, held = sum(rows), 2 * kvh * hd * MX_BITS / 8
    if op == "append":
        # the fused rows in, q out, keys and values into the pages, out of them and out; a cosine and a sine per pair
        return {"bytes": total * (4 * (2 * heads + 4 * kvh) * hd + 2 * held + 4 * hd), "flops": 3 * total * (heads + kvh) * hd}
    own_positions = sum(n - prefix for n in lens)
    pairs = sum(n * (total_len - n) + n * (n + 1) // 2 for n, total_len in zip(rows, lens))
    # q in, out out, each held key and value once: those of the prefix once for all
    return {"bytes": 8 * total * heads * hd + (own_positions + prefix) * held, "flops": 4 * hd * heads * pairs}


# ---------------------------------------------------------------- 64 bits

def _exact_append(case, s):
    heads, kvh, hd = case["heads"], case["kv_heads"], case["hd"]
    rows, lens = _lengths(case)
    pos = torch.cat([torch.arange(n - r, n, device=DEV) for r, n in zip(rows, lens)])
    x = s["qkv"].double().view(len(pos), -1, hd)[:, :heads]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    if case["pairs"] == "adjacent":
        q = torch.view_as_real(torch.view_as_complex(x.reshape(len(pos), heads, hd // 2, 2).contiguous()) * turn).flatten(-2)
    else:
        z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
        q = torch.cat((z.real, z.imag), -1)
    # the codes are choices: a value next to a border has no 64-bit counterpart
    return q.reshape(len(pos), heads * hd), None, None


def _exact_values(pool, page, hd):
    """A pool in 64 bits, by the fields of a code: sign, two bits of exponent, one of mantissa."""
    raw = pool.long()
    byte = raw[..., :page * hd // 2].view(*raw.shape[:2], page, hd // 2, 1)
    code = (byte >> torch.tensor([0, 4], device=DEV)).remainder(16).reshape(*raw.shape[:2], page, hd)
    sign, exponent, half = code // 8, code // 2 % 4, code % 2
    size = torch.where(exponent > 0, (2.0 + half) * 2.0 ** (exponent.double() - 2), 0.5 * half)
    scale = 2.0 ** (raw[..., page * hd // 2:].view(*raw.shape[:2], page, hd // 32).double() - 127)
    return size * (1 - 2 * sign) * scale.repeat_interleave(32, -1)


def _exact_attention(case, s):
    rows, lens = _lengths(case)
    heads, kvh, hd, page, prefix = case["heads"], case["kv_heads"], case["hd"], case["page"], case["prefix"]
    out = torch.zeros(sum(rows), heads, hd, device=DEV, dtype=torch.float64)
    table, shared, at = s["table"].long(), s["prefix_pages"].long(), 0
    for i, (r, n) in enumerate(zip(rows, lens)):
        held = table[i][table[i] >= 0]
        past = torch.arange(n, device=DEV)[None, :] > torch.arange(n - r, n, device=DEV)[:, None]
        kv = []
        for pool in (s["keys"], s["values"]):
            x = _exact_values(pool[held], page, hd).transpose(0, 1).reshape(kvh, -1, hd)[:, :n - prefix]
            if prefix:
                x = torch.cat((_exact_values(pool[shared], page, hd).transpose(0, 1).reshape(kvh, -1, hd)[:, :prefix], x), 1)
            kv.append(x)
        for h in range(kvh):
            g = slice(h * heads // kvh, (h + 1) * heads // kvh)
            q = s["q"][at:at + r].view(r, heads, hd)[:, g].double().transpose(0, 1).contiguous()
            score = (torch.matmul(q, kv[0][h].t().contiguous()) * hd ** -0.5).masked_fill(past, -math.inf)
            out[at:at + r, g] = torch.matmul(torch.softmax(score, -1), kv[1][h]).transpose(0, 1)
        at += r
    return out.reshape(sum(rows), heads * hd)


def _exact_fork(case, s):
    """Branch by branch on the host; the pool's pages as 64-bit values."""
    page, table, pool = case["page"], s["table"].cpu().tolist(), s["pool"].double()
    refs, lens, want = s["refs"].tolist(), s["kv_len"].tolist(), s["want"].tolist()
    lacking = [0, 0]

    def take():
        free = [i for i, n in enumerate(refs) if n <= 0]
        if free:
            refs[free[0]] = 1
        return free[0] if free else -1

    # copies of a page keep what lies behind the filled slots; references of shared pages are counted after all pages are taken
    more = []
    for p, c in zip(s["parents"].tolist(), s["children"].tolist()):
        full, filled = divmod(lens[p], page)
        last = take() if filled else -1
        if filled and last < 0:
            lacking[0] += 1
            continue
        for e in range(full):
            table[c][e] = table[p][e]
            more.append(table[p][e])
        if filled:
            table[c][full] = last
            pool[:, :, last, :, :filled] = pool[:, :, table[p][full], :, :filled]
        lens[c] = lens[p]
    for i in more:
        refs[i] += 1
    for row, n in zip(table, want):
        for e in range(-(-n // page)):
            if row[e] < 0:
                row[e] = take()
                lacking[1] += row[e] < 0
    ints = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (table, refs, lens, lacking)]
    return (*ints, pool)


def _exact_compact(case, s):
    table, refs, shared = (t.cpu().tolist() for t in s["found"])
    pool = s["pool"].double()
    used = sum(n > 0 for n in refs)
    holes = [i for i in range(used) if refs[i] <= 0]
    now = {}
    for i in range(used, len(refs)):
        if refs[i] > 0:
            now[i] = holes.pop(0)
            pool[:, :, now[i]] = pool[:, :, i]
            refs[now[i]], refs[i] = refs[i], 0
    table = [[now.get(e, e) for e in row] for row in table]
    shared = [now.get(e, e) for e in shared]
    ints = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (table, refs, shared, [used])]
    return (*ints, pool)


def _exact_logits(case, s):
    x = s["logits"].double()
    starts, prompts = s["token_start"].tolist(), s["n_prompt"].tolist()
    biases, grammars = s["bias_start"].tolist(), s["mask_of"].tolist()
    word = torch.arange(case["vocab"], device=DEV)
    for r in range(case["rows"]):
        told = s["tokens"][starts[r]:starts[r + 1]].long()
        met = torch.unique(told)
        rep = float(s["repetition"][r])
        x[r, met] = torch.where(x[r, met] > 0, x[r, met] / rep, x[r, met] * rep)
        n = torch.bincount(told[prompts[r]:], minlength=case["vocab"]).double()
        x[r] -= float(s["frequency"][r]) * n + float(s["presence"][r]) * (n > 0)
        b = slice(biases[r], biases[r + 1])
        x[r, s["bias_ids"][b].long()] += s["bias"][b].double()
        if grammars[r] >= 0:
            allowed = (s["mask"][grammars[r]].long()[word // 32] >> (word % 32)) % 2 == 1
            x[r, ~allowed] = -math.inf
    return x


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    return (_exact_append if op == "append" else _exact_attention if op == "attention" else _exact_fork if op == "fork"
            else _exact_compact if op == "compact" else _exact_logits)(case, s)
