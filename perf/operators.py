"""Serving steps over a paged K/V cache, and the scoring of logits, as measurable cases.

Three kinds of calls, each with its plain form in torch operations:

* `append`: the rows that a QKV projection left (one fused row per token) are
  rotated to their positions, and their keys and values go to the pages of
  their sequences;
* `attention`: causal attention of a ragged batch over those pages, also where
  the sequences share one prefix whose pages are held once;
* `logprobs`: log probabilities of given tokens, the entropy and the most
  probable alternatives, from rows of logits.

Activations are f32, as everywhere in the forward path; the pages hold f32,
f16 or bf16.  Lengths belong to the case (`lengths` is the start of their
random stream), values to the seed.
"""
import ctypes
import math
import random

import torch

own = False   # False: the plain forms; True: the library's entry points

DEV = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one decoded token of one conversation: the smallest call
        dict(name="append_step", op="append", dtype="f16", heads=32, kv_heads=8, hd=64, page=16, pairs="adjacent",
             seqs=1, rows_lo=1, rows_hi=1, singles=1.0, past_lo=600, past_hi=600, prefix=0, lengths=1),
        # one decode step of a full batch
        dict(name="append_batch", op="append", dtype="bf16", heads=32, kv_heads=8, hd=128, page=64, pairs="half",
             seqs=64, rows_lo=1, rows_hi=1, singles=1.0, past_lo=50, past_hi=6000, prefix=0, lengths=2),
        # the prompts of several new conversations in one call
        dict(name="append_prompts", op="append", dtype="f16", heads=32, kv_heads=8, hd=128, page=16, pairs="adjacent",
             seqs=7, rows_lo=300, rows_hi=2500, singles=0.0, past_lo=1, past_hi=500, prefix=0, lengths=3),
        # one decoded token at a context of some 600 positions
        dict(name="decode_one", op="attention", dtype="f16", heads=32, kv_heads=8, hd=64, page=16,
             seqs=1, rows_lo=1, rows_hi=1, singles=1.0, past_lo=600, past_hi=600, prefix=0, lengths=4),
        # a decode step of a full batch whose conversations differ in length
        dict(name="decode_batch", op="attention", dtype="bf16", heads=32, kv_heads=8, hd=128, page=64,
             seqs=64, rows_lo=1, rows_hi=1, singles=1.0, past_lo=100, past_hi=8000, prefix=0, lengths=5),
        # two documents at the end of a context of 131072
        dict(name="decode_long", op="attention", dtype="f16", heads=32, kv_heads=8, hd=64, page=256,
             seqs=2, rows_lo=1, rows_hi=1, singles=1.0, past_lo=125000, past_hi=131071, prefix=0, lengths=6),
        # prompts and further turns of a few conversations
        dict(name="prompts", op="attention", dtype="f16", heads=32, kv_heads=8, hd=64, page=16,
             seqs=4, rows_lo=600, rows_hi=3000, singles=0.0, past_lo=1, past_hi=1500, prefix=0, lengths=5),
        # prompts beside decoded tokens, 9 heads on 3 kv heads, an f32 cache
        dict(name="mixed_f32", op="attention", dtype="f32", heads=9, kv_heads=3, hd=64, page=32,
             seqs=13, rows_lo=41, rows_hi=300, singles=0.8, past_lo=1, past_hi=1900, prefix=0, lengths=32),
        # a decode step of many conversations that opened with one document
        dict(name="prefix_batch", op="attention", dtype="bf16", heads=32, kv_heads=8, hd=128, page=64,
             seqs=96, rows_lo=1, rows_hi=1, singles=1.0, past_lo=20, past_hi=400, prefix=6001, lengths=9),
        # a few conversations on one system text, some of them with several rows
        dict(name="prefix_small", op="attention", dtype="f32", heads=4, kv_heads=2, hd=32, page=16,
             seqs=7, rows_lo=1, rows_hi=5, singles=0.4, past_lo=1, past_hi=60, prefix=333, lengths=10),
        # one sampled token: its log probability, the entropy, 20 alternatives
        dict(name="logprobs_step", op="logprobs", dtype="f32", rows=1, vocab=128256, top=20),
        # a document scored token by token
        dict(name="logprobs_document", op="logprobs", dtype="f32", rows=700, vocab=128256, top=5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: layouts of the repository's models, lengths by their
    logarithm, so many sequences and rows that the largest listed case is not
    passed."""
    op = rng.choice(["append", "append", "attention", "attention", "attention", "prefix", "prefix", "logprobs", "logprobs"])
    if op == "logprobs":
        vocab = rng.choice([512, 2048, 49152, 128256, rng.randint(40, 130000)])
        return dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), rows=_log_int(rng, 1, min(2000, 80_000_000 // vocab)),
                    vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]))
    heads, kv_heads, hd = rng.choice([(32, 8, 64), (32, 8, 128), (9, 3, 64), (8, 1, 128), (4, 2, 32), (2, 2, 128), (4, 1, 64)])
    c = dict(op="append" if op == "append" else "attention", dtype=rng.choice(["f32", "f16", "bf16"]), heads=heads,
             kv_heads=kv_heads, hd=hd, page=rng.choice([16, 32, 64, 128, 256]), lengths=rng.randint(0, 10**6))
    if op == "append":
        c["pairs"] = rng.choice(["adjacent", "half"])
    kind = rng.choice(["decode", "decode", "turns", "prompts"])
    if kind == "decode":
        c.update(seqs=_log_int(rng, 1, 64), rows_lo=1, rows_hi=1, singles=1.0, past_lo=1, past_hi=_log_int(rng, 16, 8000))
    elif kind == "turns":
        c.update(seqs=_log_int(rng, 2, 24), rows_lo=1, rows_hi=_log_int(rng, 2, 200), singles=0.5, past_lo=1, past_hi=_log_int(rng, 2, 3000))
    else:
        c.update(seqs=rng.randint(1, 4), rows_lo=20, rows_hi=_log_int(rng, 41, 1400), singles=0.0, past_lo=1, past_hi=_log_int(rng, 2, 500))
    c["prefix"] = _log_int(rng, 10, 3000 if kind != "prompts" else 500) if op == "prefix" else 0
    return c


# ---------------------------------------------------------------- lengths

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


# ---------------------------------------------------------------- inputs

def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000 + salt)
    return g


def _normal(seed, salt, *shape):
    return torch.randn(*shape, generator=_gen(seed, salt), device=DEV, dtype=torch.float32)


def prepare(case, seed):
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # most of a vocabulary is improbable, a few tokens stand out, some are banned
        x = 2.5 * _normal(seed, 1, rows, vocab)
        x += 8.0 * (_normal(seed, 2, rows, vocab) > 3.7)
        x[:, torch.randint(0, vocab, (3,), generator=_gen(seed, 3), device=DEV)] = -math.inf
        tokens = torch.randint(0, vocab, (rows,), generator=_gen(seed, 4), device=DEV, dtype=torch.int32)
        return {"case": case, "logits": x.to(DTYPES[case["dtype"]]), "tokens": tokens}
    rows, lens = _lengths(case)
    heads, kvh, hd, page, prefix = case["heads"], case["kv_heads"], case["hd"], case["page"], case["prefix"]
    total = sum(rows)
    need = [-(-(n - prefix) // page) for n in lens]     # pages that each sequence holds of its own
    shared = -(-prefix // page)
    n_pages = sum(need) + shared + 3                    # a few pages are free
    order = torch.randperm(n_pages, generator=_gen(seed, 5), device=DEV).to(torch.int32)
    table = torch.full((len(rows), max(need)), -1, dtype=torch.int32)
    ids, at = order.cpu(), shared
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    starts = [0]
    for n in rows:
        starts.append(starts[-1] + n)
    s = {"case": case, "table": table.to(DEV), "prefix_pages": order[:max(1, shared)].contiguous(),
         "kv_len": torch.tensor(lens, dtype=torch.int32, device=DEV),
         "row_start": torch.tensor(starts, dtype=torch.int32, device=DEV), "max_rows": max(rows), "max_len": max(lens)}
    shape = (n_pages, kvh, page, hd)
    s["keys"] = _normal(seed, 1, *shape).to(DTYPES[case["dtype"]])
    s["values"] = _normal(seed, 2, *shape).to(DTYPES[case["dtype"]])
    if case["op"] == "append":
        s["qkv"] = _normal(seed, 3, total, (heads + 2 * kvh) * hd)
        s["q_out"] = torch.empty(total, heads * hd, device=DEV)
        # the tables of a model at theta 500000, as far as its longest sequence
        angle = torch.arange(max(lens), device=DEV, dtype=torch.float64)[:, None] * torch.pow(
            500000.0, -torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)[None]
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = _normal(seed, 3, total, heads * hd)
        s["out"] = torch.empty(total, heads * hd, device=DEV)
    return s


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
    own_pos = pos - c["prefix"]
    where = s["table"][seq, own_pos // page].long()
    s["keys"][where, :, own_pos % page] = rot[:, heads:].to(s["keys"].dtype)
    s["values"][where, :, own_pos % page] = x[:, heads + kvh:].to(s["values"].dtype)
    s["q_out"].copy_(rot[:, :heads].reshape(total, heads * hd))
    return s["q_out"], s["keys"], s["values"]


def _gathered(s, pool):
    """The pool's pages in the sequences' order, in f32: [seqs][kv_heads][prefix + own positions][hd]."""
    c = s["case"]
    seqs, kvh, hd, prefix = c["seqs"], c["kv_heads"], c["hd"], c["prefix"]
    x = pool[s["table"].clamp_min(0).long()].transpose(1, 2).reshape(seqs, kvh, -1, hd)
    if prefix:
        p = pool[s["prefix_pages"].long()].transpose(0, 1).reshape(kvh, -1, hd)[None, :, :prefix]
        x = torch.cat((p.expand(seqs, -1, -1, -1), x), 2)
    return x.float()


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


def _plain_logprobs(s):
    top = s["case"]["top"]
    x = s["logits"].float()
    d = x - x.amax(-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    logp = d - torch.log(total)
    chosen = logp.gather(1, s["tokens"].long()[:, None])[:, 0]
    entropy = torch.log(total[:, 0]) - torch.where(e > 0, d * e, 0.0).sum(-1) / total[:, 0]
    # equal values in the order of their ids
    ids = torch.sort(x, dim=-1, stable=True, descending=True)[1][:, :top]
    return chosen, entropy, ids.to(torch.int32), logp.gather(1, ids)


# ---------------------------------------------------------------- the library's calls

def _ok(Y, status):
    if status != 0:
        raise RuntimeError("yallma3: %d: %s" % (status, Y.lib().yl_last_error().decode()))


def _cache(Y, s):
    k = s["keys"]
    return Y.PagedCacheDesc(k.data_ptr(), s["values"].data_ptr(), Y.DTYPES[s["case"]["dtype"]], k.shape[0], k.shape[2],
                            k.shape[1], k.shape[3])


def _batch(Y, s, total):
    c, table = s["case"], s["table"]
    # one row per sequence in order needs no row_start
    start = None if total == c["seqs"] and s["max_rows"] == 1 else s["row_start"].data_ptr()
    return Y.PagedBatchDesc(c["seqs"], total, table.shape[1], s["max_len"], table.data_ptr(), s["kv_len"].data_ptr(),
                            start, c["prefix"], s["prefix_pages"].data_ptr() if c["prefix"] else None)


def _own_append(s):
    import yallma3_mini_inference_amd as Y
    c, x, q = s["case"], s["qkv"], s["q_out"]
    heads, kvh, hd, ld = c["heads"], c["kv_heads"], c["hd"], x.shape[1]
    cache, batch, at = _cache(Y, s), _batch(Y, s, x.shape[0]), x.data_ptr()
    _ok(Y, Y.lib().yl_paged_append(ctypes.byref(cache), ctypes.byref(batch), heads, q.data_ptr(), q.shape[1], at, ld,
                                   at + 4 * heads * hd, ld, at + 4 * (heads + kvh) * hd, ld,
                                   Y.ROPE_PAIRS[c["pairs"]], s["cos"].data_ptr(), s["sin"].data_ptr(), s["cos"].shape[0],
                                   torch.cuda.current_stream().cuda_stream))
    return q, s["keys"], s["values"]


def _own_attention(s):
    import yallma3_mini_inference_amd as Y
    c, q, out = s["case"], s["q"], s["out"]
    cache, batch, L = _cache(Y, s), _batch(Y, s, q.shape[0]), Y.lib()
    need = L.yl_paged_attention_workspace(ctypes.byref(cache), ctypes.byref(batch), c["heads"])
    space = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    _ok(Y, L.yl_paged_attention(out.data_ptr(), out.shape[1], q.data_ptr(), q.shape[1], ctypes.byref(cache),
                                ctypes.byref(batch), c["heads"], 1.0 / math.sqrt(c["hd"]), space.data_ptr(), need,
                                torch.cuda.current_stream().cuda_stream))
    return out


def _own_logprobs(s):
    import yallma3_mini_inference_amd as Y
    c, x, L = s["case"], s["logits"], Y.lib()
    rows, vocab, top = c["rows"], c["vocab"], c["top"]
    chosen, entropy = torch.empty(rows, device=DEV), torch.empty(rows, device=DEV)
    ids, logp = torch.empty(rows, top, device=DEV, dtype=torch.int32), torch.empty(rows, top, device=DEV)
    need = L.yl_token_logprobs_workspace(rows, vocab, top)
    space = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    _ok(Y, L.yl_token_logprobs(x.data_ptr(), Y.DTYPES[c["dtype"]], rows, vocab, vocab, s["tokens"].data_ptr(),
                               chosen.data_ptr(), entropy.data_ptr(), top, ids.data_ptr() if top else None,
                               logp.data_ptr() if top else None, space.data_ptr(), need,
                               torch.cuda.current_stream().cuda_stream))
    return chosen, entropy, ids, logp


def run(s):
    op = s["case"]["op"]
    if own:
        return (_own_append if op == "append" else _own_attention if op == "attention" else _own_logprobs)(s)
    return (_plain_append if op == "append" else _plain_attention if op == "attention" else _plain_logprobs)(s)


# ---------------------------------------------------------------- what it takes

def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        # per logit: an exponential, the two sums; the row's results beside it
        return {"bytes": n * BYTES[case["dtype"]] + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}
    rows, lens = _lengths(case)
    heads, kvh, hd, prefix = case["heads"], case["kv_heads"], case["hd"], case["prefix"]
    total, size = sum(rows), BYTES[case["dtype"]]
    if case["op"] == "append":
        # the fused rows in, q out, keys and values out, a cosine and a sine per pair
        return {"bytes": total * (4 * (2 * heads + 2 * kvh) * hd + 2 * kvh * hd * size + 4 * hd),
                "flops": 3 * total * (heads + kvh) * hd}
    own_positions = sum(n - prefix for n in lens)
    pairs = sum(n * (total_len - n) + n * (n + 1) // 2 for n, total_len in zip(rows, lens))
    # q in, out out, each held key and value once: those of the prefix once for all
    return {"bytes": 8 * total * heads * hd + 2 * (own_positions + prefix) * kvh * hd * size,
            "flops": 4 * pairs * heads * hd}


# ---------------------------------------------------------------- in 64 bits

def _exact_append(case, s):
    heads, kvh, hd, page, prefix = case["heads"], case["kv_heads"], case["hd"], case["page"], case["prefix"]
    rows, lens = _lengths(case)
    pos = torch.cat([torch.arange(n - r, n) for r, n in zip(rows, lens)]).to(DEV)
    seq = torch.cat([torch.full((r,), i) for i, r in enumerate(rows)]).to(DEV)
    # a pair as a complex number, turned by (cos, sin)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None, :]
    q, k, v = s["qkv"].double().split([heads * hd, kvh * hd, kvh * hd], 1)

    def turned(x, n):
        x = x.reshape(-1, n, hd)
        if case["pairs"] == "adjacent":
            z = torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous()) * turn
            return torch.view_as_real(z).reshape(-1, n, hd)
        z = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * turn
        return torch.cat((z.real, z.imag), -1)

    slot = s["table"].long()[seq, (pos - prefix) // page] * page + (pos - prefix) % page
    pools = []
    for pool, new in ((s["keys"], turned(k, kvh)), (s["values"], v.reshape(-1, kvh, hd))):
        flat = pool.double().permute(0, 2, 1, 3).reshape(-1, kvh, hd)
        flat[slot] = new
        pools.append(flat.reshape(pool.shape[0], page, kvh, hd).permute(0, 2, 1, 3).contiguous())
    return turned(q, heads).reshape(-1, heads * hd), pools[0], pools[1]


def _exact_attention(case, s):
    heads, kvh, hd, prefix = case["heads"], case["kv_heads"], case["hd"], case["prefix"]
    rows, lens = _lengths(case)
    out = torch.empty(sum(rows), heads, hd, device=DEV, dtype=torch.float64)
    table, shared, at = s["table"].long(), s["prefix_pages"].long(), 0
    for i, (r, n) in enumerate(zip(rows, lens)):
        held = table[i][table[i] >= 0]
        past = torch.arange(n, device=DEV)[None, :] > torch.arange(n - r, n, device=DEV)[:, None]
        for h in range(kvh):
            kv = []
            for pool in (s["keys"], s["values"]):
                x = pool[held, h].reshape(-1, hd)[:n - prefix]
                if prefix:
                    x = torch.cat((pool[shared, h].reshape(-1, hd)[:prefix], x))
                kv.append(x.double())
            g = slice(h * heads // kvh, (h + 1) * heads // kvh)
            q = s["q"][at:at + r].view(r, heads, hd)[:, g].double().transpose(0, 1).contiguous()
            score = (torch.matmul(q, kv[0].t().contiguous()) * hd ** -0.5).masked_fill(past, -math.inf)
            out[at:at + r, g] = torch.matmul(torch.softmax(score, -1), kv[1]).transpose(0, 1)
        at += r
    return out.reshape(sum(rows), heads * hd)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    x = s["logits"].double()
    logp = torch.log_softmax(x, -1)
    p = logp.exp()
    ids = torch.sort(x, dim=-1, stable=True, descending=True)[1][:, :case["top"]]
    return (logp.gather(1, s["tokens"].long()[:, None])[:, 0], -(p * logp).nan_to_num(0.0).sum(-1), ids.to(torch.int32),
            logp.gather(1, ids))
