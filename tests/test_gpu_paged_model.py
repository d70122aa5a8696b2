"""Whole layers, and a whole model, built from the per-op entries over a paged
cache, as a program that serves many conversations builds them: beside the
model's own forward path, which keeps one conversation."""
import numpy as np
import pytest

from gguf_np import Gguf
from paged_np import U, logprobs, to_cache

pytestmark = pytest.mark.gpu


class Served:
    """An F16 GGUF model's layers from the ops, its caches in pages."""

    def __init__(self, path, cfg, dtype, page, n_pages):
        from yallma3_mini_inference_amd import ops
        from yallma3_mini_inference_amd._lib import RopeParams
        from yallma3_mini_inference_amd.weight_type import QuantizedWeight
        g, self.cfg, self.hd, self.page = Gguf(path), cfg, cfg.dim // cfg.n_heads, page
        att, kv, dim, hidden = cfg.dim, cfg.n_kv_heads * self.hd, cfg.dim, cfg.hidden
        f16 = lambda name, o, n: (QuantizedWeight.upload_f16(g.raw(name)[0].view(np.float16), o, n), n, o)
        shapes = {"attn_q": (att, dim), "attn_k": (kv, dim), "attn_v": (kv, dim), "attn_output": (dim, att),
                  "ffn_gate": (hidden, dim), "ffn_up": (hidden, dim), "ffn_down": (dim, hidden)}
        self.w = [{n: f16(f"blk.{l}.{n}.weight", *s) for n, s in shapes.items()} for l in range(cfg.n_layers)]
        self.norms = [[g.f32(f"blk.{l}.{n}.weight").astype(np.float32) for n in ("attn_norm", "ffn_norm")] for l in range(cfg.n_layers)]
        self.out_norm, self.emb = g.f32("output_norm.weight").astype(np.float32), f16("token_embd.weight", cfg.vocab, dim)
        self.rows = g.f32("token_embd.weight").astype(np.float32).reshape(cfg.vocab, dim)
        self.cos, self.sin = ops.rope_table(RopeParams(self.hd, cfg.n_heads, cfg.n_kv_heads, cfg.rope_theta, 1.0, 0.0, 1.0, cfg.ctx_len),
                                            "adjacent", cfg.ctx_len)
        shape = (n_pages, cfg.n_kv_heads, page, self.hd)
        self.pools = [[to_cache(np.zeros(shape), dtype) for _ in range(2)] for _ in range(cfg.n_layers)]

    def step(self, tokens, batch):
        """Logits of all rows; their keys and values go to the batch's pages."""
        from yallma3_mini_inference_amd import ops
        from yallma3_mini_inference_amd.weight_type import matmul_f32
        cfg = self.cfg
        mm = lambda x, w: matmul_f32(x, *w)
        x = self.rows[tokens]
        for l, w in enumerate(self.w):
            xn = ops.rmsnorm_quantize(x, self.norms[l][0], cfg.rms_eps)[0]
            q, *self.pools[l] = ops.paged_append(*self.pools[l], batch, mm(xn, w["attn_q"]), mm(xn, w["attn_k"]), mm(xn, w["attn_v"]),
                                                 cfg.n_heads, "adjacent", self.cos, self.sin)
            x = x + mm(ops.paged_attention(*self.pools[l], batch, q, cfg.n_heads, self.hd ** -0.5), w["attn_output"])
            xn = ops.rmsnorm_quantize(x, self.norms[l][1], cfg.rms_eps)[0]
            x = x + mm(ops.swiglu_quantize(mm(xn, w["ffn_gate"]), mm(xn, w["ffn_up"]))[0], w["ffn_down"])
        return mm(ops.rmsnorm_quantize(x, self.out_norm, cfg.rms_eps)[0], self.emb)


@pytest.mark.parametrize("name,prefix,page", [("tiny_f16", 0, 16), ("tiny_f16", 21, 16), ("small_f16", 0, 32), ("small_f16", 40, 16)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_conversations_of_a_model(gpu, model_dir, name, prefix, page, dtype):
    """Prompts, further turns and decoded tokens of three conversations (on one
    opening, with a prefix) in ragged batches: every conversation's logits are
    the model's own of that conversation alone.

    The steps in common are the model's own arithmetic; the attention's sums
    differ in order: by at most 2 (hd + 12 + n) U of the largest value (some 300 U
    here) per layer, of which each layer after it passes on a few times as
    much: 10 layers' worth, 3000 U of the largest logit.  An f16 cache rounds
    each key and value by 2^-11: 20 times that at most (scores of some units, 10
    again).  Log probabilities follow the logits, twice for log Z's."""
    from yallma3_mini_inference_amd import Transformer, ops, synth
    path, cfg = synth.ensure(name, model_dir), synth.CONFIGS[name]
    model = Transformer(path)
    rng = np.random.default_rng(prefix + page)
    n_pages, entries = 40, 10
    served = Served(path, cfg, dtype, page, n_pages)
    order = rng.permutation(n_pages).astype(np.int32)
    shared = -(-prefix // page)
    table = order[shared:shared + 3 * entries].reshape(3, entries)
    opening = rng.integers(0, cfg.vocab, prefix)
    if prefix:                               # its own batch: the prefix's pages as a sequence's
        served.step(opening, ops.PagedBatch(order[None, :shared], np.array([prefix]), np.array([0, prefix])))
    held = [list(opening) for _ in range(3)]
    sessions = [model.create_session() for _ in range(3)]
    if prefix:
        for s in sessions:
            model.forward_x(opening.astype(np.uint32), 0, s)
    tight = 3000 * U if dtype == "f32" else 200 * 2.0 ** -11
    for rows in ([20, 1, 33], [1, 1, 1], [1, 9, 0], [1, 1, 1], [0, 2, 40]):
        new = [rng.integers(0, cfg.vocab, r) for r in rows]
        for h, t in zip(held, new):
            h.extend(t)
        starts = np.concatenate([[0], np.cumsum(rows)])
        batch = ops.PagedBatch(table, np.array([len(h) for h in held]), starts, prefix, order[:max(1, shared)] if prefix else None)
        logits = served.step(np.concatenate(new).astype(int), batch)
        tokens = rng.integers(0, cfg.vocab, len(logits))
        lp, ent, ids, tlp = ops.token_logprobs(logits, tokens, 5)
        for c in range(3):
            if not rows[c]:
                continue
            want = model.forward_x(new[c].astype(np.uint32), len(held[c]) - rows[c], sessions[c])
            last = int(starts[c + 1]) - 1
            bound = tight * np.abs(want).max()
            assert np.abs(logits[last] - want).max() <= bound, f"{np.abs(logits[last] - want).max() / np.abs(want).max() / U:.0f} U"
            rlp, rent, _, _ = logprobs(want.astype(np.float64)[None], tokens[last:last + 1], 5)
            assert abs(lp[last] - rlp[0]) <= 2 * bound + 100 * U
            assert ids[last][0] == want.argmax() or want.max() - want[ids[last][0]] <= 2 * bound
