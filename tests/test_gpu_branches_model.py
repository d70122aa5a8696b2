"""A whole model from the per-op entries over MXFP4 pages that the page
operations hand out, branch, free and move, its tokens chosen under rules: as a
program that samples several answers to a conversation runs them."""
import numpy as np
import pytest

import mx_np as X
from paged_np import U
from test_gpu_paged_model import Served

pytestmark = pytest.mark.gpu


class ServedMx(Served):
    """Served over MXFP4 pages; beside it the same layers over f32 pages of the values that those stand for."""

    def __init__(self, path, cfg, page, n_pages):
        super().__init__(path, cfg, "f32", page, n_pages)
        shape = (n_pages, cfg.n_kv_heads, page, 17 * self.hd // 32)
        self.pools = [tuple(np.zeros(shape, np.uint8) for _ in range(2)) for _ in range(cfg.n_layers)]

    def step(self, tokens, batch):
        """(logits of all rows, those of the f32 pages)"""
        from yallma3_mini_inference_amd import ops
        from yallma3_mini_inference_amd.weight_type import matmul_f32
        cfg = self.cfg
        mm = lambda x, w: matmul_f32(x, *w)  # noqa: E731
        xs = [self.rows[tokens], self.rows[tokens]]
        for l, w in enumerate(self.w):
            for side in range(2):
                x = xs[side]
                xn = ops.rmsnorm_quantize(x, self.norms[l][0], cfg.rms_eps)[0]
                qkv = mm(xn, w["attn_q"]), mm(xn, w["attn_k"]), mm(xn, w["attn_v"])
                if side == 0:
                    q, *self.pools[l] = ops.paged_append(*self.pools[l], batch, *qkv, cfg.n_heads, "adjacent", self.cos, self.sin)
                    pools = self.pools[l]
                else:                        # (its own keys and values would be rounded to other codes here and there)
                    pools = [X.unpacked(p) for p in self.pools[l]]
                    q = ops.paged_append(*pools, batch, *qkv, cfg.n_heads, "adjacent", self.cos, self.sin)[0]
                x = x + mm(ops.paged_attention(*pools, batch, q, cfg.n_heads, self.hd ** -0.5), w["attn_output"])
                xn = ops.rmsnorm_quantize(x, self.norms[l][1], cfg.rms_eps)[0]
                xs[side] = x + mm(ops.swiglu_quantize(mm(xn, w["ffn_gate"]), mm(xn, w["ffn_up"]))[0], w["ffn_down"])
        return [mm(ops.rmsnorm_quantize(x, self.out_norm, cfg.rms_eps)[0], self.emb) for x in xs]


@pytest.mark.parametrize("name,page,n_pages", [("tiny_f16", 16, 30), ("small_f16", 32, 20)])
def test_answers_of_a_model(gpu, model_dir, name, page, n_pages):
    """Two conversations, three answers to each, two of which go on after the others and the conversations have ended.

    Both sides run the same steps but for the attention, whose sums differ in order: bounds as in
    test_gpu_paged_model.py, 3000 U of the largest logit."""
    from yallma3_mini_inference_amd import ops, synth
    path, cfg = synth.ensure(name, model_dir), synth.CONFIGS[name]
    rng = np.random.default_rng(page)
    served = ServedMx(path, cfg, page, n_pages)
    rows = 8
    t = ops.PagedTables(np.full((rows, 5), -1), np.zeros(rows), np.zeros(n_pages), page)
    told = [list(rng.integers(0, cfg.vocab, n)) for n in (20, 33)] + [[] for _ in range(6)]
    prompts = [len(x) for x in told]

    def check(both):
        got, want = both
        assert np.abs(got - want).max() <= 3000 * U * np.abs(want).max(), f"{np.abs(got - want).max() / np.abs(want).max() / U:.0f} U"
        return got

    # the prompts
    want = np.zeros(rows, int)
    want[:2] = prompts[:2]
    assert ops.paged_reserve(t, want) == 0
    t.kv_len[:] = want
    batch = ops.PagedBatch(t.page_table[:2], t.kv_len[:2], np.cumsum([0, *prompts[:2]]))
    logits = check(served.step(np.array(told[0] + told[1]), batch))
    last = logits[np.cumsum(prompts[:2]) - 1]
    # three answers each, whose first tokens are the most probable ones under a grammar of their own
    lacking, served.pools = ops.paged_fork(t, served.pools, [0, 0, 0, 1, 1, 1], range(2, 8))
    assert lacking == 0 and np.array_equal(t.kv_len[2:], np.repeat(t.kv_len[:2], 3))
    for c in range(2, 8):
        told[c] = list(told[(c - 2) // 3])
        prompts[c] = len(told[c])
    grammars = rng.integers(0, 1 << 32, (3, -(-cfg.vocab // 32)), dtype=np.uint64).astype(np.uint32)
    allowed = (grammars[:, np.arange(cfg.vocab) // 32] >> (np.arange(cfg.vocab) % 32)) & 1

    def choose(live, logits, of):
        out = ops.adjust_logits(logits, [told[c] for c in live], [prompts[c] for c in live], [1.2] * len(live), [0.5] * len(live),
                                [0.1] * len(live), [([7, 3], [1.5, -2.0])] * len(live), grammars, of)
        _, _, ids, tlp = ops.token_logprobs(out, np.zeros(len(live)), top=4)
        for r, c in enumerate(live):
            x = logits[r].astype(np.float64)
            for i in set(told[c]):
                x[i] = x[i] / np.float32(1.2) if x[i] > 0 else x[i] * np.float32(1.2)
            for i in set(told[c][prompts[c]:]):
                x[i] -= 0.5 + np.float32(0.1) * told[c][prompts[c]:].count(i)
            x[7], x[3] = x[7] + 1.5, x[3] - 2.0
            if of[r] >= 0:
                x[allowed[of[r]] == 0] = -np.inf
            assert np.array_equal(np.isneginf(x), np.isneginf(out[r]))
            fine = np.isfinite(x)
            assert np.abs(out[r][fine] - x[fine]).max() <= 8 * U * (np.abs(logits[r]).max() + 4)
            assert ids[r][0] == np.lexsort((np.arange(cfg.vocab), -out[r]))[0] and np.isfinite(out[r][ids[r][0]])
        return ids[:, 0].astype(int)

    first = choose(range(2, 8), np.repeat(last, 3, 0), [0, 1, -1, 2, -1, 0])
    live = list(range(2, 8))
    for step in range(20):                    # past page ends
        for c, token in zip(live, first):
            told[c].append(int(token))
        want = t.kv_len.astype(int)
        want[live] += 1
        assert ops.paged_reserve(t, want) == 0
        t.kv_len[:] = want
        logits = check(served.step(first, ops.PagedBatch(t.page_table[live], t.kv_len[live])))
        first = choose(live, logits, [[0, 1, -1, 2, -1, 0][c - 2] for c in live])
        if step == 2:                         # the conversations and all answers but two end, the rest moves together
            ops.paged_release(t, [0, 1, 2, 3, 6, 7])
            first, live = first[2:4], [4, 5]
            used, served.pools = ops.paged_compact(t, served.pools)
            named = t.page_table[t.page_table >= 0]
            assert used == len(named) == len(set(named)) == named.max() + 1 < n_pages
    # branches that shared pages end with histories of their own: what the pages hold is what each was told
    k, _ = ops.paged_gather(*served.pools[0], ops.PagedBatch(t.page_table[live], t.kv_len[live], np.cumsum([0, *t.kv_len[live]])), int(t.kv_len[live].sum()))
    at = 0
    for c in live:
        n = int(t.kv_len[c])
        assert n == len(told[c])
        x = served.rows[np.array(told[c])]
        from yallma3_mini_inference_amd.weight_type import matmul_f32
        xn = ops.rmsnorm_quantize(x, served.norms[0][0], cfg.rms_eps)[0]
        scratch = np.zeros((5, cfg.n_kv_heads, page, served.hd), np.float32)
        own = ops.PagedBatch(np.arange(5)[None], np.array([n]), np.array([0, n]))
        kk, vv = (matmul_f32(xn, *served.w[0][w]) for w in ("attn_k", "attn_v"))
        _, ks, vs = ops.paged_append(scratch, scratch, own, None, kk, vv, cfg.n_heads, "adjacent", served.cos, served.sin)
        want_k, _ = ops.paged_gather(ks, vs, own, n)
        assert np.array_equal(k[at:at + n], X.rounded(want_k.reshape(n, cfg.n_kv_heads, served.hd)).reshape(n, -1))
        at += n
