"""yl_adjust_logits against the rules token by token in 64 bits: every step is
rounded to f32 and the result once to the logits' type."""
import ctypes as C

import numpy as np
import pytest

from hip_rt import Graph, Stream, buffer, filled
from paged_np import to_cache, widened

pytestmark = pytest.mark.gpu

# half a step of the type, relative, and half of its least subnormal
STEP = {"f32": (2.0 ** -24, 2.0 ** -150), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 2.0 ** -134)}


class Rows:
    def __init__(self, rows, vocab, dtype, seed=0, past=40, biases=9, grammars=3, ties=True):
        self.rng = r = np.random.default_rng(seed)
        self.dtype, self.vocab = dtype, vocab
        self.x = to_cache((3 * r.standard_normal((rows, vocab))).astype(np.float32), dtype)
        sizes = r.integers(0, past + 1, rows)
        self.tokens = [np.minimum(r.zipf(1.3, n) - 1, vocab + 3).astype(np.uint32) for n in sizes]     # repeated; some are no ids
        self.n_prompt = np.array([r.integers(0, n + 2) for n in sizes], np.uint32)
        self.repetition, self.presence, self.frequency = (r.uniform(*b, rows).astype(np.float32) for b in ((0.7, 2.0), (-1.0, 1.5), (-0.3, 0.5)))
        self.biases = [(r.integers(0, vocab + 2, n).astype(np.uint32), (4 * r.standard_normal(n)).astype(np.float32))
                       for n in r.integers(0, biases + 1, rows)]
        self.mask = r.integers(0, 1 << 32, (grammars, -(-vocab // 32)), dtype=np.uint64).astype(np.uint32)
        self.mask_of = r.integers(-1, grammars + 1, rows).astype(np.int32)      # none, a grammar, one that there is not

    def rules(self, **kw):
        r = dict(tokens=self.tokens, n_prompt=self.n_prompt, repetition=self.repetition, presence=self.presence, frequency=self.frequency,
                 biases=self.biases, mask=self.mask, mask_of=self.mask_of)
        r.update(kw)
        return r

    def check(self, out, tokens=None, n_prompt=None, repetition=None, presence=None, frequency=None, biases=None, mask=None, mask_of=None):
        """The bound: a quotient or product, the frequency's product, two
        differences and the bias's sum, each rounded by U of its size in f32; the result by half a step of its type."""
        U, out = 2.0 ** -24, widened(out)
        step, least = STEP[self.dtype]
        for r in range(len(out)):
            x = widened(self.x[r:r + 1])[0]
            size = np.abs(np.where(np.isfinite(x), x, 0))
            if tokens is not None:
                told = [int(t) for t in tokens[r] if t < self.vocab]
                answer = [int(t) for t in tokens[r][(n_prompt[r] if n_prompt is not None else 0):] if t < self.vocab]
                rep, pre, fre = (float(v[r]) if v is not None else d for v, d in ((repetition, 1.0), (presence, 0.0), (frequency, 0.0)))
                for t in set(told):
                    x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
                    n = answer.count(t)
                    size[t] = max(size[t], abs(x[t]) if np.isfinite(x[t]) else 0)
                    if n:
                        x[t] = x[t] - fre * n - pre
                        size[t] += abs(fre * n) + abs(pre)
            if biases is not None:
                for i, b in {int(i): float(b) for i, b in zip(*biases[r])}.items():
                    if i < self.vocab:
                        x[i] += b
                        size[i] += abs(b) if np.isfinite(b) else 0
            if mask is not None:
                g = int(mask_of[r]) if mask_of is not None else r
                ids = np.arange(self.vocab)
                if g >= len(mask):
                    x[:] = -np.inf
                elif g >= 0:
                    x[(mask[g][ids // 32] >> (ids % 32)) & 1 == 0] = -np.inf
            fine = np.isfinite(x)
            assert np.array_equal(np.isnan(x), np.isnan(out[r])) and np.array_equal(x[~fine & ~np.isnan(x)], out[r][~fine & ~np.isnan(x)])
            changed = widened(self.x[r:r + 1])[0] != x
            assert np.array_equal(out[r][fine & ~changed], x[fine & ~changed])       # what no rule changes keeps its bits
            err = np.abs(out[r][fine] - x[fine])
            assert (err <= (5 * U * size + step * (1 + 2.0 ** -8) * np.abs(x) + 5 * U * step * size + least)[fine]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (5, 8), (4, 31), (4, 33), (9, 511), (3, 2048), (2, 8191), (2, 8192), (2, 8193), (3, 20001), (2, 128256)])
def test_all_rules(gpu, dtype, rows, vocab):
    from yallma3_mini_inference_amd import ops
    w = Rows(rows, vocab, dtype, seed=vocab)
    w.check(ops.adjust_logits(w.x, **w.rules()), **w.rules())


@pytest.mark.parametrize("only", [["tokens", "repetition"], ["tokens", "presence"], ["tokens", "frequency", "n_prompt"], ["tokens", "repetition", "frequency"],
                                  ["biases"], ["mask"], ["mask", "mask_of"], ["tokens"], ["mask", "mask_of", "biases"], []])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_single_rules(gpu, dtype, only):
    from yallma3_mini_inference_amd import ops
    w = Rows(3, 9001, dtype, seed=1)
    rules = {k: v for k, v in w.rules().items() if k in only}
    w.check(ops.adjust_logits(w.x, **rules), **rules)


def test_long_histories(gpu):
    """More tokens than a workgroup has threads, one id many times, and a row whose tokens are all its prompt's."""
    from yallma3_mini_inference_amd import ops
    w = Rows(4, 20000, "f32", seed=2)
    r = w.rng
    w.tokens = [np.concatenate([np.full(70000, 7), r.integers(0, 20000, 60000)]).astype(np.uint32), r.integers(0, 30, 5000).astype(np.uint32),
                np.arange(19990, 20010).astype(np.uint32), np.empty(0, np.uint32)]
    w.n_prompt = np.array([3, 0xFFFFFFFF, 5, 9], np.uint32)
    w.frequency *= np.float32(0.01)
    w.check(ops.adjust_logits(w.x, **w.rules()), **w.rules())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_values_that_are_no_numbers(gpu, dtype):
    """-inf stays so under penalties; NaN stays NaN unless it is masked; infinite biases; logits of zero."""
    from yallma3_mini_inference_amd import ops
    w = Rows(4, 300, dtype, seed=3)
    x = widened(w.x).astype(np.float32)
    x[:, 0:4] = [-np.inf, np.nan, np.inf, 0.0]
    x[:, 40:44] = [-np.inf, np.nan, np.inf, -0.0]
    w.x = to_cache(np.nan_to_num(x, nan=0.0, posinf=np.inf, neginf=-np.inf), dtype).copy()
    w.x[np.isnan(x)] = 0x7FC0 if dtype == "bf16" else np.nan
    w.tokens = [np.array([0, 1, 2, 3, 50, 50], np.uint32)] * 4
    w.biases = [(np.array([40, 41, 42, 43, 60, 61], np.uint32), np.array([1, 1, 1, 1, np.inf, -np.inf], np.float32))] * 4
    w.n_prompt[:] = [0, 2, 5, 6]
    rules = w.rules()
    w.check(ops.adjust_logits(w.x, **rules), **rules)


def test_large_results(gpu):
    """A row whose grammar allows nothing, and f16 logits that a bias takes past the type's largest."""
    from yallma3_mini_inference_amd import ops
    x = np.full((2, 64), 60000.0, np.float16)
    out = ops.adjust_logits(x, biases=[(np.array([5, 6], np.uint32), np.array([9000.0, -9000.0], np.float32))] * 2, mask=np.zeros((1, 2), np.uint32), mask_of=[-1, 0])
    assert out[0, 5] == np.inf and out[0, 6] == np.float16(51000.0) and (out[0, 7:] == 60000).all() and np.isneginf(out[1]).all()


class Call:
    """A call on device arrays: rows at odd strides from an odd address, into another array or in place."""

    def __init__(self, yl, w, ld, out_ld, in_place):
        self.yl, self.w, self.ld, self.out_ld, self.in_place = yl, w, ld, out_ld, in_place
        rows = len(w.x)
        host = np.zeros(1 + rows * ld, w.x.dtype)
        host[1:].reshape(rows, ld)[:, :w.vocab] = w.x
        self.size = host.itemsize
        self.x, self.out = buffer(host), filled(1 + rows * out_ld, 7, w.x.dtype)
        lists = [np.concatenate(w.tokens), np.cumsum([0] + [len(t) for t in w.tokens]).astype(np.uint32), w.n_prompt, w.repetition, w.presence, w.frequency,
                 np.concatenate([b[0] for b in w.biases]), np.concatenate([b[1] for b in w.biases]), np.cumsum([0] + [len(b[0]) for b in w.biases]).astype(np.uint32),
                 w.mask, w.mask_of]
        self.held = h = [buffer(a) for a in lists]
        self.rules = yl.LogitRules(h[0].ptr, h[1].ptr, h[2].ptr, lists[0].size, h[3].ptr, h[4].ptr, h[5].ptr, h[6].ptr, h[7].ptr, h[8].ptr, lists[6].size,
                                   h[9].ptr, w.mask.shape[1], w.mask.shape[0], h[10].ptr)

    def __call__(self, stream=None):
        x = self.x.ptr + self.size
        out = x if self.in_place else self.out.ptr + self.size
        self.yl.check(self.yl.lib().yl_adjust_logits(out, self.out_ld, x, self.ld, self.yl.DTYPES[self.w.dtype], len(self.w.x), self.w.vocab,
                                                     C.byref(self.rules), stream))

    def result(self):
        self.yl.check(self.yl.lib().yl_synchronize())
        rows = (self.x if self.in_place else self.out).numpy()[1:].reshape(len(self.w.x), self.out_ld)
        return rows[:, :self.w.vocab], rows[:, self.w.vocab:]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("in_place", [False, True])
def test_strides_and_alignment(gpu, dtype, in_place):
    w = Rows(6, 8205, dtype, seed=4)
    call = Call(gpu, w, 8211, 8211 if in_place else 8209, in_place)
    call()
    out, between = call.result()
    w.check(out, **w.rules())
    assert (between == (0 if in_place else 7)).all()


def test_more_rows_than_a_grid_holds(gpu):
    from yallma3_mini_inference_amd import ops
    rows = 65540
    x = np.random.default_rng(5).standard_normal((rows, 3)).astype(np.float32)
    out = ops.adjust_logits(x, tokens=[[i % 3] for i in range(rows)], presence=np.ones(rows))
    want = x.copy()
    want[np.arange(rows), np.arange(rows) % 3] -= 1
    assert np.array_equal(out, want)


def test_starts_that_do_not_ascend(gpu):
    """Starts beyond the list, or falling: entries of the list at most, or none."""
    w = Rows(3, 100, "f32", seed=6)
    call = Call(gpu, w, 100, 100, False)
    call.held[1].upload(np.array([0, 0xFFFFFFFF, 2, 0x80000000], np.uint32))
    call.held[8].upload(np.array([5, 1, 0xFFFFFFF0, 0xFFFFFFFF], np.uint32))
    call()
    out, _ = call.result()
    assert np.isfinite(out[w.mask_of < 0]).all()


def test_a_captured_call(gpu):
    """Replayed with other tokens, lengths and grammars, an eager call between the replays; then scored."""
    w = Rows(4, 5000, "f32", seed=7, past=60)
    captured, eager = Call(gpu, w, 5000, 5000, False), Call(gpu, w, 5000, 5000, False)
    graph = Graph(captured)
    n, tokens = len(np.concatenate(w.tokens)), np.concatenate(w.tokens)
    for k in range(4):
        cuts = np.sort(w.rng.integers(0, n + 1, 3))
        starts = np.concatenate([[0], cuts, [n]]).astype(np.uint32)
        tokens = w.rng.permutation(tokens)
        w.tokens = [tokens[a:b] for a, b in zip(starts, starts[1:])]
        w.mask_of = w.rng.integers(-1, 3, 4).astype(np.int32)
        for c in (captured, eager):
            c.held[0].upload(tokens)
            c.held[1].upload(starts)
            c.held[10].upload(w.mask_of)
        graph.replay()
        eager()
        a, b = captured.result()[0], eager.result()[0]
        assert np.array_equal(a, b)
        w.check(a, **w.rules())


def test_streams_side_by_side(gpu):
    ws = [Rows(20, 30001, "f16", seed=8), Rows(2, 128256, "f32", seed=9)]
    calls, streams = [Call(gpu, w, w.vocab, w.vocab, False) for w in ws], [Stream() for _ in ws]
    gpu.check(gpu.lib().yl_synchronize())
    for _ in range(5):
        for c, st in zip(calls, streams):
            c(st.handle)
    for c, w in zip(calls, ws):
        w.check(c.result()[0], **w.rules())


def test_adjusted_then_scored(gpu):
    """The rules before the scoring, as a step of constrained decoding runs them: banned ids have probability 0 and never come up."""
    from yallma3_mini_inference_amd import ops
    w = Rows(5, 3001, "f32", seed=10, grammars=4)
    w.mask_of = np.array([0, 1, -1, 3, 2], np.int32)
    out = ops.adjust_logits(w.x, **w.rules())
    lp, ent, ids, tlp = ops.token_logprobs(out, np.full(5, 17), top=5)
    for r in range(5):
        p = np.exp(out[r].astype(np.float64) - out[r].max())
        p /= p.sum()
        assert np.array_equal(ids[r], np.lexsort((np.arange(3001), -out[r]))[:5])
        assert np.isfinite(out[r][ids[r]]).all() and np.abs(np.exp(tlp[r]) - p[ids[r]]).max() <= 1e-5
        assert np.isneginf(lp[r]) == np.isneginf(out[r, 17])
