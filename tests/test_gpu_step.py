"""One model step from the hidden state to the next token, as a host strings it together: RMS norm, grouped q/k/v, rotation
into the paged cache, attention, out-projection with the residual, norm, lm_head, sampling.  Each stage is checked against
its definition on what the device gave it; then the step is recorded and replayed with the sampled tokens."""
import numpy as np
import pytest

from cache_cases import Batch, attention_reference, rope_reference, widen
from q4_cases import assert_close
from test_gpu_sample import reference as sample_reference

pytestmark = pytest.mark.gpu

HIDDEN, Q_HEADS, KV_HEADS, HEAD, ROTARY, VOCAB, BASE = 512, 6, 2, 64, 32, 1003, 1e6


class Step:
    """Weights of one layer and a head, the buffers of up to `rows` tokens, and the calls."""

    def __init__(self, q4b, orc, ctx, batch, rows):
        self.q4b, self.ctx, self.batch, self.rows = q4b, ctx, batch, rows
        self.planes, self.weights = {}, {}
        for i, (name, n, k) in enumerate([("q", Q_HEADS * HEAD, HIDDEN), ("k", KV_HEADS * HEAD, HIDDEN), ("v", KV_HEADS * HEAD, HIDDEN),
                                          ("o", HIDDEN, Q_HEADS * HEAD), ("head", VOCAB, HIDDEN)]):
            self.planes[name] = orc.synth_weight(90 + i, 0, n, k // 64)
            self.weights[name] = ctx.upload(*self.planes[name], n, k // 64)
        rng = np.random.default_rng(1)
        self.gain = [rng.uniform(0.5, 1.5, HIDDEN).astype(np.float32) for _ in range(2)]
        self.d_gain = [ctx.to_device(g) for g in self.gain]
        self.embedding = rng.standard_normal((VOCAB, HIDDEN)).astype(np.float32)
        self.d = {name: ctx.alloc(rows * width) for name, width in
                  [("hidden", HIDDEN * 4), ("x", HIDDEN * 2), ("q", Q_HEADS * HEAD * 2), ("k", KV_HEADS * HEAD * 2),
                   ("v", KV_HEADS * HEAD * 2), ("turned", Q_HEADS * HEAD * 2), ("mixed", Q_HEADS * HEAD * 2), ("after", HIDDEN * 4),
                   ("x2", HIDDEN * 2), ("logits", VOCAB * 4), ("u", 4), ("token", 4), ("share", 4), ("heat", 4), ("p", 4)]}
        self.cache, self.described = batch.upload(q4b, ctx)
        self.rope = q4b.Rope(rotary_size=ROTARY, pairing=q4b.ROPE_HALVES, base=BASE)
        self.scale = HEAD ** -0.5

    def queue(self, rows):
        q4b, ctx, d, w = self.q4b, self.ctx, self.d, self.weights
        ctx.rmsnorm(d["hidden"].ptr, q4b.F32, self.d_gain[0].ptr, d["x"].ptr, HIDDEN, rows)
        ctx.matmul_group([w["q"], w["k"], w["v"]], d["x"].ptr, q4b.F16, rows, [d["q"].ptr, d["k"].ptr, d["v"].ptr])
        ctx.rope_append(self.cache, self.described, self.rope, d["q"].ptr, d["k"].ptr, d["v"].ptr, q4b.F16, Q_HEADS, d["turned"].ptr)
        ctx.attention(self.cache, self.described, d["turned"].ptr, Q_HEADS, d["mixed"].ptr, self.scale, window=40, sinks=2)
        ctx.matmul(w["o"], d["mixed"].ptr, q4b.F16, rows, d["after"].ptr, q4b.F32, residual_ptr=d["hidden"].ptr,
                   residual_dtype=q4b.F32, ld_residual=HIDDEN)
        ctx.rmsnorm(d["after"].ptr, q4b.F32, self.d_gain[1].ptr, d["x2"].ptr, HIDDEN, rows)
        ctx.matmul(w["head"], d["x2"].ptr, q4b.F16, rows, d["logits"].ptr, q4b.F32)
        ctx.sample(d["logits"].ptr, q4b.F32, rows, VOCAB, d["u"].ptr, d["token"].ptr, temperature=d["heat"].ptr, top_p=d["p"].ptr,
                   probability_ptr=d["share"].ptr)

    def feed(self, hidden, u):
        self.d["hidden"].upload(hidden)
        self.d["u"].upload(u)

    def check(self, orc, rows, hidden, u, heat, p, keys_before, values_before):
        read = lambda name, dtype, *shape: self.d[name].download(dtype, shape)
        b = self.batch
        x = orc.rmsnorm(hidden, self.gain[0])
        assert (read("x", np.float16, rows, HIDDEN).view(np.uint16) == x.view(np.uint16)).all()
        got = {}
        for name, heads in (("q", Q_HEADS), ("k", KV_HEADS), ("v", KV_HEADS)):
            got[name] = read(name, np.float16, rows, heads * HEAD)
            assert_close(got[name], orc.matmul(*self.planes[name], HIDDEN // 64, x, want32=False)[1], name)
        frequencies = [BASE ** (-2.0 * i / ROTARY) for i in range(ROTARY // 2)]
        places = np.concatenate([[b.place(s, i) for i in range(int(n))] for s, n in enumerate(b.counts)])
        slots = [b.slot(s, b.place(s, i)) for s, n in enumerate(b.counts) for i in range(int(n))]
        turned = read("turned", np.float16, rows, Q_HEADS, HEAD)
        keys, values = (buffer.download(np.float16, b.keys.shape) for buffer in (b.d_keys, b.d_values))
        want_keys, want_values = widen(keys_before, "f16"), widen(values_before, "f16")
        turned_k = rope_reference(got["k"].reshape(rows, KV_HEADS, HEAD), places, ROTARY, "halves", frequencies)
        for r, (page, place) in enumerate(slots):
            want_keys[page, :, place], want_values[page, :, place] = turned_k[r], got["v"][r].reshape(KV_HEADS, HEAD)
        # fp16's rounding of the result, fp32's of the turn
        near = lambda a, w: (np.abs(a - w) <= 2.0 ** -11 * np.abs(w) + 2.0 ** -20 * np.abs(w).max() + 2.0 ** -25).all()
        assert near(widen(keys, "f16"), want_keys) and (widen(values, "f16") == want_values).all()
        assert near(widen(turned, "f16"), rope_reference(got["q"].reshape(rows, Q_HEADS, HEAD), places, ROTARY, "halves", frequencies))
        b.keys, b.values = keys, values
        mixed = read("mixed", np.float16, rows, Q_HEADS, HEAD)
        want, tolerance = attention_reference(b, turned, Q_HEADS, self.scale, 40, 2)
        assert (np.abs(widen(mixed, "f16") - want) <= tolerance).all()
        after = read("after", np.float32, rows, HIDDEN)
        assert_close(after, orc.matmul(*self.planes["o"], Q_HEADS * HEAD // 64, mixed.reshape(rows, -1), residual=hidden,
                                       want32=False)[1], "out-projection")
        logits = read("logits", np.float32, rows, VOCAB)
        assert_close(logits, orc.matmul(*self.planes["head"], HIDDEN // 64, orc.rmsnorm(after, self.gain[1]), want32=False)[1], "head")
        tokens = read("token", np.uint32, rows)
        for r in range(rows):
            token, share, margin = sample_reference(logits[r].astype(np.float64), float(u[r]), float(heat[r]), 0, float(p[r]))
            assert margin < 1e-8 or tokens[r] == token
        return tokens


def test_a_prompt_and_recorded_steps_after_it(q4b, orc):
    with q4b.Q4Context(0) as ctx:
        rng = np.random.default_rng(2)
        counts = [37, 5]
        batch = Batch(rng, counts, counts, 16, KV_HEADS, HEAD, "f16", spare=0)
        # room for the tokens to come, in pages of their own
        batch.stride, batch.pages = 4, 8
        batch.table = rng.permutation(8).astype(np.uint32).reshape(2, 4)
        batch.keys = rng.standard_normal((8, KV_HEADS, 16, HEAD)).astype(np.float16)
        batch.values = rng.standard_normal(batch.keys.shape).astype(np.float16)
        step = Step(q4b, orc, ctx, batch, 42)
        heat, p = rng.uniform(0.5, 1.5, 42).astype(np.float32), rng.uniform(0.5, 1.0, 42).astype(np.float32)
        step.d["heat"].upload(heat)
        step.d["p"].upload(p)
        hidden, u = step.embedding[rng.integers(0, VOCAB, 42)] * 0.5, rng.random(42).astype(np.float32)
        before = batch.keys.copy(), batch.values.copy()
        step.feed(hidden, u)
        step.queue(42)
        tokens = step.check(orc, 42, hidden, u, heat, p, *before)
        last = tokens[[36, 41]]
        # from here one token per sequence: the same calls, recorded once
        batch.counts, batch.begin, batch.used, batch.tokens = np.array([1, 1]), np.array([0, 1, 2], dtype=np.uint32), 2, 2
        batch.d_begin.upload(batch.begin)
        step.described.tokens, step.described.most_tokens = 2, 1
        for warm in range(2):   # the shapes' workspaces; a recorded pass allocates nothing
            if warm:
                ctx.graph_begin()
            step.queue(2)
            if warm:
                graph = ctx.graph_end()
        ctx.sync()
        batch.keys, batch.values = (buffer.download(np.float16, batch.keys.shape) for buffer in (batch.d_keys, batch.d_values))
        for _ in range(5):
            batch.lengths = batch.lengths + 1
            batch.d_lengths.upload(batch.lengths.astype(np.uint32))
            hidden, u = step.embedding[last] * 0.5, rng.random(2).astype(np.float32)
            before = batch.keys.copy(), batch.values.copy()
            step.feed(hidden, u)
            graph.launch()
            last = step.check(orc, 2, hidden, u, heat, p, *before)
